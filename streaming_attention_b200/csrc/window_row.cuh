// A row of the windowed attention computed from its visible keys alone: what the
// tensor-core kernels do with rows that came out non-finite, since a hidden NaN or
// infinity reaches a product as 0 times it.
#pragma once

#include <math.h>

#include "serving.cuh"

namespace sa {

constexpr int kRepairWidth = 128;   // head widths that the tensor-core kernels take at most

// The non-finite columns of one output row (they have been written by this
// warp's lanes, or before a barrier), in float32 by one warp: lanes hold columns,
// keys come four at a time under a running maximum, and a key whose weight is 0
// is not looked at, whatever its value holds.  It ends early once every such
// column is NaN: it stays that.  `beat`, where given, counts on while it works,
// for those who wait for this warp (Abort::beats).  32 heads x 8192 queries of
// 128, window 1024, 188 us without such values: 0.7 ms where all see a NaN among
// the first tokens, 67 ms where one hidden beside them makes all of the rows ones
// to repair (0.3 us a key for each of an SM's eight warps, latency).
template <int DT>
__device__ __noinline__ void repair_row(const WindowArgs& a, int64_t qoff, int64_t koff, int64_t voff, int64_t ooff,
                                        int64_t p, int64_t m, int* beat) {
  using T = typename Elem<DT>::T;
  constexpr int kMine = kRepairWidth / 32, kKeys = 4;
  const int lane = threadIdx.x & 31;
  const T* q = static_cast<const T*>(a.q) + qoff;
  const T* k = static_cast<const T*>(a.k) + koff;
  const T* v = static_cast<const T*>(a.v) + voff;
  T* out = static_cast<T*>(a.out) + ooff;
  const KeyRanges kr = key_ranges(p, p, m, a.window, a.sinks);
  const int64_t count = kr.first + kr.end - kr.begin, k_n = a.k_n, v_n = a.v_n;
  const float scale = a.scale;
  float qv[kMine], acc[kMine], top = -INFINITY, l = 0.0f;
  int kc[kMine], vc[kMine];   // columns, held within the rows so that every load can be made, and early
  bool wanted[kMine], in[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int c = lane + 32 * i;
    in[i] = c < a.d;
    kc[i] = min(c, a.d - 1);
    vc[i] = min(c, a.dv - 1);
    qv[i] = in[i] ? to_f32(q[c]) : 0.0f;
    wanted[i] = c < a.dv && !(fabsf(to_f32(out[c])) < INFINITY);
    acc[i] = 0.0f;
  }
#pragma unroll 1
  for (int64_t u = 0; u < count; u += kKeys) {
    float x[kKeys], mx = -INFINITY;
    T y[kKeys][kMine], z[kKeys][kMine];
    bool nan = false;
#pragma unroll
    for (int e = 0; e < kKeys; ++e) {
      const int64_t w = min(u + e, count - 1), j = w < kr.first ? w : kr.begin + w - kr.first;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        y[e][i] = k[j * k_n + kc[i]];
        z[e][i] = v[j * v_n + vc[i]];
      }
    }
#pragma unroll
    for (int e = 0; e < kKeys; ++e) {
      x[e] = 0.0f;
#pragma unroll
      for (int i = 0; i < kMine; ++i) x[e] = fmaf(qv[i], in[i] ? to_f32(y[e][i]) : 0.0f, x[e]);
    }
#pragma unroll
    for (int e = 0; e < kKeys; ++e) {
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) x[e] += __shfl_xor_sync(0xffffffffu, x[e], d);
      x[e] = u + e < count ? x[e] * scale : -INFINITY;
      nan |= x[e] != x[e];
      mx = fmaxf(mx, x[e]);
    }
    if (beat && lane == 0) atomicAdd(beat, 1);
    if (nan) {   // a score that is NaN: so is the row
      l = NAN;
      break;
    }
    if (mx > top) {
      const float f = expf(top - mx);   // from -inf: 0
      l *= f;
#pragma unroll
      for (int i = 0; i < kMine; ++i) acc[i] = f == 0.0f ? 0.0f : acc[i] * f;
      top = mx;
    }
    if (top == -INFINITY) continue;
    bool open = false;
#pragma unroll
    for (int e = 0; e < kKeys; ++e) {
      const float w = u + e < count ? expf(x[e] - top) * 0x1p-24f : 0.0f;
      l += w;
#pragma unroll
      for (int i = 0; i < kMine; ++i)
        acc[i] = w != 0.0f ? fmaf(w, to_f32(z[e][i]), acc[i]) : acc[i];
    }
#pragma unroll
    for (int i = 0; i < kMine; ++i) open |= wanted[i] && acc[i] == acc[i];
    if (!__any_sync(0xffffffffu, open)) break;
  }
#pragma unroll
  for (int i = 0; i < kMine; ++i)
    if (wanted[i]) out[lane + 32 * i] = from_f32<T>(l == 0.0f ? 0.0f : acc[i] / l);
}

}  // namespace sa
