// A row of the windowed attention computed from its visible keys alone: what the
// tensor-core kernels do with rows that a hidden NaN or infinity reached (0 times
// it in a product).
#pragma once

#include <math.h>

#include "serving.cuh"

namespace sa {

// One output row from its visible keys alone, in float32 by one thread.
template <int DT>
__device__ __noinline__ void row_again(const WindowArgs& a, int64_t qoff, int64_t koff, int64_t voff, int64_t ooff,
                                       int64_t p, int64_t m) {
  using T = typename Elem<DT>::T;
  const T* q = static_cast<const T*>(a.q) + qoff;
  const T* k = static_cast<const T*>(a.k) + koff;
  const T* v = static_cast<const T*>(a.v) + voff;
  T* out = static_cast<T*>(a.out) + ooff;
  const KeyRanges kr = key_ranges(p, p, m, a.window, a.sinks);
  auto score = [&](int64_t j) {
    float x = 0.0f;
    for (int c = 0; c < a.d; ++c) x = fmaf(to_f32(q[c]), to_f32(k[j * a.k_n + c]), x);
    return x * a.scale;
  };
  float top = -INFINITY;
  bool nan = false;
  const int64_t count = kr.first + kr.end - kr.begin;
  for (int64_t u = 0; u < count; ++u) {
    const float x = score(u < kr.first ? u : kr.begin + u - kr.first);
    nan |= x != x;
    top = fmaxf(top, x);
  }
  top = nan ? NAN : (top == -INFINITY ? 0.0f : top);
  for (int c0 = 0; c0 < a.dv; c0 += 16) {
    float acc[16], l = 0.0f;
    for (int c = 0; c < 16; ++c) acc[c] = 0.0f;
    for (int64_t u = 0; u < count; ++u) {
      const int64_t j = u < kr.first ? u : kr.begin + u - kr.first;
      const float e = expf(score(j) - top) * 0x1p-24f;
      l += e;
      if (e != 0.0f)
        for (int c = 0; c < 16 && c0 + c < a.dv; ++c) acc[c] = fmaf(e, to_f32(v[j * a.v_n + c0 + c]), acc[c]);
    }
    for (int c = 0; c < 16 && c0 + c < a.dv; ++c) out[c0 + c] = from_f32<T>(l == 0.0f ? 0.0f : acc[c] / l);
  }
}

}  // namespace sa
