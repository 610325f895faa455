// Attention of a request's newest tokens over its pages of the 4-bit cache.
//
//   out = softmax over the visible tokens j of scale q.k_j, times v_j;
//   query i of n stands at position length - n + i; visible as in the windowed
//   attention (serving.cuh); nothing visible gives zeros.
//
// One CTA per (query head and token, request), four warps; a warp takes every
// fourth visible token, a lane the columns lane, lane + 32, ...; each warp
// keeps a running maximum, sum and float32 output, joined at the end.
#include <math.h>

#include "kv4.cuh"

namespace sa {

namespace {

constexpr int kWarps = 4;
constexpr int kCols = 8;   // columns per lane: d <= 256

template <int DT>
__global__ void __launch_bounds__(kWarps * 32) attend_kernel(const Kv4AttendArgs a) {
  using T = typename Elem<DT>::T;
  __shared__ float o_s[kWarps][256];
  __shared__ float m_s[kWarps], l_s[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.x % a.heads, i = blockIdx.x / a.heads, r = blockIdx.y;
  const int hk = h / (a.heads / a.c.heads);
  const int64_t length = max(a.lengths[r], 0);
  const int64_t cap = (int64_t)a.width << a.c.page_shift;
  if (length > cap && threadIdx.x == 0) report(a.status, kBadLength, r);
  const int64_t p = length - a.n + i;
  const KeyRanges kr = key_ranges(p, p, min(length, cap), a.window, a.sinks);
  const T* q = static_cast<const T*>(a.q) + r * a.q_r + i * a.q_n + h * a.q_h;
  float qv[kCols], acc[kCols];
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    qv[c] = lane + 32 * c < a.c.d ? to_f32(q[lane + 32 * c]) * a.scale : 0.0f;
    acc[c] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  const int bytes = a.c.dp >> 1;
  for (int part = 0; part < 2; ++part) {
    const int64_t jb = part ? kr.begin : 0, je = part ? kr.end : kr.first;
    for (int64_t j = jb + warp; j < je; j += kWarps) {
      const int page = a.tables[(int64_t)r * a.width + (j >> a.c.page_shift)];
      if (page < 0 || page >= a.c.pages) {
        if (lane == 0) report(a.status, kBadPage, page);
        continue;
      }
      const int off = (int)(j & ((1 << a.c.page_shift) - 1));
      const int64_t cell = ((int64_t)page * a.c.heads + hk) << a.c.page_shift;
      const __nv_bfloat16* kp = a.c.k_params + 2 * (cell + off);
      const __nv_bfloat16* vp = a.c.v_params + 2 * (cell + off);
      const float ks = __bfloat162float(kp[0]), km = __bfloat162float(kp[1]);
      const float vs = __bfloat162float(vp[0]), vm = __bfloat162float(vp[1]);
      float dot = 0.0f;
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        const int col = lane + 32 * c;
        if (col < a.c.d) {
          const uint32_t byte = a.c.k_codes[(cell + off) * bytes + (col >> 1)];
          dot = fmaf(qv[c], fmaf((float)((byte >> (4 * (col & 1))) & 15), ks, km), dot);
        }
      }
#pragma unroll
      for (int s = 16; s >= 1; s >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, s);
      const float m_new = fmaxf(m, dot);
      const float alpha = m_new == -INFINITY ? 1.0f : expf(m - m_new);
      const float e = m_new == -INFINITY ? 0.0f : expf(dot - m_new);
      m = m_new;
      l = l * alpha + e;
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        const int col = lane + 32 * c;
        if (col < a.c.d) {
          const uint32_t byte = a.c.v_codes[cell * bytes + ((int64_t)(off >> 2) * bytes + (col >> 1)) * 4 + (off & 3)];
          acc[c] = fmaf(e, fmaf((float)((byte >> (4 * (col & 1))) & 15), vs, vm), acc[c] * alpha);
        }
      }
    }
  }
  if (lane == 0) {
    m_s[warp] = m;
    l_s[warp] = l;
  }
#pragma unroll
  for (int c = 0; c < kCols; ++c) o_s[warp][lane + 32 * c] = acc[c];
  __syncthreads();
  float top = -INFINITY, sum = 0.0f;
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, m_s[w]);
  for (int w = 0; w < kWarps; ++w) sum += m_s[w] == -INFINITY ? 0.0f * l_s[w] : l_s[w] * expf(m_s[w] - top);
  T* o = static_cast<T*>(a.out) + (((int64_t)r * a.n + i) * a.heads + h) * a.c.d;
  for (int c = threadIdx.x; c < a.c.d; c += kWarps * 32) {
    float x = 0.0f;
    for (int w = 0; w < kWarps; ++w)
      if (m_s[w] != -INFINITY) x += o_s[w][c] * expf(m_s[w] - top);
    o[c] = from_f32<T>(sum == 0.0f ? 0.0f : x / sum);
  }
}

}  // namespace

int launch_kv4_attend(const Kv4AttendArgs& a, cudaStream_t s) {
  dim3 grid((unsigned)(a.heads * a.n), (unsigned)a.requests);
  if (a.dtype == SA_REP_FLOAT32)
    attend_kernel<SA_REP_FLOAT32><<<grid, kWarps * 32, 0, s>>>(a);
  else if (a.dtype == SA_REP_FLOAT16)
    attend_kernel<SA_REP_FLOAT16><<<grid, kWarps * 32, 0, s>>>(a);
  else
    attend_kernel<SA_REP_BFLOAT16><<<grid, kWarps * 32, 0, s>>>(a);
  return check_launch("kv4 attend_kernel");
}

}  // namespace sa
