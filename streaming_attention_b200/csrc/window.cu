// Attention with a sliding window and first tokens that stay visible, on the
// CUDA cores (fp32 FMA): the shapes and types the tensor-core kernel does not
// take, and the SA_FORCE_SIMT comparison path.
//
//   out_i = sum_j softmax_j(scale q_i.k_j) v_j over the visible keys
//   j <= p_i and (j > p_i - window or j < sinks),  p_i = m - n + i;
//   a row that sees nothing is zero.
//
// One CTA per (64-query tile, query head), 256 threads: four threads per query
// row, each scoring 8 of a 32-key tile and accumulating a quarter of the value
// columns (float32 throughout, online softmax).  Only tiles that hold a visible
// key are read: the first tokens' tiles, then the window's.  Bound by the FMA pipe
// and its shared-memory operands: 2 x 8 heads x 4096 of 64 with a window of 512
// 1159 us, where the tensor cores' form takes 137.
#include <math.h>

#include "serving.cuh"

namespace sa {

namespace {

constexpr int kWQ = 64;
constexpr int kWK = 32;
constexpr int kWThreads = 256;

__device__ __forceinline__ float load_elem(const void* p, int64_t at, int dtype) {
  if (dtype == SA_REP_FLOAT32) return __ldg(static_cast<const float*>(p) + at);
  if (dtype == SA_REP_FLOAT16) return __half2float(static_cast<const __half*>(p)[at]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
}

__device__ __forceinline__ void store_elem(void* p, int64_t at, int dtype, float x) {
  if (dtype == SA_REP_FLOAT32)
    static_cast<float*>(p)[at] = x;
  else if (dtype == SA_REP_FLOAT16)
    static_cast<__half*>(p)[at] = __float2half_rn(x);
  else
    static_cast<__nv_bfloat16*>(p)[at] = __float2bfloat16_rn(x);
}

template <int DP, int DVP>
__global__ void __launch_bounds__(kWThreads) window_simt_kernel(const WindowArgs a) {
  constexpr int CPT = DVP / 4;
  extern __shared__ float4 window_smem4[];
  auto Kt = reinterpret_cast<float(*)[kWK + 4]>(window_smem4);
  auto Vs = reinterpret_cast<float(*)[DVP]>(&Kt[DP][0]);
  auto Qs = reinterpret_cast<float(*)[DP + 1]>(&Vs[kWK][0]);
  auto E = reinterpret_cast<float(*)[kWK + 1]>(&Qs[kWQ][0]);

  const int tid = threadIdx.x;
  const int qi = tid >> 2, cg = tid & 3;
  if (a.dtype == SA_REP_FLOAT32)
    zero_unwritten_rows<float>(a, kWQ, tid, kWThreads, nullptr);
  else
    zero_unwritten_rows<uint16_t>(a, kWQ, tid, kWThreads, nullptr);   // zero has the same bits in both 16-bit types
  const int h = blockIdx.y, hk = h / (a.heads / a.kv_heads);
  int64_t tile;
  const int b = tile_request(a, blockIdx.x, kWQ, &tile);
  const Request rq = request_of(a, b);
  const int64_t i0 = tile * kWQ;
  if (tile < 0 || i0 >= rq.n) return;
  const int nq = (int)min((int64_t)kWQ, rq.n - i0);
  const int64_t p0 = rq.m - rq.n + i0;      // position of the tile's first query
  const int64_t p = p0 + qi;
  const bool valid = qi < nq;
  const KeyRanges kr = key_ranges(p0, p0 + nq - 1, rq.m, a.window, a.sinks);

  const int64_t qoff = b * a.q_b + h * a.q_h + (rq.q0 + i0) * a.q_n;
  for (int e = tid; e < kWQ * DP; e += kWThreads) {
    const int r = e / DP, c = e - r * DP;
    Qs[r][c] = (r < nq && c < a.d) ? load_elem(a.q, qoff + r * a.q_n + c, a.dtype) * a.scale : 0.0f;
  }
  float acc[CPT];
#pragma unroll
  for (int c = 0; c < CPT; ++c) acc[c] = 0.0f;
  float m = -INFINITY, l = 0.0f;

  const int64_t koff = b * a.k_b + hk * a.k_h + rq.k0 * a.k_n;
  const int64_t voff = b * a.v_b + hk * a.v_h + rq.k0 * a.v_n;
  for (int part = 0; part < 2; ++part) {
    const int64_t jb = part ? kr.begin : 0, je = part ? kr.end : kr.first;
    for (int64_t j0 = jb; j0 < je; j0 += kWK) {
      const int tk = (int)min((int64_t)kWK, je - j0);
      __syncthreads();
      for (int e = tid; e < kWK * DP; e += kWThreads) {
        const int r = e / DP, c = e - r * DP;
        Kt[c][r] = (r < tk && c < a.d) ? load_elem(a.k, koff + (j0 + r) * a.k_n + c, a.dtype) : 0.0f;
      }
      for (int e = tid; e < kWK * DVP; e += kWThreads) {
        const int r = e / DVP, c = e - r * DVP;
        Vs[r][c] = (r < tk && c < a.dv) ? load_elem(a.v, voff + (j0 + r) * a.v_n + c, a.dtype) : 0.0f;
      }
      __syncthreads();
      float x[8];
#pragma unroll
      for (int rr = 0; rr < 8; ++rr) x[rr] = 0.0f;
      for (int c = 0; c < a.d; ++c) {
        const float qa = Qs[qi][c];
        const float4 k0 = *reinterpret_cast<const float4*>(&Kt[c][cg * 8]);
        const float4 k1 = *reinterpret_cast<const float4*>(&Kt[c][cg * 8 + 4]);
        x[0] = fmaf(qa, k0.x, x[0]);
        x[1] = fmaf(qa, k0.y, x[1]);
        x[2] = fmaf(qa, k0.z, x[2]);
        x[3] = fmaf(qa, k0.w, x[3]);
        x[4] = fmaf(qa, k1.x, x[4]);
        x[5] = fmaf(qa, k1.y, x[5]);
        x[6] = fmaf(qa, k1.z, x[6]);
        x[7] = fmaf(qa, k1.w, x[7]);
      }
      bool on[8];
      float pm = -INFINITY;
#pragma unroll
      for (int rr = 0; rr < 8; ++rr) {
        const int64_t j = j0 + cg * 8 + rr;
        on[rr] = valid && j < je && j <= p && (j > p - a.window || j < a.sinks);
        if (on[rr]) pm = fmaxf(pm, x[rr]);
      }
      pm = fmaxf(pm, __shfl_xor_sync(0xffffffffu, pm, 1));
      pm = fmaxf(pm, __shfl_xor_sync(0xffffffffu, pm, 2));
      const float m_new = fmaxf(m, pm);
      // m_new = -inf: nothing visible yet, everything stays 0
      const float alpha = (m_new == -INFINITY) ? 1.0f : expf(m - m_new);
      // weights are at most 2^-24, so that 2^24 of them times values near
      // float32's largest still sum below it
      const float m_off = m_new + 16.635532f;
      float es = 0.0f;
#pragma unroll
      for (int rr = 0; rr < 8; ++rr) {
        const float e = on[rr] && x[rr] != -INFINITY ? expf(x[rr] - m_off) : 0.0f;   // NaN before any maximum stays NaN
        E[qi][cg * 8 + rr] = e;
        es += e;
      }
      es += __shfl_xor_sync(0xffffffffu, es, 1);
      es += __shfl_xor_sync(0xffffffffu, es, 2);
      m = m_new;
      l = l * alpha + es;
#pragma unroll
      for (int c = 0; c < CPT; ++c) acc[c] *= alpha;
      __syncwarp();   // a row's four threads share a warp
      for (int r = 0; r < tk; ++r) {
        const float e = E[qi][r];
        if (e == 0.0f) continue;   // a hidden key's value is not looked at, whatever it holds
        const float4* vrow = reinterpret_cast<const float4*>(&Vs[r][cg * CPT]);
#pragma unroll
        for (int c4 = 0; c4 < CPT / 4; ++c4) {
          const float4 vv = vrow[c4];
          acc[4 * c4 + 0] = fmaf(e, vv.x, acc[4 * c4 + 0]);
          acc[4 * c4 + 1] = fmaf(e, vv.y, acc[4 * c4 + 1]);
          acc[4 * c4 + 2] = fmaf(e, vv.z, acc[4 * c4 + 2]);
          acc[4 * c4 + 3] = fmaf(e, vv.w, acc[4 * c4 + 3]);
        }
      }
    }
  }
  if (valid) {
    const int64_t o = b * a.o_b + h * a.o_h + (rq.q0 + i0 + qi) * a.o_n;
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      const int col = cg * CPT + c;
      if (col < a.dv) store_elem(a.out, o + col, a.dtype, l == 0.0f ? 0.0f : __fdiv_rn(acc[c], l));
    }
  }
}

template <int DP, int DVP>
int launch_dims(const WindowArgs& a, cudaStream_t s) {
  const size_t smem = sizeof(float) * ((size_t)DP * (kWK + 4) + (size_t)kWK * DVP + (size_t)kWQ * (DP + 1) +
                                       (size_t)kWQ * (kWK + 1));
  cudaError_t e =
      cudaFuncSetAttribute(window_simt_kernel<DP, DVP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return set_error(SA_ERR_CUDA, "window_simt smem attribute: %s", cudaGetErrorString(e));
  const int64_t tiles = tile_count(a, kWQ);
  if (tiles > 2147483647LL || a.heads > 65535) return set_error(SA_ERR_UNSUPPORTED, "window attention: grid too large");
  dim3 grid((unsigned)tiles, (unsigned)a.heads);
  window_simt_kernel<DP, DVP><<<grid, kWThreads, smem, s>>>(a);
  return check_launch("window_simt_kernel");
}

template <int DP>
int launch_dp(const WindowArgs& a, cudaStream_t s) {
  if (a.dv <= 64) return launch_dims<DP, 64>(a, s);
  if (a.dv <= 128) return launch_dims<DP, 128>(a, s);
  return launch_dims<DP, 256>(a, s);
}

}  // namespace

int launch_window_simt(const WindowArgs& a, cudaStream_t s) {
  if (a.d <= 64) return launch_dp<64>(a, s);
  if (a.d <= 128) return launch_dp<128>(a, s);
  return launch_dp<256>(a, s);
}

}  // namespace sa
