// Root-mean-square norm of each head's query or key and its rotation by the
// token's position, in one pass:
//
//   y = x / sqrt(mean(x^2) + eps) * w
//   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin),  angle = position * frequency[i]
//   (a, b) = (i, i + half) or, interleaved, (2 i, 2 i + 1);  columns from 2 half on are not rotated.
//
// One CTA per token: its threads first take the cosines and sines of the
// token's angles (in turns, reduced in float64, so that far positions lose
// nothing), then each warp norms and rotates one head at a time in float32 and
// rounds once.
#include "serving.cuh"

namespace sa {

namespace {

constexpr int kRotThreads = 256;
constexpr int kRotMaxDim = 256;

struct RotaryArgs {
  const void* q;
  const void* k;
  void* q_out;
  void* k_out;
  const int32_t* positions;
  const void* q_weight;
  const void* k_weight;
  const double* frequencies;
  int64_t q_t, q_h, k_t, k_h, qo_t, qo_h, ko_t, ko_h;   // strides in elements
  int64_t tokens;
  int heads, kv_heads, d, half;
  float eps;
  int interleaved, zero_skipped;
};

template <int DT>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotaryArgs a) {
  using T = typename Elem<DT>::T;
  __shared__ float cs[kRotMaxDim / 2], sn[kRotMaxDim / 2];
  __shared__ float row[kRotThreads / 32][kRotMaxDim];
  const int64_t t = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int position = a.positions[t];
  if (position >= 0) {
    for (int i = tid; i < a.half; i += kRotThreads) {
      const double turns = (double)position * a.frequencies[i] * 0.15915494309189533577;
      const float f = (float)(turns - rint(turns));
      sincospif(2.0f * f, &sn[i], &cs[i]);
    }
  }
  __syncthreads();
  for (int h = warp; h < a.heads + a.kv_heads; h += kRotThreads / 32) {
    const bool isq = h < a.heads;
    const T* x = isq ? static_cast<const T*>(a.q) + t * a.q_t + h * a.q_h
                     : static_cast<const T*>(a.k) + t * a.k_t + (h - a.heads) * a.k_h;
    T* o = isq ? static_cast<T*>(a.q_out) + t * a.qo_t + h * a.qo_h
               : static_cast<T*>(a.k_out) + t * a.ko_t + (h - a.heads) * a.ko_h;
    const T* w = static_cast<const T*>(isq ? a.q_weight : a.k_weight);
    if (position < 0) {
      if (a.zero_skipped)
        for (int c = lane; c < a.d; c += 32) o[c] = from_f32<T>(0.0f);
      continue;
    }
    float ss = 0.0f;
    for (int c = lane; c < a.d; c += 32) {
      const float v = to_f32(x[c]);
      row[warp][c] = v;
      ss = fmaf(v, v, ss);
    }
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, s);
    const float r = 1.0f / sqrtf(ss / (float)a.d + a.eps);
    __syncwarp();
    for (int c = lane; c < a.d; c += 32) {
      const float y = row[warp][c] * r * (w ? to_f32(w[c]) : 1.0f);
      float out = y;
      if (c < 2 * a.half) {
        const int i = a.interleaved ? c >> 1 : (c < a.half ? c : c - a.half);
        const bool second = a.interleaved ? (c & 1) : c >= a.half;
        const int pc = a.interleaved ? (c ^ 1) : (second ? c - a.half : c + a.half);
        const float z = row[warp][pc] * r * (w ? to_f32(w[pc]) : 1.0f);
        out = second ? y * cs[i] + z * sn[i] : y * cs[i] - z * sn[i];
      }
      o[c] = from_f32<T>(out);
    }
    __syncwarp();
  }
}

}  // namespace

int launch_rotary(const void* q, const void* k, void* q_out, void* k_out, const int32_t* positions,
                  const void* q_weight, const void* k_weight, const double* frequencies, const int64_t* strides,
                  int64_t tokens, int heads, int kv_heads, int d, int half, float eps, int interleaved,
                  int zero_skipped, int dtype, cudaStream_t s) {
  const RotaryArgs a{q,          k,          q_out,      k_out,      positions,  q_weight, k_weight,
                     frequencies, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5],
                     strides[6], strides[7], tokens,     heads,      kv_heads,   d,        half,
                     eps,        interleaved, zero_skipped};
  if (tokens > 2147483647LL) return set_error(SA_ERR_UNSUPPORTED, "rotary: more than 2^31 - 1 tokens");
  const unsigned g = (unsigned)tokens;
  if (dtype == SA_REP_FLOAT32)
    rotary_kernel<SA_REP_FLOAT32><<<g, kRotThreads, 0, s>>>(a);
  else if (dtype == SA_REP_FLOAT16)
    rotary_kernel<SA_REP_FLOAT16><<<g, kRotThreads, 0, s>>>(a);
  else
    rotary_kernel<SA_REP_BFLOAT16><<<g, kRotThreads, 0, s>>>(a);
  return check_launch("rotary_kernel");
}

}  // namespace sa
