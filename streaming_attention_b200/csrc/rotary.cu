// Root-mean-square norm of each head's query or key and its rotation by the
// token's position, in one pass:
//
//   y = x / sqrt(mean(x^2) + eps) * w
//   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin),  angle = position * frequency[i]
//   (a, b) = (i, i + half) or, interleaved, (2 i, 2 i + 1);  columns from 2 half on are not rotated.
//
// float32 throughout, one rounding; the angles are taken in turns and reduced in
// float64, so that far positions lose nothing.  Bound by the rows' bytes.
//
// Rows on 16-byte borders of widths (and halves) that are multiples of 8: a lane
// holds eight columns of a row and the cosines and sines of their angles, which
// serve every head of the token; lanes (1, 2, .. 32 to a row) sum squares and
// trade partners by shuffles, four rows' loads in flight; no shared memory.  A
// warp takes some of a token's heads: all of them where tokens abound.
// Others: one CTA per token, angles in shared memory, element by element.
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

// log2 of the lanes to a row; a warp takes `span` rows (heads of q, then of k) of a token.
template <int DT, int LOG>
__global__ void __launch_bounds__(kRotThreads) rotary_vec_kernel(const RotaryArgs a, int spans, int span) {
  using T = typename Elem<DT>::T;
  constexpr int kLanes = 1 << LOG, kRowsAtOnce = 32 >> LOG, kAhead = 4;
  const int lane = threadIdx.x & 31, li = lane & (kLanes - 1), sub = lane >> LOG;
  const int64_t w = (int64_t)blockIdx.x * (kRotThreads / 32) + (threadIdx.x >> 5);
  const int64_t t = w / spans;
  if (t >= a.tokens) return;
  const int first = (int)(w - t * spans) * span, rows = min(first + span, a.heads + a.kv_heads);
  const int position = a.positions[t];
  if (position < 0 && !a.zero_skipped) return;
  const int c0 = li * 8;
  const bool in = c0 < a.d;              // a row may take fewer lanes than it has
  const bool turned = c0 < 2 * a.half;   // whole lanes are: half is a multiple of 8 (of 4 where interleaved)
  const int shift = a.interleaved ? 0 : a.half >> 3;
  const bool second = !a.interleaved && c0 >= a.half;
  const int partner = turned && !a.interleaved ? (second ? lane - shift : lane + shift) : lane;
  float cs[8], sn[8], wq[8], wk[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cs[e] = 1.0f;
    sn[e] = 0.0f;
    wq[e] = wk[e] = 1.0f;
  }
  auto load = [&](float (&x)[8], int row) {
    if (in && row < rows)
      load8(x, (row < a.heads ? static_cast<const T*>(a.q) + t * a.q_t + row * a.q_h
                              : static_cast<const T*>(a.k) + t * a.k_t + (row - a.heads) * a.k_h) + c0);
    else
      for (int e = 0; e < 8; ++e) x[e] = 0.0f;
  };
  float x[kAhead][8];
  if (position >= 0)
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load(x[i], first + i * kRowsAtOnce + sub);
  if (turned && position >= 0) {
    if (a.interleaved) {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const double turns = (double)position * a.frequencies[(c0 + e) >> 1] * 0.15915494309189533577;
        float s, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
        cs[e] = cs[e + 1] = c;
        sn[e] = -s;
        sn[e + 1] = s;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double turns = (double)position * a.frequencies[c0 + e - (second ? a.half : 0)] * 0.15915494309189533577;
        float s;
        sincospif(2.0f * (float)(turns - rint(turns)), &s, &cs[e]);
        sn[e] = second ? s : -s;
      }
    }
  }
  if (in && a.q_weight) load8(wq, static_cast<const T*>(a.q_weight) + c0);
  if (in && a.k_weight) load8(wk, static_cast<const T*>(a.k_weight) + c0);
  const float inv_d = 1.0f / (float)a.d;
  for (int r0 = first; r0 < rows; r0 += kAhead * kRowsAtOnce) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int row = r0 + i * kRowsAtOnce + sub;
      const bool isq = row < a.heads;
      float y[8];
      if (position >= 0) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(x[i][e], x[i][e], ss);
#pragma unroll
        for (int d = 1; d < kLanes; d *= 2) ss += __shfl_xor_sync(0xffffffffu, ss, d);
        const float r = 1.0f / sqrtf(fmaf(ss, inv_d, a.eps));
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = x[i][e] * r * (isq ? wq[e] : wk[e]);
        load(x[i], row + kAhead * kRowsAtOnce);
        float z[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = a.interleaved ? y[e ^ 1] : __shfl_sync(0xffffffffu, y[e], partner);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = fmaf(y[e], cs[e], z[e] * sn[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = 0.0f;
      }
      if (in && row < rows)
        store8((isq ? static_cast<T*>(a.q_out) + t * a.qo_t + row * a.qo_h
                    : static_cast<T*>(a.k_out) + t * a.ko_t + (row - a.heads) * a.ko_h) + c0, y);
    }
  }
}

template <int DT>
int launch_vec(const RotaryArgs& a, cudaStream_t s) {
  int log = 0;
  while ((8 << log) < a.d) ++log;
  // rows of a token to a warp: all of them, or as few as its lanes hold in flight
  // once while the grid has less than 16 warps an SM
  const int rows = a.heads + a.kv_heads, at_once = 4 * (32 >> log);
  int spans = 1;
  while (a.tokens * spans < 148 * 16 && (rows + spans - 1) / spans > at_once) ++spans;
  int span = (rows + spans - 1) / spans;
  span = (span + (32 >> log) - 1) / (32 >> log) * (32 >> log);   // whole warps of rows
  spans = (rows + span - 1) / span;
  const int64_t ctas = ceil_div(a.tokens * spans, kRotThreads / 32);
  if (ctas > 2147483647LL) return set_error(SA_ERR_UNSUPPORTED, "rotary: grid too large");
  const unsigned g = (unsigned)ctas;
  if (log == 0) rotary_vec_kernel<DT, 0><<<g, kRotThreads, 0, s>>>(a, spans, span);
  else if (log == 1) rotary_vec_kernel<DT, 1><<<g, kRotThreads, 0, s>>>(a, spans, span);
  else if (log == 2) rotary_vec_kernel<DT, 2><<<g, kRotThreads, 0, s>>>(a, spans, span);
  else if (log == 3) rotary_vec_kernel<DT, 3><<<g, kRotThreads, 0, s>>>(a, spans, span);
  else if (log == 4) rotary_vec_kernel<DT, 4><<<g, kRotThreads, 0, s>>>(a, spans, span);
  else rotary_vec_kernel<DT, 5><<<g, kRotThreads, 0, s>>>(a, spans, span);
  return check_launch("rotary_vec_kernel");
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
  const int elem = elem_size(dtype);
  const bool vec = d % 8 == 0 && (interleaved ? half % 4 == 0 : half % 8 == 0) && rows_aligned(q, elem, a.q_t, a.q_h) &&
                   rows_aligned(k, elem, a.k_t, a.k_h) && rows_aligned(q_out, elem, a.qo_t, a.qo_h) &&
                   rows_aligned(k_out, elem, a.ko_t, a.ko_h) && rows_aligned(q_weight, elem, 0, 0) &&
                   rows_aligned(k_weight, elem, 0, 0);
  if (vec) {
    if (dtype == SA_REP_FLOAT32) return launch_vec<SA_REP_FLOAT32>(a, s);
    if (dtype == SA_REP_FLOAT16) return launch_vec<SA_REP_FLOAT16>(a, s);
    return launch_vec<SA_REP_BFLOAT16>(a, s);
  }
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
