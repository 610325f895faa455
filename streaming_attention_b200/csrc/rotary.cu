// Root-mean-square norm of each head's query or key and its rotation by the
// token's position, in one pass:
//
//   y = x / sqrt(mean(x^2) + eps) * w
//   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin),  angle = position * frequency[i]
//   (a, b) = (i, i + half) or, interleaved, (2 i, 2 i + 1);  columns from 2 half on are not rotated.
//
// float32 throughout, one rounding; the angles are taken in turns and reduced in
// float64, so that far positions lose nothing.  Bound by the rows' bytes: 16384
// tokens of 32 + 8 heads of 128 in bfloat16 (336 MB, 52 us) take 76 us.
//
// Rows on 16-byte borders of widths (and halves) that are multiples of 8: a lane
// holds eight columns of a row and, for every head of the token, what they are
// multiplied with: out_a = r (x_a (w_a cos) - x_b (w_b sin)).  Lanes (1, 2, .. 32 to
// a row) sum squares and trade the rows' bits by shuffles, two rows' loads in
// flight (and a third CTA an SM for it); no shared memory.  A warp takes some of a token's heads: all of them
// where tokens abound.
// Others: one CTA per token, angles in shared memory, element by element.
#include <type_traits>

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

// Eight elements' bits.
template <typename T>
struct Bits {
  static constexpr int kWords = sizeof(T) * 2;
  uint32_t w[kWords];
};

template <typename T>
__device__ __forceinline__ void floats(float (&x)[8], const Bits<T>& b) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if constexpr (sizeof(T) == 4) {
      x[e] = __uint_as_float(b.w[e]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      x[e] = __uint_as_float(e & 1 ? b.w[e >> 1] & 0xffff0000u : b.w[e >> 1] << 16);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&b.w[e >> 1]));
      x[e] = e & 1 ? f.y : f.x;
    }
  }
}

// log2 of the lanes to a row; a warp takes `span` rows (heads of q, then of k) of a token.
template <int DT, int LOG>
__global__ void __launch_bounds__(kRotThreads, DT == SA_REP_FLOAT32 ? 2 : 3) rotary_vec_kernel(const RotaryArgs a, int spans, int span) {
  using T = typename Elem<DT>::T;
  constexpr int kLanes = 1 << LOG, kRowsAtOnce = 32 >> LOG, kAhead = 2;
  const int lane = threadIdx.x & 31, li = lane & (kLanes - 1), sub = lane >> LOG;
  const uint32_t w = blockIdx.x * (kRotThreads / 32) + (threadIdx.x >> 5);
  const uint32_t t32 = w / (uint32_t)spans;
  const int64_t t = t32;
  if (t >= a.tokens) return;
  const int first = (int)(w - t32 * spans) * span, rows = min(first + span, a.heads + a.kv_heads);
  const int position = a.positions[t];
  const int c0 = li * 8;
  const bool in = c0 < a.d;              // a row may take fewer lanes than it has
  if (position < 0) {
    if (a.zero_skipped && in) {
      const float none[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
      for (int row = first + sub; row < rows; row += kRowsAtOnce)
        store8((row < a.heads ? static_cast<T*>(a.q_out) + t * a.qo_t + row * a.qo_h
                              : static_cast<T*>(a.k_out) + t * a.ko_t + (row - a.heads) * a.ko_h) + c0, none);
    }
    return;
  }
  const bool turned = c0 < 2 * a.half;   // whole lanes are: half is a multiple of 8 (of 4 where interleaved)
  const int shift = a.half >> 3;
  const bool second = c0 >= a.half;
  const int partner = turned && !a.interleaved ? (second ? lane - shift : lane + shift) : lane;
  float cs[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cs[e] = 1.0f;
    sn[e] = 0.0f;
  }
  if (turned) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = a.interleaved ? (c0 + e) >> 1 : c0 + e - (second ? a.half : 0);
      const double turns = (double)position * a.frequencies[i] * 0.15915494309189533577;
      float s;
      sincospif(2.0f * (float)(turns - rint(turns)), &s, &cs[e]);
      sn[e] = (a.interleaved ? (e & 1) != 0 : second) ? s : -s;
    }
  }
  const float inv_d = 1.0f / (float)a.d;
#pragma unroll 1
  for (int part = 0; part < 2; ++part) {   // queries, then keys
    const int lo = part ? max(first, a.heads) - a.heads : first, hi = part ? rows - a.heads : min(rows, a.heads);
    if (lo >= hi) continue;
    const T* from = (part ? static_cast<const T*>(a.k) + t * a.k_t : static_cast<const T*>(a.q) + t * a.q_t) + c0;
    T* to = (part ? static_cast<T*>(a.k_out) + t * a.ko_t : static_cast<T*>(a.q_out) + t * a.qo_t) + c0;
    const int64_t from_h = part ? a.k_h : a.q_h, to_h = part ? a.ko_h : a.qo_h;
    auto load = [&](Bits<T>& x, int row) {
#pragma unroll
      for (int i = 0; i < Bits<T>::kWords; i += 4) {
        uint4 y = make_uint4(0, 0, 0, 0);
        if (in && row < hi) y = *(reinterpret_cast<const uint4*>(from + row * from_h) + i / 4);
        x.w[i] = y.x;
        x.w[i + 1] = y.y;
        x.w[i + 2] = y.z;
        x.w[i + 3] = y.w;
      }
    };
    Bits<T> x[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load(x[i], lo + i * kRowsAtOnce + sub);
    // own[e] = w_e cos, other[e] = w_partner (-+ sin)
    float own[8], other[8];
    const T* weight = static_cast<const T*>(part ? a.k_weight : a.q_weight);
#pragma unroll
    for (int e = 0; e < 8; ++e) own[e] = 1.0f;
    if (weight && in) load8(own, weight + c0);
#pragma unroll
    for (int e = 0; e < 8; ++e) other[e] = a.interleaved ? own[e ^ 1] : __shfl_sync(0xffffffffu, own[e], partner);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      own[e] *= cs[e];
      other[e] *= sn[e];
    }
#pragma unroll 1
    for (int r0 = lo; r0 < hi; r0 += kAhead * kRowsAtOnce) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int row = r0 + i * kRowsAtOnce + sub;
        float y[8], z[8];
        floats(y, x[i]);
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(y[e], y[e], ss);
#pragma unroll
        for (int d = 1; d < kLanes; d *= 2) ss += __shfl_xor_sync(0xffffffffu, ss, d);
        if (a.interleaved) {
#pragma unroll
          for (int e = 0; e < 8; ++e) z[e] = y[e ^ 1];
        } else {
          Bits<T> b;
#pragma unroll
          for (int e = 0; e < Bits<T>::kWords; ++e) b.w[e] = __shfl_sync(0xffffffffu, x[i].w[e], partner);
          floats(z, b);
        }
        load(x[i], row + kAhead * kRowsAtOnce);
        const float r = rsqrtf(fmaf(ss, inv_d, a.eps));
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = r * fmaf(y[e], own[e], z[e] * other[e]);
        if (in && row < hi) store8(to + row * to_h, y);
      }
    }
  }
}

template <int DT>
int launch_vec(const RotaryArgs& a, cudaStream_t s) {
  int log = 0;
  while ((8 << log) < a.d) ++log;
  // rows of a token to a warp: all of them, or as few as its lanes hold in flight
  // once while the grid has less than 16 warps an SM
  const int rows = a.heads + a.kv_heads, at_once = 2 * (32 >> log);
  int spans = 1;
  while (a.tokens * spans < 148 * 16 && (rows + spans - 1) / spans > at_once) ++spans;
  int span = (rows + spans - 1) / spans;
  span = (span + (32 >> log) - 1) / (32 >> log) * (32 >> log);   // whole warps of rows
  spans = (rows + span - 1) / span;
  const int64_t ctas = ceil_div(a.tokens * spans, kRotThreads / 32);
  if (ctas > (1 << 28)) return set_error(SA_ERR_UNSUPPORTED, "rotary: grid too large");
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
