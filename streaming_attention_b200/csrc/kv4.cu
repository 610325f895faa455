// A paged key/value cache held in 4 bits: the quantising write and the read.
//
// Each (token, head) row of keys and of values has its own scale and least
// value, in bfloat16 (float32's range, so no row is too large for it):
//   least = bf16(min x), scale = bf16((max x - min x) / 15),
//   code = clamp(rint((x - least) / scale), 0, 15)   (ties to even),   value = scale * code + least.
// The quotient's rounding is decided exactly: float32 decides where it is far
// from a border between two codes, float64 where it is near.  A row holding
// something that bfloat16 cannot (NaN, an infinity, a least value that rounds
// to one) gets NaN for scale and least value; scale 0 gives code 0.
//
// Layout (page = page_size tokens, a power of two >= 16; dp = the head width
// filled up to 32, 64, 128 or 256; byte b of a row: column 2 b low, 2 b + 1 high):
//   k_codes [pages, heads, page, dp / 2]         a token's row is contiguous
//   v_codes [pages, heads, page / 4, dp / 2, 4]  four tokens' bytes of a column pair share a word: the pairs
//                                                along the token axis that the product P V contracts
//   k_params, v_params [pages, heads, page, 2]   scale, least
#include <math.h>

#include "kv4.cuh"

namespace sa {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 4;   // byte columns per lane: dp <= 256

// The code of x, decided as in exact arithmetic.
__device__ __forceinline__ uint32_t code_of(float x, float least, float scale) {
  if (!(scale > 0.0f)) return 0;
  const float t = __fdiv_rn(x - least, scale);
  const float r = rintf(t);
  // |t - exact| is a few 2^-24 of t: far from k + 1/2 the rounding stands
  if (t > -1.0f && t < 16.0f && fabsf(fabsf(t - r) - 0.5f) < 1e-4f) {
    const double e = rint(((double)x - (double)least) / (double)scale);
    return (uint32_t)fmin(fmax(e, 0.0), 15.0);
  }
  return (uint32_t)fminf(fmaxf(r, 0.0f), 15.0f);
}

// One warp per (token, head, k or v) row.
template <int DT>
__global__ void __launch_bounds__(kThreads) append_kernel(const Kv4AppendArgs a) {
  using T = typename Elem<DT>::T;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int64_t rows = a.tokens * a.c.heads * 2;
  if (row >= rows) return;
  const bool isv = row & 1;
  const int h = (int)((row >> 1) % a.c.heads);
  const int64_t t = (row >> 1) / a.c.heads;
  const int64_t slot = a.slots[t];
  if (slot < 0) return;
  const int64_t page = slot >> a.c.page_shift;
  const int off = (int)(slot & ((1 << a.c.page_shift) - 1));
  if (page >= a.c.pages) {
    if (lane == 0) report(a.status, kBadSlot, t);
    return;
  }
  const T* x = isv ? static_cast<const T*>(a.v) + t * a.v_t + h * a.v_h : static_cast<const T*>(a.k) + t * a.k_t + h * a.k_h;
  float lo = INFINITY, hi = -INFINITY;
  float v[2 * kMaxPairs];
  bool bad = false;
#pragma unroll
  for (int j = 0; j < kMaxPairs; ++j) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int c = 2 * (lane + 32 * j) + e;
      const bool in = c < a.c.d;
      const float y = in ? to_f32(x[c]) : 0.0f;
      v[2 * j + e] = y;
      if (in) {
        bad |= !(fabsf(y) < INFINITY);
        lo = fminf(lo, y);
        hi = fmaxf(hi, y);
      }
    }
  }
#pragma unroll
  for (int s = 16; s >= 1; s >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, s));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, s));
  }
  bad = __any_sync(0xffffffffu, bad);
  __nv_bfloat162 sm;
  sm.x = __float2bfloat16_rn((float)(((double)hi - (double)lo) / 15.0));
  sm.y = __float2bfloat16_rn(lo);
  if (bad || !(fabsf(__bfloat162float(sm.y)) < INFINITY)) sm.x = sm.y = __float2bfloat16_rn(NAN);
  const float scale = __bfloat162float(sm.x), least = __bfloat162float(sm.y);
  const int64_t cell = (page * a.c.heads + h) * ((int64_t)1 << a.c.page_shift);
  const int bytes = a.c.dp >> 1;
#pragma unroll
  for (int j = 0; j < kMaxPairs; ++j) {
    const int b = lane + 32 * j;
    if (b >= bytes) break;
    const uint32_t c0 = 2 * b < a.c.d ? code_of(v[2 * j], least, scale) : 0;
    const uint32_t c1 = 2 * b + 1 < a.c.d ? code_of(v[2 * j + 1], least, scale) : 0;
    const uint8_t byte = (uint8_t)(c0 | (c1 << 4));
    if (isv)
      a.c.v_codes[cell * bytes + ((int64_t)(off >> 2) * bytes + b) * 4 + (off & 3)] = byte;
    else
      a.c.k_codes[(cell + off) * bytes + b] = byte;
  }
  if (lane == 0) *reinterpret_cast<__nv_bfloat162*>((isv ? a.c.v_params : a.c.k_params) + 2 * (cell + off)) = sm;
}

template <int DT>
__global__ void __launch_bounds__(kThreads) read_kernel(const Kv4ReadArgs a) {
  using T = typename Elem<DT>::T;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int64_t rows = a.tokens * a.c.heads * 2;
  if (row >= rows) return;
  const bool isv = row & 1;
  const int h = (int)((row >> 1) % a.c.heads);
  const int64_t t = (row >> 1) / a.c.heads;
  const int64_t slot = a.slots[t];
  T* o = static_cast<T*>(isv ? a.v : a.k) + (t * a.c.heads + h) * a.c.d;
  const int64_t page = slot >> a.c.page_shift;
  const int off = (int)(slot & ((1 << a.c.page_shift) - 1));
  const bool in = slot >= 0 && page < a.c.pages;
  if (!in && slot >= 0 && lane == 0) report(a.status, kBadSlot, t);
  const int64_t cell = ((in ? page : 0) * a.c.heads + h) * ((int64_t)1 << a.c.page_shift);
  const int bytes = a.c.dp >> 1;
  float scale = 0.0f, least = 0.0f;
  if (in) {
    const __nv_bfloat16* p = (isv ? a.c.v_params : a.c.k_params) + 2 * (cell + off);
    scale = __bfloat162float(p[0]);
    least = __bfloat162float(p[1]);
  }
  for (int b = lane; 2 * b < a.c.d; b += 32) {
    uint32_t byte = 0;
    if (in)
      byte = isv ? a.c.v_codes[cell * bytes + ((int64_t)(off >> 2) * bytes + b) * 4 + (off & 3)]
                 : a.c.k_codes[(cell + off) * bytes + b];
    o[2 * b] = from_f32<T>(fmaf((float)(byte & 15), scale, least));
    if (2 * b + 1 < a.c.d) o[2 * b + 1] = from_f32<T>(fmaf((float)(byte >> 4), scale, least));
  }
}

}  // namespace

int launch_kv4_append(const Kv4AppendArgs& a, int dtype, cudaStream_t s) {
  const int64_t ctas = ceil_div(a.tokens * a.c.heads * 2, kThreads / 32);
  if (ctas > 2147483647LL) return set_error(SA_ERR_UNSUPPORTED, "kv4 append: too many rows");
  if (dtype == SA_REP_FLOAT32)
    append_kernel<SA_REP_FLOAT32><<<(unsigned)ctas, kThreads, 0, s>>>(a);
  else if (dtype == SA_REP_FLOAT16)
    append_kernel<SA_REP_FLOAT16><<<(unsigned)ctas, kThreads, 0, s>>>(a);
  else
    append_kernel<SA_REP_BFLOAT16><<<(unsigned)ctas, kThreads, 0, s>>>(a);
  return check_launch("kv4 append_kernel");
}

int launch_kv4_read(const Kv4ReadArgs& a, int dtype, cudaStream_t s) {
  const int64_t ctas = ceil_div(a.tokens * a.c.heads * 2, kThreads / 32);
  if (ctas > 2147483647LL) return set_error(SA_ERR_UNSUPPORTED, "kv4 read: too many rows");
  if (dtype == SA_REP_FLOAT32)
    read_kernel<SA_REP_FLOAT32><<<(unsigned)ctas, kThreads, 0, s>>>(a);
  else if (dtype == SA_REP_FLOAT16)
    read_kernel<SA_REP_FLOAT16><<<(unsigned)ctas, kThreads, 0, s>>>(a);
  else
    read_kernel<SA_REP_BFLOAT16><<<(unsigned)ctas, kThreads, 0, s>>>(a);
  return check_launch("kv4 read_kernel");
}

}  // namespace sa
