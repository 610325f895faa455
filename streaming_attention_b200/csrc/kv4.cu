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
// 20011 tokens of 8 heads of 128 (bfloat16): the write 68 us (104 MB; bound by the
// instructions that find the codes, 72 % of the issue slots), the read of the same
// to float32 48 us (186 MB, 3.9 TB/s).
#include <math.h>

#include "kv4.cuh"

namespace sa {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 4;   // byte columns per lane: dp <= 256

// The code of x, decided as in exact arithmetic.
__device__ __forceinline__ uint32_t code_of(float x, float least, float scale) {
  if (!(scale > 0.0f)) return 0;
  const float d = x - least;
  const float t = __fdiv_rn(d, scale);
  const float r = rintf(t);
  // |t - exact| is a few 2^-24 of t: far from k + 1/2 the rounding stands, where
  // the difference did not overflow
  if ((t > -1.0f && t < 16.0f && fabsf(fabsf(t - r) - 0.5f) < 1e-4f) || !(fabsf(d) < INFINITY)) {
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

// The codes of eight values, a nibble each.  The quotient, as a product with the
// reciprocal clamped by saturation, is less than 3e-6 off.  Where one of the eight
// lies within 1e-5 of a border b = k + 1/2 (often: ties are common among bfloat16
// values) the sign of x - least - b scale decides, which float32 gives exactly:
// b scale has 13 bits, the difference x - least is kept with its rounding error,
// and near the border the subtraction is exact.  Whole numbers stay floats until
// four of them make 16 bits, so that nearly all of it runs on the FMA pipe.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float least, float scale) {
  const float inv = scale > 0.0f ? 1.0f / (15.0f * scale) : 0.0f;   // 0 or infinite where 15 scale over- or underflows
  constexpr float kWhole = 12582912.0f;   // 1.5 2^23: sums with it round to whole numbers
  bool near = false;
  float c[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float u = __saturatef((x[e] - least) * inv);
    c[e] = fmaf(u, 15.0f, kWhole) - kWhole;
    near |= fabsf(fmaf(u, 15.0f, -c[e])) > 0.49999f;
  }
  if (scale > 0.0f && !(inv > 0.0f && inv < INFINITY)) {
    uint32_t w = 0;
#pragma unroll 1
    for (int e = 0; e < 8; ++e) {
      float y = x[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) y = e == i ? x[i] : y;   // keeps x in registers
      w |= code_of(y, least, scale) << (4 * e);
    }
    return w;
  }
  if (near) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = x[e] - least, t = d - x[e];
      const float lost = (x[e] - (d - t)) - (least + t);   // x - least = d + lost, exactly
      const float b = c[e] + copysignf(0.5f, fmaf(__saturatef(d * inv), 15.0f, -c[e]));
      const float side = fmaf(-b, scale, d) + lost;
      const float even = 2.0f * (fmaf(b, 0.5f, kWhole) - kWhole);   // the even one of b - 1/2, b + 1/2: b / 2 is 1/4 from it
      c[e] = fminf(fmaxf(side == 0.0f ? even : b + copysignf(0.5f, side), 0.0f), 15.0f);
    }
  }
  const float lo = fmaf(c[3], 4096.0f, fmaf(c[2], 256.0f, fmaf(c[1], 16.0f, c[0]))) + kWhole;
  const float hi = fmaf(c[7], 4096.0f, fmaf(c[6], 256.0f, fmaf(c[5], 16.0f, c[4]))) + kWhole;
  return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x5410);
}

// Rows on 16-byte borders of widths that are multiples of 8: a lane holds eight
// columns (four bytes of codes), 1 << LOG lanes a row, and takes four neighbouring
// tokens t0 .. t0 + 3 of one head.  Keys: each row's bytes are contiguous.
// Values: where four tokens fill a word group of the cache (slots 4 m .. 4 m + 3),
// the lane that finds the first of them among its own transposes their bytes
// and stores 16 at once; its neighbours leave those tokens to it.  Other tokens
// store single bytes.
template <int DT, int LOG>
__global__ void __launch_bounds__(kThreads) append_vec_kernel(const Kv4AppendArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int kLanes = 1 << LOG;
  const int lane = threadIdx.x & 31, li = lane & (kLanes - 1);
  uint32_t item = (uint32_t)(((int64_t)blockIdx.x * kThreads + threadIdx.x) >> LOG);   // (k or v, quad of tokens, head)
  const uint32_t items = (uint32_t)((a.tokens + 3) >> 2) * a.c.heads;
  const bool isv = item >= items;
  if (isv) item -= items;
  const uint32_t quad = item / (uint32_t)a.c.heads;
  const int h = (int)(item - quad * a.c.heads);
  const int64_t t0 = item < items ? (int64_t)quad * 4 : a.tokens;
  const int c0 = li * 8, bytes = a.c.dp >> 1, page_mask = (1 << a.c.page_shift) - 1;
  const bool in = c0 < a.c.d;
  auto slot_of = [&](int64_t t) -> int { return t >= 0 && t < a.tokens ? __ldg(a.slots + t) : -1; };
  int64_t from = t0;     // the group this lane stores whole: tokens from .. from + 3
  bool whole = false;
  int taken = 0;         // bit i: token t0 + i belongs to a group
  if (isv) {
    // bit j: token t0 - 3 + j is followed by the next slot; opens a word group of the cache
    uint32_t next = 0, first = 0;
    int s0 = slot_of(t0 - 3);
#pragma unroll
    for (int j = 0; j < 9; ++j) {
      const int s1 = slot_of(t0 - 2 + j);
      if (s0 >= 0 && s1 == s0 + 1) next |= 1u << j;
      if (s0 >= 0 && (s0 & 3) == 0 && (s0 >> a.c.page_shift) < a.c.pages) first |= 1u << j;
      s0 = s1;
    }
    const uint32_t opens = first & next & (next >> 1) & (next >> 2) & 127u;   // j: tokens t0 - 3 + j .. t0 + j
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if ((opens >> j) & 1u) taken |= j < 3 ? 15 >> (3 - j) : 15 << (j - 3);
    whole = (opens >> 3) != 0;
    from = t0 + __ffs(opens >> 3) - (whole ? 1 : 0);
    taken &= 15;
  }
  // codes of token t, as four bytes, and its params
  auto code_row = [&](int64_t t, __nv_bfloat162& sm) -> uint32_t {
    float x[8];
    const bool here = in && t < a.tokens;
    if (here)
      load8(x, (isv ? static_cast<const T*>(a.v) + t * a.v_t + h * a.v_h : static_cast<const T*>(a.k) + t * a.k_t + h * a.k_h) + c0);
    float lo = INFINITY, hi = -INFINITY, odd = 0.0f;
    if (here)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        odd = fmaf(x[e], 0.0f, odd);   // NaN once a value is not finite
        lo = fminf(lo, x[e]);
        hi = fmaxf(hi, x[e]);
      }
    if (odd != 0.0f) lo = -INFINITY, hi = INFINITY;   // spreads to the row
#pragma unroll
    for (int d = 1; d < kLanes; d *= 2) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
    }
    sm.x = __float2bfloat16_rn((float)(((double)hi - (double)lo) / 15.0));
    sm.y = __float2bfloat16_rn(lo);
    if (!(fabsf(__bfloat162float(sm.y)) < INFINITY)) sm.x = sm.y = __float2bfloat16_rn(NAN);
    const float scale = __bfloat162float(sm.x), least = __bfloat162float(sm.y);
    return here ? codes_of(x, least, scale) : 0u;
  };
  // single tokens (every key; values outside whole groups)
  const bool singles = __any_sync(0xffffffffu, taken != 15);
#pragma unroll 1
  for (int i = 0; singles && i < 4; ++i) {
    const int64_t t = t0 + i;
    const int slot = slot_of(t);
    bool put = slot >= 0 && !((taken >> i) & 1);
    if (put && (slot >> a.c.page_shift) >= a.c.pages) {
      if (li == 0) report(a.status, kBadSlot, t);
      put = false;
    }
    if (!__any_sync(0xffffffffu, put)) continue;
    __nv_bfloat162 sm;
    const uint32_t w = code_row(t, sm);
    if (!put) continue;
    const int64_t cell = (((int64_t)(slot >> a.c.page_shift) * a.c.heads + h) << a.c.page_shift);
    const int off = slot & page_mask;
    if (li == 0) *reinterpret_cast<__nv_bfloat162*>((isv ? a.c.v_params : a.c.k_params) + 2 * (cell + off)) = sm;
    if (c0 >= a.c.dp) continue;
    if (!isv) {
      *reinterpret_cast<uint32_t*>(a.c.k_codes + (cell + off) * bytes + li * 4) = w;
    } else {
      uint8_t* to = a.c.v_codes + cell * bytes + ((int64_t)(off >> 2) * bytes + li * 4) * 4 + (off & 3);
#pragma unroll
      for (int e = 0; e < 4; ++e) to[4 * e] = (uint8_t)(w >> (8 * e));
    }
  }
  if (__any_sync(0xffffffffu, whole)) {
    uint32_t w[4], sm[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __nv_bfloat162 x;
      w[i] = code_row(from + i, x);
      sm[i] = *reinterpret_cast<const uint32_t*>(&x);
    }
    if (whole) {
      const int slot = slot_of(from);
      const int64_t cell = (((int64_t)(slot >> a.c.page_shift) * a.c.heads + h) << a.c.page_shift) + (slot & page_mask);
      if (li == 0) *reinterpret_cast<uint4*>(a.c.v_params + 2 * cell) = make_uint4(sm[0], sm[1], sm[2], sm[3]);
      // byte e of the four words side by side
      const uint32_t l0 = __byte_perm(w[0], w[1], 0x5140), h0 = __byte_perm(w[2], w[3], 0x5140);
      const uint32_t l1 = __byte_perm(w[0], w[1], 0x7362), h1 = __byte_perm(w[2], w[3], 0x7362);
      if (c0 < a.c.dp)
        *reinterpret_cast<uint4*>(a.c.v_codes + cell * bytes + li * 16) =
            make_uint4(__byte_perm(l0, h0, 0x5410), __byte_perm(l0, h0, 0x7632), __byte_perm(l1, h1, 0x5410),
                       __byte_perm(l1, h1, 0x7632));
    }
  }
}

// 1 << LOG lanes a row, eight columns a lane.
template <int DT, int LOG>
__global__ void __launch_bounds__(kThreads) read_vec_kernel(const Kv4ReadArgs a) {
  using T = typename Elem<DT>::T;
  const int lane = threadIdx.x & 31, li = lane & ((1 << LOG) - 1);
  const uint32_t row = (uint32_t)(((int64_t)blockIdx.x * kThreads + threadIdx.x) >> LOG);
  const uint32_t each = (uint32_t)a.tokens * a.c.heads;
  if (row >= 2 * each || li * 8 >= a.c.d) return;
  // k's rows, then v's: neighbouring groups write neighbouring rows
  const bool isv = row >= each;
  const uint32_t u = isv ? row - each : row;
  const uint32_t t = u / (uint32_t)a.c.heads;
  const int h = (int)(u - t * a.c.heads);
  const int slot = __ldg(a.slots + t);
  T* o = static_cast<T*>(isv ? a.v : a.k) + (int64_t)u * a.c.d + li * 8;
  const int bytes = a.c.dp >> 1;
  float x[8];
  if (slot < 0 || (slot >> a.c.page_shift) >= a.c.pages) {
    if (slot >= 0 && li == 0) report(a.status, kBadSlot, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.0f;
  } else {
    const int off = slot & ((1 << a.c.page_shift) - 1);
    const int64_t cell = (((int64_t)(slot >> a.c.page_shift) * a.c.heads + h) << a.c.page_shift);
    const uint32_t p = *reinterpret_cast<const uint32_t*>((isv ? a.c.v_params : a.c.k_params) + 2 * (cell + off));
    const float scale = __uint_as_float(p << 16), least = __uint_as_float(p & 0xffff0000u);
    uint32_t w;
    if (!isv) {
      w = *reinterpret_cast<const uint32_t*>(a.c.k_codes + (cell + off) * bytes + li * 4);
    } else {
      // four columns' words of four tokens: this token's byte of each
      const uint4 y = *reinterpret_cast<const uint4*>(a.c.v_codes + cell * bytes + ((int64_t)(off >> 2) * bytes + li * 4) * 4);
      const int sel = (off & 3) | (((off & 3) + 4) << 4);
      w = __byte_perm(__byte_perm(y.x, y.y, sel), __byte_perm(y.z, y.w, sel), 0x5410);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf((float)((w >> (4 * e)) & 15u), scale, least);
  }
  store8(o, x);
}

// log2 of the lanes that hold a row of dp columns, eight each.
int row_lanes_log(int dp) { return dp == 32 ? 2 : (dp == 64 ? 3 : (dp == 128 ? 4 : 5)); }

template <int DT>
int append_vec(const Kv4AppendArgs& a, cudaStream_t s) {
  const int log = row_lanes_log(a.c.dp);
  const int64_t ctas = ceil_div((((a.tokens + 3) >> 2) * a.c.heads * 2) << log, kThreads);
  if (ctas > 2147483647LL) return set_error(SA_ERR_UNSUPPORTED, "kv4 append: too many rows");
  const unsigned g = (unsigned)ctas;
  if (log == 2) append_vec_kernel<DT, 2><<<g, kThreads, 0, s>>>(a);
  else if (log == 3) append_vec_kernel<DT, 3><<<g, kThreads, 0, s>>>(a);
  else if (log == 4) append_vec_kernel<DT, 4><<<g, kThreads, 0, s>>>(a);
  else append_vec_kernel<DT, 5><<<g, kThreads, 0, s>>>(a);
  return check_launch("kv4 append_vec_kernel");
}

template <int DT>
int read_vec(const Kv4ReadArgs& a, cudaStream_t s) {
  const int log = row_lanes_log(a.c.dp);
  const int64_t ctas = ceil_div((a.tokens * a.c.heads * 2) << log, kThreads);
  if (ctas > 2147483647LL) return set_error(SA_ERR_UNSUPPORTED, "kv4 read: too many rows");
  const unsigned g = (unsigned)ctas;
  if (log == 2) read_vec_kernel<DT, 2><<<g, kThreads, 0, s>>>(a);
  else if (log == 3) read_vec_kernel<DT, 3><<<g, kThreads, 0, s>>>(a);
  else if (log == 4) read_vec_kernel<DT, 4><<<g, kThreads, 0, s>>>(a);
  else read_vec_kernel<DT, 5><<<g, kThreads, 0, s>>>(a);
  return check_launch("kv4 read_vec_kernel");
}

}  // namespace

int launch_kv4_append(const Kv4AppendArgs& a, int dtype, cudaStream_t s) {
  const int elem = elem_size(dtype);
  if (a.c.d % 8 == 0 && a.tokens * a.c.heads < (1 << 30) && rows_aligned(a.k, elem, a.k_t, a.k_h) && rows_aligned(a.v, elem, a.v_t, a.v_h)) {
    if (dtype == SA_REP_FLOAT32) return append_vec<SA_REP_FLOAT32>(a, s);
    if (dtype == SA_REP_FLOAT16) return append_vec<SA_REP_FLOAT16>(a, s);
    return append_vec<SA_REP_BFLOAT16>(a, s);
  }
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
  if (a.c.d % 8 == 0 && a.tokens * a.c.heads < (1 << 30) && (((uintptr_t)a.k | (uintptr_t)a.v) & 15) == 0) {
    if (dtype == SA_REP_FLOAT32) return read_vec<SA_REP_FLOAT32>(a, s);
    if (dtype == SA_REP_FLOAT16) return read_vec<SA_REP_FLOAT16>(a, s);
    return read_vec<SA_REP_BFLOAT16>(a, s);
  }
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
