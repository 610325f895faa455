// The queries of all requests over a prefix that they share, on the 5th-generation
// tensor cores (tcgen05 kind::f16, TMEM): float16 and bfloat16, head widths up to 128.
// What the prefix of a batch adds to each row: an unfinished sum, its maximum and total
// for kTail (kv4_attend.cuh), as kPrefix there, which takes the other types and few rows.
//
// Operands are float16.  A scale has 8 bits and a code less 8 at most 3, so their
// product is exact in float16's 11, and with x = least + 8 scale
//   score_j = scale (sum_c q_c k'_jc + x_j sum(Q)),   k' = scale (code - 8),
// the second term as 16 more columns of the same product: x_j and sum(Q) in three pieces
// each.  Values are rounded once, to float16 (half a step, 2^-11 of them at most), and so are
// probabilities: fewer bits than kv4_attend.cuh keeps (16 of a probability, codes as they are), which
// bfloat16's rounding hides and float16's does not quite (errors of 2.5e-4, not 2.1e-4, of the result);
// two pieces of either would be twice the products.  Powers of two keep all in float16's range: one for each query row, one
// for the keys and one for the values of a CTA, from the largest of what some row sees.
// Where a token's are so much smaller than the largest that they would lose bits (2^-16 for
// keys, 2^-13 for values), the CTA's rows go over their tokens in float32 instead (plain_rows),
// a warp a row and a token at a time: right, and slow (64 requests of 32 heads over 8 of 128, one such token: behind
// 4000 tokens 39 -> 2150 us, behind 32000 72 -> 14400).
// (Scales outside the products, bfloat16 codes inside: each score then wants 16 bytes of
// parameters out of shared memory, 2048 of its cycles a tile, and the kernel took 85 us.)
// 64 requests of 32 heads over 8 of 128 behind 32000 tokens: 60 us (33 GFLOP, 20 us at the
// measured GEMM rate).  Its 28 tiles a CTA take about 1 us each, a chain of waits, and set-up and end 8: of the
// other 24 us the cause is not known.  Left out in turn, products were worth 4 us, decoding 7, the
// exponentials none, all of them together 11.
//
// A CTA holds two tiles of 128 query rows of one key head (a row: request, query, head)
// and a part of the prefix in tiles of 64 tokens; all rows see (nearly) all of it, so a
// decoded tile serves 256 rows.  Warps: 0..7 and 8..15 are the softmax of a row tile, two
// threads a row (the exponentials' unit is shared, and four warps beside it keep it busy where
// two, in step, left it idle half of the time); 16..19 decode keys and 20..23 values, from raw tiles
// that warp 26 brings in ahead (bulk copies) to swizzled ones; 24 and 25 issue the products of a
// row tile, one elected lane.  TMEM: of each row tile two S of 64 columns and O; P overwrites the first
// half of its S.  The issuer goes P V(j), S(j + 2), so that scores are there while a softmax
// runs.
//
// Order inside the tiles.  A word of a key row holds eight columns' codes, of which one
// logical operation gives two (columns i and i + 4) as 1024 + code or 64 + code, so keys and
// queries hold columns in the order 0 4 1 5 2 6 3 7.  A word of values holds four tokens of
// two columns, and gives tokens 0 and 2, 1 and 3: values lie a column to a row, tokens in the
// order 0 2 1 3, and P's halves are packed to match.
//
// A token whose value is not finite gets values of 0 and a key that is NaN: whoever sees
// it comes out NaN, and nobody else.
#include <math.h>

#include <algorithm>
#include <cmath>

#include "kv4_attend.cuh"
#include "tc_util.cuh"

namespace sa {

namespace {

using namespace tc;

constexpr int kTileRows = 128;
constexpr int kTokens = 64;        // of a tile
constexpr int kRowTiles = 2;
constexpr int kCtaRows = kRowTiles * kTileRows;
constexpr int kHalf = kTokens / 2;
constexpr int kSoftmax = 2 * kCtaRows;   // two threads a row, each of half of a tile's tokens
constexpr int kDecoders = 128;     // of keys, and as many of values
constexpr int kIssuer = (kSoftmax + 2 * kDecoders) / 32;   // the first of two warps
constexpr int kLoader = kIssuer + kRowTiles;
constexpr int kPrefixThreads = (kLoader + 2) * 32;          // whole groups of four warps
// Registers of a thread: launched with 72 (65536 / 896, in steps of 8), then dealt out by groups of four
// warps: 4 x 80 + 2 x 64 + 56 = 7 x 72.
constexpr int kSoftmaxRegs = 80, kDecoderRegs = 64, kOtherRegs = 56;
static_assert(4 * kSoftmaxRegs + 2 * kDecoderRegs + kOtherRegs <= 7 * 72, "more registers than the launch has");
constexpr float kShiftP = 6.0f;    // P = 2^(x - m + 6), m at most kMove below the largest x: 2^14 at most, and 2^-14,
                                   // where float16 starts to lose bits, is 2^-20 of a row's usual largest.  It shows where a token
                                   // of value 0 has nearly all weight: results of others that have 2^-26 / 2^-28 of it each are 0.3 /
                                   // 1 % off.  With m moved at 4, and P up to 2^15, that is 0.05 / 0.07 %, and 64 requests behind 32000
                                   // tokens 72 -> 80 us.

constexpr int kErrK = 521, kErrV = 522, kErrP = 523, kErrS = 524, kErrEmpty = 525, kErrO = 526, kErrDrain = 527, kErrRaw = 528;

struct PrefixParams {
  Kv4AttendArgs a;
  int rows;      // requests * n * group
  uint64_t wait_ns;
};

template <int DP>
struct PrefixLayout {
  static constexpr int kChunks = (DP + 63) / 64;             // of 64 columns: a row of 128 bytes
  static constexpr int kQ = kChunks * kTileRows * 128;
  static constexpr int kK = kChunks * kTokens * 128;
  static constexpr int kV = DP * 128;
  static constexpr int kStages = 3;
  // the 16 columns of the sums and of the offsets: rows of 32 bytes
  static constexpr int kQSum = kTileRows * 32, kKOff = kTokens * 32;
  // a raw tile: keys, values, their parameters, and which tokens of each block of 16 some row sees
  static constexpr int kRawV = kTokens * DP / 2, kRawKp = 2 * kRawV, kRawVp = kRawKp + kTokens * 4;
  static constexpr int kRawInfo = kRawVp + kTokens * 4, kRaw = kRawInfo + 16;
  static constexpr int kRawStages = 4;
  static constexpr int kKeys = kRowTiles * kQ;
  static constexpr int kValues = kKeys + kStages * kK;
  static constexpr int kSums = kValues + kStages * kV;
  static constexpr int kOffsets = kSums + kRowTiles * kQSum;
  static constexpr int kPowers = kOffsets + kStages * kKOff;   // of the rows
  static constexpr int kRows = kPowers + kCtaRows * 4;         // where the rows of q start
  static constexpr int kTops = kRows + kCtaRows * 8;           // what a row's threads tell each other: [two turns][half][row]
  static constexpr int kPositions = kTops + 4 * kCtaRows * 4;
  static constexpr int kRaws = kPositions + kCtaRows * 4;
  static constexpr int kBars = kRaws + kRawStages * kRaw;
  static constexpr int kBytes = kBars + (4 * kStages + 2 * kRawStages + 12) * 8 + 64 + 1024;
  static_assert(kBytes <= 227 * 1024, "shared memory");
  static_assert(kValues % 1024 == 0 && kKeys % 1024 == 0 && kSums % 1024 == 0 && kOffsets % 1024 == 0 && kRaws % 16 == 0 &&
                kRaw % 16 == 0 && kBars % 8 == 0, "alignment of tiles, copies and barriers");
};

__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t x, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Ties loaded registers to this point of the program: what follows uses them after the
// wait that stands before.
__device__ __forceinline__ void tie16(float* v) {
  asm volatile("" : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
               "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]));
}
__device__ __forceinline__ void tie32(float (&v)[32]) {
  tie16(v);
  tie16(v + 16);
}

// The barrier of two warps.  A warp that gives up arrives there once more, so that its
// mate, should it wait, goes on to find the abort word set.
__device__ __forceinline__ void pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ void pair_leave(int id) { asm volatile("bar.arrive %0, 64;" ::"r"(id) : "memory"); }

template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

// O of a row times alpha, in TMEM (rare).
__device__ __noinline__ void scale_row(uint32_t to, int columns, float alpha) {
#pragma unroll 1
  for (int c = 0; c < columns; c += 16) {
    float o[16];
    tmem_ld16(to + c, o);
    tmem_wait_ld();
    tie16(o);
    uint32_t os[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) os[e] = __float_as_uint(o[e] * alpha);
    tmem_st16(to + c, os);
  }
  tmem_wait_st();
}

// What the roles need of the set-up, in shared memory: what a register held from there on would be spilled,
// and beside this much shared memory a spilled one is read from L2.
struct Span {
  int p_lo, p_hi;              // least and largest position of the CTA's rows
  uint32_t k_size, v_size;     // bits of the largest of its keys and values
  uint32_t k_least, v_least;   // and of the smallest that are not zero
  uint32_t bad;                // whether pages are not there
  int low;                     // no row's window begins before
  int bound;                   // no token stands there or behind
  int first, tiles;            // this part's tiles
  int sink_tiles, win_tile;    // tile t of all is the t-th of the sequence, or from sink_tiles on the (win_tile + t - sink_tiles)-th
  // the first token of this part's tile j
  __device__ __forceinline__ int token_of(int j) const {
    const int t = first + j;
    return (t < sink_tiles ? t : win_tile + t - sink_tiles) * kTokens;
  }
  // whether what a token holds may be so small beside the largest that float16 loses bits of it
  __device__ __forceinline__ bool wide() const {
    return __uint_as_float(k_size) > 65536.0f * __uint_as_float(k_least) || __uint_as_float(v_size) > 8192.0f * __uint_as_float(v_least);
  }
};

// The x lowest bits set (x may be anything).
__device__ __forceinline__ uint32_t low_bits(int x) {
  return x >= 32 ? 0xffffffffu : (x <= 0 ? 0u : (1u << x) - 1u);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ uint32_t fma_f16(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t mul_f16(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t add_f16(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Eight codes less kBias, two at a time (nibble i of each half of w), as float16: a code in a
// mantissa's low bits is added to 1024, four bits further up to 64.
template <int kBias>
__device__ __forceinline__ void codes16(uint32_t w, uint32_t (&c)[4]) {
  constexpr uint32_t kLow = kBias == 0 ? 0xe400e400u : 0xe408e408u, kHigh = kBias == 0 ? 0xd400d400u : 0xd480d480u;   // -1024, -1032; -64, -72
  const uint32_t u = w >> 8;
  c[0] = add_f16((w & 0x000f000fu) | 0x64006400u, kLow);
  c[1] = add_f16((w & 0x00f000f0u) | 0x54005400u, kHigh);
  c[2] = add_f16((u & 0x000f000fu) | 0x64006400u, kLow);
  c[3] = add_f16((u & 0x00f000f0u) | 0x54005400u, kHigh);
}

// Shared-memory matrix descriptor of rows of 32 bytes, 32-byte swizzle (layout type 6): the 16-byte halves of
// rows 4..7 of eight are swapped.
__device__ __forceinline__ uint64_t sdesc_sw32(uint32_t saddr) {
  return (sdesc_sw128(saddr, 16, 256) & ~(7ull << 61)) | (6ull << 61);
}
__device__ __forceinline__ int sw32(int row, int half) { return row * 32 + ((half ^ ((row >> 2) & 1)) << 4); }

// The power of two that brings a value of this size to [2^to, 2^(to + 1)); 1 for zero, infinities and NaN.
__device__ __forceinline__ int power_for(float size, int to) {
  const int e = (int)(__float_as_uint(size) >> 23) & 255;
  return size == 0.0f || e == 255 ? 0 : min(max(to + 127 - e, -126), 126);
}
__device__ __forceinline__ float power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Whether both parameters of a row are finite (their halves' sum is then).
__device__ __forceinline__ bool finite(const float2& params) {
  return fmaf(0.5f, fabsf(params.x), 0.5f * fabsf(params.y)) < INFINITY;
}

// The size of a row of these parameters: of finite ones finite, of others none (NaN).
__device__ __forceinline__ float size_of(const float2& params, float size) {
  return finite(params) ? fminf(size, 3.40282347e38f) : NAN;
}

// x in three float16 pieces.
__device__ __forceinline__ void pieces(float x, float (&y)[3]) {
#pragma unroll
  for (int e = 0; e < 3; ++e) {
    y[e] = __half2float(__float2half_rn(x));
    x -= y[e];
  }
}

// P of 32 tokens: p = 2^(s c2 + off), its sum, and in float16 to TMEM.
__device__ __forceinline__ void exp_chunk(const float (&s)[32], uint64_t c22, uint64_t off2, uint64_t (&sum2)[2], uint32_t to) {
  uint32_t pk[16];
#pragma unroll
  for (int g = 0; g < 8; ++g) {   // four tokens: pairs 0 2 and 1 3
    float x[4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      unpack2(fma2(pack2(s[4 * g + 2 * e], s[4 * g + 2 * e + 1]), c22, off2), x[2 * e], x[2 * e + 1]);
      x[2 * e] = ex2(x[2 * e]);
      x[2 * e + 1] = ex2(x[2 * e + 1]);
      sum2[e] = add2(sum2[e], pack2(x[2 * e], x[2 * e + 1]));
    }
    pk[2 * g] = pack_f16(x[0], x[2]);
    pk[2 * g + 1] = pack_f16(x[1], x[3]);
  }
  tmem_st16(to, pk);
}

__device__ __forceinline__ float max32(const float (&s)[32]) {
  float t[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
  for (int e = 4; e < 28; e += 8)
#pragma unroll
    for (int x = 0; x < 4; ++x) t[x] = max3(t[x], s[e + 2 * x], s[e + 2 * x + 1]);
  return fmaxf(max3(t[0], t[1], s[28]), max3(max3(t[2], t[3], s[29]), s[30], s[31]));
}

// A part's rows over its tokens in float32, a warp a row and a token at a time: where float16 would not do.
template <int DT, int DP>
__device__ __noinline__ void plain_rows(const Kv4AttendArgs& a, int rows, const Span& sp, const int64_t* starts, const int* positions) {
  using T = typename Elem<DT>::T;
  constexpr int kCols = DP / 32;   // column lane + 32 i
  const int lane = threadIdx.x & 31;
  const float sc = a.scale * 1.4426950408889634f;
  const int64_t of = (int64_t)blockIdx.x * a.c.heads + blockIdx.z;
  for (int r = threadIdx.x >> 5; r < kCtaRows; r += kPrefixThreads / 32) {
    const int row = blockIdx.y * kCtaRows + r;
    if (row >= rows) break;
    const int position = positions[r];
    float q[kCols], o[kCols], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < kCols; ++i) {
      const int c = lane + 32 * i;
      q[i] = c < a.c.d ? to_f32(static_cast<const T*>(a.q)[starts[r] + c]) : 0.0f;
      o[i] = 0.0f;
    }
#pragma unroll 1
    for (int x = 0; position >= 0 && x < sp.tiles * kTokens; ++x) {
      const int j = sp.token_of(x / kTokens) + x % kTokens;
      if (j >= sp.bound || !(position - j < a.window || j < a.sinks)) continue;
      const int page = __ldg(a.prefix_table + (j >> a.c.page_shift));
      if (page < 0 || page >= a.c.pages) continue;
      const int64_t cell = ((page * (int64_t)a.c.heads + blockIdx.z) << a.c.page_shift) + (j & ((1 << a.c.page_shift) - 1));
      const float2 k = params(__ldg(reinterpret_cast<const uint32_t*>(a.c.k_params) + cell));
      const float2 v = params(__ldg(reinterpret_cast<const uint32_t*>(a.c.v_params) + cell));
      float s = 0.0f, value[kCols];
#pragma unroll
      for (int i = 0; i < kCols; ++i) {
        const int c = lane + 32 * i, shift = 4 * (c & 1);
        s = fmaf(q[i], fmaf((float)((a.c.k_codes[cell * (DP / 2) + (c >> 1)] >> shift) & 15), k.x, k.y), s);
        value[i] = fmaf((float)((a.c.v_codes[(cell & ~(int64_t)3) * (DP / 2) + (c >> 1) * 4 + (cell & 3)] >> shift) & 15), v.x, v.y);
      }
#pragma unroll
      for (int d = 16; d >= 1; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
      s *= sc;
      const float top = fmaxf(m, s), alpha = top == -INFINITY ? 1.0f : ex2(m - top);
      const float p = ex2(s + kShift - (top == -INFINITY ? 0.0f : top));
      m = top;
      l = fmaf(l, alpha, p);
#pragma unroll
      for (int i = 0; i < kCols; ++i) o[i] = fmaf(o[i], alpha, p * value[i]);
    }
    if (lane == 0) a.part_ml[of * rows + row] = make_float2(m, l);
#pragma unroll
    for (int i = 0; i < kCols; ++i) {
      const int c = lane + 32 * i;
      a.part_o[((of * (DP / 4) + c / 4) * rows + row) * 4 + c % 4] = m == -INFINITY ? 0.0f : o[i];
    }
  }
}

template <int DT, int DP>
__global__ void __launch_bounds__(kPrefixThreads, 1) prefix_tc_kernel(const __grid_constant__ PrefixParams p) {
  using L = PrefixLayout<DP>;
  using T = typename Elem<DT>::T;
  constexpr int kStages = L::kStages;
  next_may_start();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t* kempty = kfull + kStages;
  uint64_t* vfull = kempty + kStages;
  uint64_t* vempty = vfull + kStages;
  uint64_t* rfull = vempty + kStages;
  uint64_t* rempty = rfull + L::kRawStages;
  uint64_t* sfull = rempty + L::kRawStages;   // [row tile][score buffer]
  uint64_t* pfull = sfull + 4;           // likewise
  uint64_t* pvdone = pfull + 4;          // [row tile]: a P V has ended
  uint64_t* drain = pvdone + 2;          // [row tile]: every product has
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  int* abort_word = reinterpret_cast<int*>(tmem_slot + 1);
  Span* span = reinterpret_cast<Span*>(abort_word + 2);
  static_assert(sizeof(Span) + 12 <= 64, "behind the barriers");

  const Kv4AttendArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = blockIdx.x, parts = gridDim.x, row0 = blockIdx.y * kCtaRows, hk = blockIdx.z;
  const int group = a.heads / a.c.heads;
  const int live = p.rows - row0 > kTileRows ? 2 : 1;   // row tiles with rows
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&kfull[s], kDecoders / 32);
      mbar_init(&kempty[s], live);
      mbar_init(&vfull[s], kDecoders / 32);
      mbar_init(&vempty[s], live);
    }
    for (int s = 0; s < L::kRawStages; ++s) {
      mbar_init(&rfull[s], 1);
      mbar_init(&rempty[s], 2 * kDecoders / 32);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sfull[i], 1);
      mbar_init(&pfull[i], 8);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&pvdone[i], 1);
      mbar_init(&drain[i], 1);
    }
    abort_word[0] = abort_word[1] = 0;
    *span = Span{2147483647, -1, 0, 0, 0x7f800000u, 0x7f800000u, 0, 0, 0, 0, 0, 0, 0};
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == kIssuer) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  __syncthreads();
  const int cap = a.width << a.c.page_shift;
  const int length = max(a.prefix_length[0], 0), bound = min(length, cap);
  if (length > cap && threadIdx.x == 0) report(a.status, kBadPrefix, 0);
  // a softmax thread's row: where it stands, -1 where it sees nothing
  const int half = (warp >> 2) & 1, rt = (warp >> 3) * kTileRows + (warp & 3) * 32 + lane;   // (of the softmax's threads)
  const int row = row0 + rt;
  if (threadIdx.x < kSoftmax) {
    int position = -1;
    int64_t start = -1;   // no row
    if (row < p.rows) {
      const int x = row / group, q = x / a.n;
      start = q * a.q_r + (x - q * a.n) * a.q_n + (int64_t)(hk * group + row - x * group) * a.q_h;
      const int own = max(a.lengths[q], 0) - a.n + (x - q * a.n);   // only a request's own tokens ask
      if (own >= 0) position = (int)min((int64_t)length + own, (int64_t)2147483646);
    }
    if (half == 0) {
      reinterpret_cast<int64_t*>(smem + L::kRows)[rt] = start;
      reinterpret_cast<int*>(smem + L::kPositions)[rt] = position;
    }
    const int least = __reduce_min_sync(0xffffffffu, position < 0 ? 2147483647 : position);
    const int most = __reduce_max_sync(0xffffffffu, position);
    if (lane == 0) {
      atomicMin(&span->p_lo, least);
      atomicMax(&span->p_hi, most);
    }
  }
  __syncthreads();
  // the tiles of 64 tokens, from multiples of 64 on, that hold what rows see, and this part's of them
  Span all_of = *span;
  KeyRanges kr{0, 0, 0};
  if (all_of.p_hi >= 0) kr = key_ranges(all_of.p_lo, all_of.p_hi, bound, a.window, a.sinks);
  all_of.bound = bound;
  all_of.low = (int)max((int64_t)all_of.p_lo - a.window + 1, (int64_t)0);
  all_of.sink_tiles = (int)((kr.first + kTokens - 1) / kTokens);
  all_of.win_tile = max((int)(kr.begin / kTokens), all_of.sink_tiles);
  const int all = all_of.sink_tiles + max((int)((kr.end + kTokens - 1) / kTokens) - all_of.win_tile, 0);
  all_of.first = (int)((int64_t)all * part / parts);
  all_of.tiles = (int)((int64_t)all * (part + 1) / parts) - all_of.first;
  const int64_t cell0 = (int64_t)hk << a.c.page_shift;
  const int64_t page_step = (int64_t)a.c.heads << a.c.page_shift;
  const int page_mask = (1 << a.c.page_shift) - 1;
  // Q: eight columns at a time, the DP / 8 lanes of a row together; loads first, all on their way at once
  constexpr int kQLoads = (kCtaRows * (DP / 8) + kPrefixThreads - 1) / kPrefixThreads;
  uint4 q_raw[kQLoads];
#pragma unroll
  for (int i = 0; i < kQLoads; ++i) {
    const int x = i * kPrefixThreads + (int)threadIdx.x, r = x / (DP / 8), c8 = x - r * (DP / 8);
    q_raw[i] = make_uint4(0, 0, 0, 0);
    const int64_t start = r < kCtaRows ? reinterpret_cast<const int64_t*>(smem + L::kRows)[r] : -1;
    if (start >= 0) {
      const T* from = static_cast<const T*>(a.q) + start + c8 * 8;
      if (a.vec_q && c8 * 8 + 8 <= a.c.d) {
        q_raw[i] = *reinterpret_cast<const uint4*>(from);
      } else {
        union {
          uint4 w;
          T e[8];
        } u;
        u.w = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c8 * 8 + e < a.c.d) u.e[e] = from[e];
        q_raw[i] = u.w;
      }
    }
  }
  // the largest of the part's keys and values
  {
    float k_size = 0.0f, v_size = 0.0f, k_least = INFINITY, v_least = INFINITY;
    bool bad = false;
#pragma unroll 2
    for (int x = threadIdx.x; x < all_of.tiles * kTokens; x += kPrefixThreads) {
      const int token = all_of.token_of(x / kTokens) + x % kTokens;
      const int page = token < bound ? __ldg(a.prefix_table + (token >> a.c.page_shift)) : 0;
      const bool out = page < 0 || page >= a.c.pages;
      if (out) {
        report(a.status, kBadPage, page);
        bad = true;
      }
      const int64_t cell = (out ? 0 : page) * page_step + cell0 + (token & page_mask);
      const bool in = !out && token < bound && (token >= all_of.low || token < a.sinks);   // some row sees it
      const float2 k = params(__ldg(reinterpret_cast<const uint32_t*>(a.c.k_params) + cell));
      const float2 v = params(__ldg(reinterpret_cast<const uint32_t*>(a.c.v_params) + cell));
      // (a row's parameters may be finite where a code that it does not have would pass float32: it is as large as any)
      const float ks = size_of(k, fmaxf(8.0f * fabsf(k.x), fabsf(fmaf(8.0f, k.x, k.y))));
      const float vs = size_of(v, fmaxf(fabsf(v.y), fabsf(fmaf(15.0f, v.x, v.y))));
      if (in && ks < INFINITY && ks > 0.0f) {
        k_size = fmaxf(k_size, ks);
        k_least = fminf(k_least, ks);
      }
      if (in && vs < INFINITY && vs > 0.0f) {
        v_size = fmaxf(v_size, vs);
        v_least = fminf(v_least, vs);
      }
    }
    const uint32_t k_bits = __reduce_max_sync(0xffffffffu, __float_as_uint(k_size));
    const uint32_t v_bits = __reduce_max_sync(0xffffffffu, __float_as_uint(v_size));
    const uint32_t k_low = __reduce_min_sync(0xffffffffu, __float_as_uint(k_least));
    const uint32_t v_low = __reduce_min_sync(0xffffffffu, __float_as_uint(v_least));
    bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) {
      atomicMax(&span->k_size, k_bits);
      atomicMax(&span->v_size, v_bits);
      atomicMin(&span->k_least, k_low);
      atomicMin(&span->v_least, v_low);
      if (bad) atomicOr(&span->bad, 1u);
    }
  }
  if (threadIdx.x == 0) {
    span->bound = all_of.bound;
    span->low = all_of.low;
    span->first = all_of.first;
    span->tiles = all_of.tiles;
    span->sink_tiles = all_of.sink_tiles;
    span->win_tile = all_of.win_tile;
  }
  // Q in the order 0 4 1 5 2 6 3 7, times the row's power; behind it the sums' pieces, which meet the
  // offsets' as 1 1 1 2 2 3
  const float sign = a.scale < 0.0f ? -1.0f : 1.0f;
#pragma unroll
  for (int i = 0; i < kQLoads; ++i) {
    const int x = i * kPrefixThreads + (int)threadIdx.x, r = x / (DP / 8), c8 = x - r * (DP / 8);
    union {
      uint4 w;
      T e[8];
    } u;
    u.w = q_raw[i];
    float v[8], top = 0.0f, sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = to_f32(u.e[e]);
      top = fmaxf(top, fabsf(v[e]));
    }
#pragma unroll
    for (int d = 1; d < DP / 8; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const int e2 = power_for(top, 7);
    const float f = power(e2) * sign;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] *= f;
      sum += v[e];
    }
#pragma unroll
    for (int d = 1; d < DP / 8; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const int t = r / kTileRows, rt = r % kTileRows;
    if (r >= kCtaRows) continue;
    *reinterpret_cast<uint4*>(smem + t * L::kQ + (c8 >> 3) * (kTileRows * 128) + rt * 128 + (((c8 & 7) ^ (rt & 7)) << 4)) =
        make_uint4(pack_f16(v[0], v[4]), pack_f16(v[1], v[5]), pack_f16(v[2], v[6]), pack_f16(v[3], v[7]));
    if (c8 < 2) {
      float y[3];
      pieces(sum, y);
      *reinterpret_cast<uint4*>(smem + L::kSums + t * L::kQSum + sw32(rt, c8)) =
          c8 == 0 ? make_uint4(pack_f16(y[0], y[1]), pack_f16(y[2], y[0]), pack_f16(y[1], y[0]), 0) : make_uint4(0, 0, 0, 0);
      if (c8 == 0) reinterpret_cast<int*>(smem + L::kPowers)[r] = e2;
    }
  }
  // of the offsets' 16 columns the last eight stay zero
  for (int x = threadIdx.x; x < kStages * kTokens; x += kPrefixThreads)
    *reinterpret_cast<uint4*>(smem + L::kOffsets + (x / kTokens) * L::kKOff + sw32(x % kTokens, 1)) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (span->wide()) {
    if (warp == kIssuer) tmem_dealloc(tmem, 512);
    plain_rows<DT, DP>(a, p.rows, *span, reinterpret_cast<const int64_t*>(smem + L::kRows), reinterpret_cast<const int*>(smem + L::kPositions));
    return;
  }
  const volatile Span* now = span;
  const int tiles = now->tiles;
  const Abort ab{abort_word, a.status, p.wait_ns};

  if (threadIdx.x < kSoftmax) {
    // ------------------------------------------------------------ softmax rows
    more_registers<kSoftmaxRegs>();
    const int t = warp >> 3;
    if (t < live) {
      const uint32_t at = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t tO = tmem + 256 + t * 128 + at + half * (DP / 2);
      const int q_power = reinterpret_cast<const volatile int*>(smem + L::kPowers)[rt];
      const int position = reinterpret_cast<const volatile int*>(smem + L::kPositions)[rt];
      const int k_power = power_for(__uint_as_float(now->k_size), 9);
      const Span sp{0, now->p_hi, 0, now->v_size, 0, 0, now->bad, 0, now->bound, now->first, tiles, now->sink_tiles, now->win_tile};
      const int window = (int)min(a.window, (int64_t)2147483647), sinks = (int)min(a.sinks, (int64_t)2147483647);
      float* tops = reinterpret_cast<float*>(smem + L::kTops);
      const int pair = 1 + t * 4 + (warp & 3);   // the barrier of the two warps of 32 rows
      // scores in base 2 from the products; the powers one after the other, since their product may leave the range
      // (0, of a scale of 0, would make NaN of a hidden score: the least that is none)
      const float c2s = fabsf(a.scale) * 1.4426950408889634f * power(-q_power) * power(-k_power), c2 = c2s == 0.0f ? 1.17549435e-38f : c2s;
      const uint64_t c22 = pack2(c2, c2);
      float m = -INFINITY, l = 0.0f;
      bool ok = true;
#pragma unroll 1
      for (int j = 0; j < tiles; ++j) {
        const int buf = j & 1;
        // whether every row that sees anything sees all 64 tokens
        const int t0 = sp.token_of(j);
        const bool whole = !sp.bad && t0 <= sp.bound - kTokens && (sp.p_hi - t0 < window || t0 <= sinks - kTokens);   // (t0 + kTokens may be 2^31)
        ok = mbar_wait_warp_lazy(&sfull[2 * t + buf], (j >> 1) & 1, ab, kErrS);
        if (!ok) break;
        tc_fence_after();
        const uint32_t ts = tmem + t * 128 + buf * kTokens + at;
        float s[32];
        tmem_ld32(ts + half * kHalf, s);
        tmem_wait_ld();
        tie32(s);
        if (!whole) {
          // token j: j < bound and (j > position - window or j < sinks); j <= position always
          const int j0 = t0 + half * kHalf;
          const uint32_t near = position - j0 < window ? 0xffffffffu : ~low_bits(position - j0 - window + 1);
          uint32_t on = low_bits(sp.bound - j0) & (near | low_bits(sinks - j0));
          for (int b = 0; sp.bad && b < 2; ++b) {   // a page that is not there
            const int first16 = j0 + 16 * b, page = first16 < sp.bound ? __ldg(a.prefix_table + (first16 >> a.c.page_shift)) : 0;
            if (page < 0 || page >= a.c.pages) on &= 0xffff0000u >> (16 * b);
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) s[e] = (on >> e) & 1u ? s[e] : -INFINITY;
        }
        // the row's maximum: both its threads hear of both halves (and have read their scores, which P overwrites)
        const float mine = max32(s);
        tops[(buf * 2 + half) * kCtaRows + rt] = mine;
        pair_sync(pair);
        if (*ab.cta) {   // the other warp may be gone
          ok = false;
          break;
        }
        // no less than the product that exp_chunk takes it from, which is not rounded (NaN, where nothing is seen, moves nothing)
        const float rounded = fmaxf(mine, tops[(buf * 2 + (half ^ 1)) * kCtaRows + rt]) * c2;
        const float top = fmaf(fabsf(rounded), 0x1p-23f, rounded);
        const bool move = top > m + kMove;
        if (__any_sync(0xffffffffu, move)) {
          const float to = move ? top : m;
          const float alpha = move ? ex2(m - to) : 1.0f;   // m = -inf: 0
          m = to;
          l *= alpha;
          if (j > 0) {   // the product of the tile before may still run (that of the one before it ended before S(j))
            ok = mbar_wait_warp_lazy(&pvdone[t], (j - 1) & 1, ab, kErrO);
            if (!ok) break;
            tc_fence_after();
            scale_row(tO, DP / 2, alpha);
          }
        }
        const float off = kShiftP - (m == -INFINITY ? 0.0f : m);
        uint64_t sum2[2] = {0, 0};
        exp_chunk(s, c22, pack2(off, off), sum2, ts + half * (kHalf / 2));
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&pfull[2 * t + buf]);
        float x0, x1, x2, x3;
        unpack2(sum2[0], x0, x1);
        unpack2(sum2[1], x2, x3);
        l += (x0 + x1) + (x2 + x3);
      }
      if (!ok) pair_leave(pair);   // nobody waits for this warp
      if (ok && tiles > 0) {
        // not pvdone: P V of the last tile but one may still run too, and a parity tells only neighbours apart
        ok = mbar_wait_warp_lazy(&drain[t], 0, ab, kErrO);
        tc_fence_after();
      }
      // this part's sums, as kTail's own p has them: [part][key head][columns / 4][row][4]
      const int64_t of = (int64_t)part * a.c.heads + hk;
      const bool some = ok && tiles > 0 && position >= 0 && m != -INFINITY;
      const float f = power((int)(kShift - kShiftP)), fo = f * power(-power_for(__uint_as_float(sp.v_size), 9));
#pragma unroll 1
      for (int c = 0; c < DP / 2; c += 16) {
        float o[16];
        if (tiles > 0) {
          tmem_ld16(tO + c, o);
          tmem_wait_ld();
          tie16(o);
        }
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          if (row < p.rows)
            *reinterpret_cast<float4*>(a.part_o + ((of * (DP / 4) + (half * (DP / 2) + c + e) / 4) * p.rows + row) * 4) =
                some ? make_float4(o[e] * fo, o[e + 1] * fo, o[e + 2] * fo, o[e + 3] * fo) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
      tc_fence_before();
      // maximum and total: the other half's through shared memory, behind the last barrier
      const bool seen = ok && tiles > 0 && position >= 0;
      if (half == 0)   // (where rows of q start, and positions, are not needed any more)
        reinterpret_cast<float2*>(smem + L::kRows)[rt] = seen ? make_float2(m, l * f) : make_float2(-INFINITY, 0.0f);
      else
        reinterpret_cast<float*>(smem + L::kPositions)[rt] = seen ? l * f : 0.0f;
    }
  } else if (warp < kIssuer) {
    // ------------------------------------------------------------ codes to tiles
    fewer_registers<kDecoderRegs>();
    const bool isv = warp >= (kSoftmax + kDecoders) / 32;
    const int d = (threadIdx.x - kSoftmax) % kDecoders;
    bool ok = true;
    if (!isv) {
      // keys: a thread takes 16 bytes (32 columns) of tokens; eight lanes are eight tokens, so that their
      // stores fall into different banks
      constexpr int kPieces = DP / 32;
      constexpr int kLoads = (kTokens * kPieces + kDecoders - 1) / kDecoders;
      const float f = power(power_for(__uint_as_float(now->k_size), 9));
#pragma unroll 1
      for (int j = 0; j < tiles; ++j) {
        const int s = j % kStages, rs = j % L::kRawStages;
        ok = mbar_wait_warp_lazy(&rfull[rs], (j / L::kRawStages) & 1, ab, kErrRaw);
        if (!ok) break;
        const uint8_t* raw = smem + L::kRaws + rs * L::kRaw;
        uint4 w[kLoads];
        uint32_t kp[kLoads], vp[kLoads];
        bool in[kLoads];
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int u = i * kDecoders + d, token = (u / (8 * kPieces)) * 8 + (u & 7), piece = (u >> 3) % kPieces;
          if (token >= kTokens) continue;
          w[i] = *reinterpret_cast<const uint4*>(raw + token * (DP / 2) + piece * 16);
          kp[i] = *reinterpret_cast<const uint32_t*>(raw + L::kRawKp + token * 4);
          vp[i] = *reinterpret_cast<const uint32_t*>(raw + L::kRawVp + token * 4);
          in[i] = (reinterpret_cast<const uint32_t*>(raw + L::kRawInfo)[token >> 4] >> (token & 15)) & 1u;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&rempty[rs]);
        if (j >= kStages) ok = mbar_wait_warp_lazy(&kempty[s], ((j / kStages) - 1) & 1, ab, kErrEmpty);
        if (!ok) break;
        uint8_t* tile = smem + L::kKeys + s * L::kK;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int u = i * kDecoders + d, token = (u / (8 * kPieces)) * 8 + (u & 7), piece = (u >> 3) % kPieces;
          if (token >= kTokens) continue;
          const float2 k = params(in[i] ? kp[i] : 0u);
          const uint32_t s2 = pack_f16(k.x * f, k.x * f);
          const uint32_t ws[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
          uint8_t* to = tile + token * 128;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int c8 = piece * 4 + e;
            uint32_t c[4];
            codes16<8>(ws[e], c);
            *reinterpret_cast<uint4*>(to + (c8 >> 3) * (kTokens * 128) + (((c8 & 7) ^ (token & 7)) << 4)) =
                make_uint4(mul_f16(c[0], s2), mul_f16(c[1], s2), mul_f16(c[2], s2), mul_f16(c[3], s2));
          }
          if (piece == 0) {
            const float2 v = params(in[i] ? vp[i] : 0u);
            float y[3];
            pieces(finite(v) ? fmaf(8.0f, k.x * f, k.y * f) : NAN, y);
            *reinterpret_cast<uint4*>(smem + L::kOffsets + s * L::kKOff + sw32(token, 0)) =
                make_uint4(pack_f16(y[0], y[0]), pack_f16(y[0], y[1]), pack_f16(y[1], y[2]), 0);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&kfull[s]);
      }
    } else {
      // values: a thread takes 8 columns of 8 tokens; eight lanes are the eight such runs of a tile
      // (the columns turned by them, so that neither loads nor stores fall into one bank); quad < DP / 8
      constexpr int kTurn = DP >= 64 ? 8 : 4;
      const int chunk = d & 7, quad = ((d >> 3) & ~(kTurn - 1)) + (((d >> 3) + chunk) & (kTurn - 1));
      const float f = power(power_for(__uint_as_float(now->v_size), 9));
#pragma unroll 1
      for (int j = 0; j < tiles; ++j) {
        const int s = j % kStages, rs = j % L::kRawStages;
        ok = mbar_wait_warp_lazy(&rfull[rs], (j / L::kRawStages) & 1, ab, kErrRaw);
        if (!ok) break;
        const uint8_t* raw = smem + L::kRaws + rs * L::kRaw;
        uint4 w[2], ps[2];
        uint32_t on = 0;   // bit e: some row sees the e-th of the eight
        if (quad < DP / 8) {
          w[0] = *reinterpret_cast<const uint4*>(raw + L::kRawV + chunk * (4 * DP) + quad * 16);
          w[1] = *reinterpret_cast<const uint4*>(raw + L::kRawV + chunk * (4 * DP) + 2 * DP + quad * 16);
          ps[0] = *reinterpret_cast<const uint4*>(raw + L::kRawVp + chunk * 32);
          ps[1] = *reinterpret_cast<const uint4*>(raw + L::kRawVp + chunk * 32 + 16);
          on = reinterpret_cast<const uint32_t*>(raw + L::kRawInfo)[chunk >> 1] >> (chunk & 1) * 8;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&rempty[rs]);
        if (j >= kStages) ok = mbar_wait_warp_lazy(&vempty[s], ((j / kStages) - 1) & 1, ab, kErrEmpty);
        if (!ok) break;
        if (quad < DP / 8) {
          uint32_t s2[4], l2[4];   // tokens 0 2, 1 3, 4 6, 5 7
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t p4[4] = {ps[h].x, ps[h].y, ps[h].z, ps[h].w};
            float2 v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              v[e] = params((on >> (4 * h + e)) & 1u ? p4[e] : 0u);
              if (!finite(v[e])) v[e] = make_float2(0.0f, 0.0f);   // its key is NaN
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              s2[2 * h + e] = pack_f16(v[e].x * f, v[e + 2].x * f);
              l2[2 * h + e] = pack_f16(v[e].y * f, v[e + 2].y * f);
            }
          }
          const uint32_t w0[4] = {w[0].x, w[0].y, w[0].z, w[0].w}, w1[4] = {w[1].x, w[1].y, w[1].z, w[1].w};
          uint8_t* tile = smem + L::kValues + s * L::kV + quad * 8 * 128;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            uint32_t c[4], e[4];
            codes16<0>(w0[b], c);
            codes16<0>(w1[b], e);
            *reinterpret_cast<uint4*>(tile + 2 * b * 128 + ((chunk ^ (2 * b)) << 4)) =
                make_uint4(fma_f16(c[0], s2[0], l2[0]), fma_f16(c[2], s2[1], l2[1]), fma_f16(e[0], s2[2], l2[2]),
                           fma_f16(e[2], s2[3], l2[3]));
            *reinterpret_cast<uint4*>(tile + (2 * b + 1) * 128 + ((chunk ^ (2 * b + 1)) << 4)) =
                make_uint4(fma_f16(c[1], s2[0], l2[0]), fma_f16(c[3], s2[1], l2[1]), fma_f16(e[1], s2[2], l2[2]),
                           fma_f16(e[3], s2[3], l2[3]));
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&vfull[s]);
      }
    }
  } else {
    fewer_registers<kOtherRegs>();
    if (warp == kLoader) {
      // ---------------------------------------------------------- raw tiles
      // a tile is one run of tokens in a page, or of two or four in pages of 32 and 16: a lane for each and each of
      // keys, values and their parameters
      const int runs = max(kTokens >> a.c.page_shift, 1), tokens = kTokens / runs;
      const Span sp{0, 0, 0, 0, 0, 0, 0, now->low, now->bound, now->first, tiles, now->sink_tiles, now->win_tile};
      const int sinks = (int)min(a.sinks, (int64_t)2147483647);
      const int64_t cell0 = (int64_t)hk << a.c.page_shift, page_step = (int64_t)a.c.heads << a.c.page_shift;
      const int page_mask = (1 << a.c.page_shift) - 1;
      const int what = lane / runs, run = lane - what * runs;
      int page_l = 0;   // pages of 32 runs, one a lane: 32 / runs tiles
      int sent = 0;
#pragma unroll 1
      for (int j = 0; j < tiles; ++j) {
        const int rs = j % L::kRawStages, at = j % (32 / runs) * runs;
        if (at == 0) {
          const int token = sp.token_of(min(j + lane / runs, tiles - 1)) + lane % runs * tokens;
          page_l = token < sp.bound ? __ldg(a.prefix_table + (token >> a.c.page_shift)) : -1;
          if (page_l >= a.c.pages) page_l = -1;   // reported above
        }
        const int page = __shfl_sync(0xffffffffu, page_l, at + run), token = sp.token_of(j) + run * tokens;
        // what stands in a block of 16: four lanes say (runs are multiples of that)
        const int block_page = __shfl_sync(0xffffffffu, page_l, at + (lane & 3) * 16 / tokens);
        if (j >= L::kRawStages && !mbar_wait_warp_lazy(&rempty[rs], ((j / L::kRawStages) - 1) & 1, ab, kErrRaw)) break;
        uint8_t* raw = smem + L::kRaws + rs * L::kRaw;
        if (lane < 4) {   // which tokens of block `lane` some row sees
          const int j0 = sp.token_of(j) + lane * 16;
          reinterpret_cast<uint32_t*>(raw + L::kRawInfo)[lane] =
              block_page < 0 ? 0u : low_bits(sp.bound - j0) & (~low_bits(sp.low - j0) | low_bits(sinks - j0));
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(&rfull[rs], kTokens * DP + 2 * kTokens * 4);
        __syncwarp();
        // where there is no page, a valid one's bytes: nobody sees them
        const int64_t cell = max(page, 0) * page_step + cell0 + (token & page_mask);
        if (what < 4) {
          const uint32_t bytes = what < 2 ? tokens * (DP / 2) : tokens * 4;
          const void* from = what == 0   ? (const void*)(a.c.k_codes + cell * (DP / 2))
                             : what == 1 ? (const void*)(a.c.v_codes + cell * (DP / 2))
                             : what == 2 ? (const void*)(a.c.k_params + 2 * cell)
                                         : (const void*)(a.c.v_params + 2 * cell);
          bulk_load(raw + (what == 0 ? 0 : what == 1 ? L::kRawV : what == 2 ? L::kRawKp : L::kRawVp) + run * bytes, from, bytes, &rfull[rs]);
        }
        sent = j + 1;
        __syncwarp();
      }
      // never leave with copies in flight
      for (int j = max(0, sent - L::kRawStages); j < sent; ++j) {
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(&rfull[j % L::kRawStages], (j / L::kRawStages) & 1)) {
          if (globaltimer_ns() - t0 > 1000000000ull) {
            if (a.status) atomicCAS(a.status, 0, kErrDrain);
            break;
          }
        }
      }
      __syncwarp();
    } else if (warp < kLoader) {
      // ---------------------------------------------------------- products of row tile t
      const int t = warp - kIssuer;
      if (t < live) {
        constexpr uint32_t id_s = idesc_f16(kTileRows, kTokens, false, false, false);
        constexpr uint32_t id_pv = idesc_f16(kTileRows, DP, false, false, false);
        const uint32_t q_smem = smem_u32(smem) + t * L::kQ, k_smem = smem_u32(smem + L::kKeys), v_smem = smem_u32(smem + L::kValues);
        const uint32_t sum_smem = smem_u32(smem + L::kSums + t * L::kQSum), off_smem = smem_u32(smem + L::kOffsets);
        const uint32_t tS = tmem + t * 128, tO = tmem + 256 + t * 128;
        auto scores = [&](int j) {   // by one lane
          const uint64_t qd = sdesc_sw128(q_smem, 16, 1024), kd = sdesc_sw128(k_smem + (j % kStages) * L::kK, 16, 1024);
          const uint32_t to = tS + (j & 1) * kTokens;
          mma_f16_ss(to, sdesc_sw32(sum_smem), sdesc_sw32(off_smem + (j % kStages) * L::kKOff), id_s, 0u);
  #pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk)
            mma_f16_ss(to, qd + (uint64_t)(((kk >> 2) * (kTileRows * 128) + (kk & 3) * 32) >> 4),
                       kd + (uint64_t)(((kk >> 2) * (kTokens * 128) + (kk & 3) * 32) >> 4), id_s, 1u);
          mma_commit(&sfull[2 * t + (j & 1)]);
          mma_commit(&kempty[j % kStages]);
        };
        bool ok = true;
  #pragma unroll 1
        for (int j = 0; j < min(tiles, 2) && ok; ++j) {
          ok = mbar_wait_warp_lazy(&kfull[j], 0, ab, kErrK);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) scores(j);
          __syncwarp();
        }
  #pragma unroll 1
        for (int j = 0; j < tiles && ok; ++j) {
          const int vs = j % kStages;
          ok = mbar_wait_warp_lazy(&vfull[vs], (j / kStages) & 1, ab, kErrV);
          if (ok) ok = mbar_wait_warp_lazy(&pfull[2 * t + (j & 1)], (j >> 1) & 1, ab, kErrP);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t vd = sdesc_sw128(v_smem + vs * L::kV, 16, 1024);
  #pragma unroll
            for (int kk = 0; kk < kTokens / 16; ++kk)
              mma_f16_ts(tO, tS + (j & 1) * kTokens + kk * 8, vd + (uint64_t)((kk * 32) >> 4), id_pv, j > 0 || kk > 0 ? 1u : 0u);
            mma_commit(&pvdone[t]);
            mma_commit(&vempty[vs]);
          }
          __syncwarp();
          if (j + 2 < tiles) {
            ok = mbar_wait_warp_lazy(&kfull[(j + 2) % kStages], ((j + 2) / kStages) & 1, ab, kErrK);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) scores(j + 2);
            __syncwarp();
          }
        }
        if (elect_one()) mma_commit(&drain[t]);
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(&drain[t], 0)) {
          if (globaltimer_ns() - t0 > 2000000000ull) {
            if (a.status) atomicCAS(a.status, 0, kErrDrain);
            break;
          }
        }
        __syncwarp();
      }
    }
  }
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x < kCtaRows && blockIdx.y * kCtaRows + threadIdx.x < p.rows) {
    const float2 ml = reinterpret_cast<const float2*>(smem + L::kRows)[threadIdx.x];
    a.part_ml[((int64_t)blockIdx.x * a.c.heads + blockIdx.z) * p.rows + blockIdx.y * kCtaRows + threadIdx.x] =
        make_float2(ml.x, ml.y + reinterpret_cast<const float*>(smem + L::kPositions)[threadIdx.x]);
  }
  if (warp == kIssuer) tmem_dealloc(tmem, 512);
}

template <int DT, int DP>
int launch_prefix(const Kv4AttendArgs& a, int64_t rows, cudaStream_t s) {
  using L = PrefixLayout<DP>;
  auto kern = prefix_tc_kernel<DT, DP>;
  static std::atomic<uint64_t> allowed{0};
  const int rc = allow_shared(kern, L::kBytes, allowed, "kv4 prefix");
  if (rc) return rc;
  PrefixParams p{};
  p.a = a;
  p.rows = (int)rows;
  p.wait_ns = wait_limit_ns();
  const int64_t pairs = ceil_div(rows, kCtaRows);
  if (a.c.heads > 65535 || pairs > 65535) return set_error(SA_ERR_UNSUPPORTED, "kv4 prefix: grid too large");
  kern<<<dim3((unsigned)a.parts, (unsigned)pairs, (unsigned)a.c.heads), kPrefixThreads, L::kBytes, s>>>(p);
  return check_launch("kv4 prefix_tc_kernel");
}

}  // namespace

// From how many query rows of a key head on the tensor cores' tile of 128 rows pays behind prefixes
// of thousands of tokens; behind some hundreds warps with mma.sync stay ahead by up to 6 us a call,
// which the rule leaves.  One call with its tails and join, this kernel / warps with mma.sync, us, D 128, bf16:
//   prefix    key heads   16 rows       32 rows       64 rows       256 rows
//   500       8           18.4 / 14.4   17.2 / 18.5   18.5 / 20.5   24.7 / 22.7
//   500       1           16.4 / 12.3   16.4 / 12.4   16.5 / 14.4   20.5 / 14.8
//   4000      8           25.9 / 20.5   25.8 / 24.6   26.7 / 28.7   30.8 / 53.4
//   4000      1           20.5 / 18.5   20.5 / 20.4   20.5 / 20.5   23.0 / 24.6
//   32000     8           53.5 / 37.3   53.8 / 55.4   55.0 / 92.8   64.6 / 305
//   32000     1           28.7 / 24.6   28.7 / 26.7   28.7 / 32.8   33.2 / 52.2
// Float32 and widths above 128 have no form here (three pieces of either operand; O of two row tiles would not
// fit TMEM) and go to mma.sync whatever the rows: 64 requests of 32 heads over 8 behind 32000 tokens, float32 of
// width 128 539 us, bfloat16 of width 256 809, where bfloat16 of width 128 takes 72.
bool kv4_prefix_tc_takes(const Kv4AttendArgs& a, int64_t rows) {
  return a.dtype != SA_REP_FLOAT32 && a.c.dp <= 128 && rows > 32;
}

// Parts of the prefix, each a CTA for every pair of row tiles and key head: no more than
// fill the GPU, and no more than pay.  A tile takes 1 us, and a part 0.09 us of the join that
// reads it: tiles / parts + 0.09 parts is least at sqrt(11 tiles).  With a part of two tiles at
// least and no other limit, one key head took 44.1 us for 256 rows of a prefix of 32000, not 33.2.
// And no fewer than keep a chain of products short: the matrix units cut off what they add,
// 7e-8 of O for each 16 tokens, always to the same side, so a part is kChain tiles at most and what
// parts hold is added rounded.  (80 pairs, one part each, over 131072 / 500000 tokens of mean 1: float16
// results 8e-4 / 3e-3 low; so 1.6e-4 / 1.2e-4, and 10.4 / 37.6 ms, not 12.0 / 44.9.)
// Every query stands behind the prefix, so rows see no more of it than window and first tokens
// allow, however far apart they stand.
constexpr int kChain = 32768 / kTokens;

int kv4_prefix_tc_parts(const Kv4AttendArgs& a, int64_t rows) {
  const int64_t longest = std::min<int64_t>((int64_t)a.prefix_width << a.c.page_shift, a.window + a.sinks + a.n);
  const int64_t ctas = ceil_div(rows, kCtaRows) * a.c.heads, tiles = ceil_div(longest, kTokens);
  const int64_t pays = std::min(tiles, (int64_t)std::sqrt(11.0 * (double)tiles) + 1);
  return (int)std::max({(int64_t)1, std::min(148 / ctas, pays), ceil_div(tiles, kChain)});
}

int launch_kv4_prefix_tc(const Kv4AttendArgs& a, int64_t rows, cudaStream_t s) {
  const bool b = a.dtype == SA_REP_BFLOAT16;
  if (a.c.dp == 32) return b ? launch_prefix<SA_REP_BFLOAT16, 32>(a, rows, s) : launch_prefix<SA_REP_FLOAT16, 32>(a, rows, s);
  if (a.c.dp == 64) return b ? launch_prefix<SA_REP_BFLOAT16, 64>(a, rows, s) : launch_prefix<SA_REP_FLOAT16, 64>(a, rows, s);
  return b ? launch_prefix<SA_REP_BFLOAT16, 128>(a, rows, s) : launch_prefix<SA_REP_FLOAT16, 128>(a, rows, s);
}

}  // namespace sa
