// Attention of a request's newest tokens over its pages of the 4-bit cache.
// One kernel in five modes, each instantiated in a file of its own:
//   kPlain     all visible tokens (kv4_attend.cu)
//   kSelected  those of listed pages, another list for every query token and key head
//   kWeigh     kPlain that also leaves every score, maximum and sum for the weights
//   kPrefix    the queries of all requests over one shared prefix: unfinished sums
//   kTail      each request's own tokens, finished with the sums of its prefix
//
//   out = softmax over the visible tokens j of scale q.k_j, times v_j;
//   query i of n stands at position length - n + i; visible as in the windowed
//   attention (serving.cuh); nothing visible gives zeros.
//
// Bound by the cache's bytes (d / 2 + 4 of a key and of a value), so codes go
// from global memory to registers and from there to the matrix units, with no
// shared memory between (mma.sync m16n8k16: eight query rows fill its n, where
// a tcgen05 tile would hold 128 rows, nearly all empty).
//
// A warp takes blocks of 16 tokens.  A code's bits, moved to the top of a
// bfloat16's mantissa under the exponent of 16, are 16 + code: a shift and one
// logical operation for two codes, exact.  With x = least - 16 scale the value is
// s (16 + code) + x, so
//   S = s_k (K_codes Q^T) + x_k sum(Q)         tokens x rows
//   O = V_codes^T (p s_v)^T + sum(p x_v)       columns x rows
// with scales and offsets in float32 on either side of the products.
//
// Sums.  The matrix units truncate as they add, and over a long cache the output
// is small against its parts, whose mean cancels: with one chain of products over
// a request the error of nearly equal weights passed that of a float16 result's
// own rounding at 12000 tokens and reached 2 % at 131072.  So a block's products
// start from zero and are added to O outside, rounded; and where the result keeps
// more than 8 bits the codes of V are centred (16 + code less 24), which takes
// their mean out of the sums.  Nearly equal weights, 131072 / 1048576 tokens: an error
// of 1.7e-4 / 3.2e-4 not centred, which is little beside bfloat16's rounding (1.6e-3)
// and not beside float16's (2.1e-4); centred it does not show there.  Full batch as
// below: bfloat16 212 us with one chain, 228 so, 238 centred too; float16 247, 254,
// 262.  Float32 centres K as well and keeps the products of lower pieces apart.
//
// What bounds it beside the bytes (94 us of 64 requests x 6000..12000 tokens x 8
// heads, 611 MB) is instructions: 480 a block and 301 us with every code centred,
// masks in every block and register double buffers; 228 us now (2.7 TB/s; issue slots
// and integer pipe half busy, tensor pipe a fifth).  Float16 operands (five integer operations for eight codes in place of
// eight) took 245: their scales cost more than they saved.  Q is
// bfloat16 as it is, float16 as two and float32 as three bfloat16 pieces (exact,
// or to 24 bits); p s_v is split into two pieces (16 bits; three for float32).
//
// Fragments.  Lane (g = lane / 4, c = lane % 4).  Row r < 8 of the token axis is
// token 2 r of the block and row r + 8 token 2 r + 1: the cache keeps four
// tokens' bytes of a value column pair in one word, and that word is then a
// whole A fragment of V^T (tokens 4 c .. 4 c + 3, columns 2 b and 2 b + 1); a word
// of a key row is half the A fragments of two k steps, with the contraction's
// columns in the order of its nibbles (Q is loaded to match).  S comes out as
// tokens x rows and is turned by movmatrix for the second product.
//
// The visible blocks of a (request, key head) are dealt out to the warps of a
// cluster of CTAs, which join their maxima, sums and outputs through (distributed)
// shared memory in a fixed order: one launch, the same bits every time.
#pragma once

#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "kv4.cuh"

namespace sa {

namespace {

namespace cg = cooperative_groups;

enum Mode { kPlain, kSelected, kWeigh, kPrefix, kTail };

constexpr float kMove = 8.0f;     // how far a maximum may be passed before it is moved (base 2)
constexpr float kShift = -12.0f;  // p <= 2^-4: 2^16 values of 1e34 still sum below float32's limit

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Two codes, nibble i of each half of w, plus kOffset, as bfloat16.
template <int I, int kOffset>
__device__ __forceinline__ uint32_t codes(uint32_t w) {
  uint32_t x = I == 0 ? w << 3 : w >> (4 * I - 3);
  x = (x & 0x00780078u) | 0x41804180u;
  if (kOffset == -8) asm("add.rn.bf16x2 %0, %0, %1;" : "+r"(x) : "r"(0xc1c0c1c0u));   // - 24
  return x;
}

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same from a sum of zero.
__device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

__device__ __forceinline__ float2 params(uint32_t w) {   // scale, least
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// What a lane holds of one block.
template <int DP>
struct Block {
  static constexpr int kK = DP / 32;                  // words of one key row's share
  static constexpr int kV = DP / 16;                  // words of V: one a 16-column tile
  uint32_t k0[kK], k1[kK], v[kV];
  uint2 kp, vp;                                       // params of tokens 2 g and 2 g + 1
};

// Blocks on their way: each lane has a queue of kDepth slots of its own in shared
// memory, filled by cp.async and read by that lane alone (no barriers).  A slot's
// pieces of 16 (or 8, 4) bytes lie a warp's width apart.
constexpr int kDepth = 4;

template <int DP>
struct Queue {
  static constexpr int kPiece = DP >= 128 ? 16 : DP / 8;     // bytes of a key row's piece
  static constexpr int kPieces = (DP / 8) / kPiece;          // pieces of a key row's share
  static constexpr int kVPiece = DP >= 64 ? 16 : 8;
  static constexpr int kVPieces = (DP / 4) / kVPiece;
  static constexpr int kSlot = 32 * (2 * (DP / 8) + DP / 4 + 16);   // bytes of a warp's slot
};

template <int N>
__device__ __forceinline__ void copy_async(uint32_t to, const uint8_t* from) {
  if constexpr (N == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(N) : "memory");
}

template <int N>
__device__ __forceinline__ void take(uint32_t* x, const uint8_t* p) {
  if constexpr (N == 16) {
    const uint4 y = *reinterpret_cast<const uint4*>(p);
    x[0] = y.x;
    x[1] = y.y;
    x[2] = y.z;
    x[3] = y.w;
  } else if constexpr (N == 8) {
    const uint2 y = *reinterpret_cast<const uint2*>(p);
    x[0] = y.x;
    x[1] = y.y;
  } else {
    x[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// The addresses of a lane's share of the cache's first block.
struct Lanes {
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* kp;
  const uint8_t* vp;
};

// off: bytes of codes from there to the block, a multiple of 8 DP (params take
// off * 8 / DP bytes); slot: the warp's slot, lane: this lane.
template <int DP>
__device__ __forceinline__ void send_block(const Lanes& at, int64_t off, uint32_t slot, int lane) {
  using Q = Queue<DP>;
  uint32_t to = slot + lane * Q::kPiece;
#pragma unroll
  for (int row = 0; row < 2; ++row)
#pragma unroll
    for (int i = 0; i < Q::kPieces; ++i, to += 32 * Q::kPiece)
      copy_async<Q::kPiece>(to, at.k + off + row * (DP / 2) + i * Q::kPiece);
  to = slot + 32 * 2 * (DP / 8) + lane * Q::kVPiece;
  // 16-byte pieces of neighbouring lanes g are neighbours
#pragma unroll
  for (int i = 0; i < Q::kVPieces; ++i, to += 32 * Q::kVPiece) copy_async<Q::kVPiece>(to, at.v + off + i * 128);
  const int64_t poff = (int64_t)((uint64_t)off / (DP / 8));
  to = slot + 32 * (2 * (DP / 8) + DP / 4) + lane * 8;
  copy_async<8>(to, at.kp + poff);
  copy_async<8>(to + 32 * 8, at.vp + poff);
}

template <int DP>
__device__ __forceinline__ void take_block(Block<DP>& b, const uint8_t* slot, int lane) {
  using Q = Queue<DP>;
  const uint8_t* from = slot + lane * Q::kPiece;
#pragma unroll
  for (int i = 0; i < Q::kPieces; ++i, from += 32 * Q::kPiece) take<Q::kPiece>(b.k0 + i * Q::kPiece / 4, from);
#pragma unroll
  for (int i = 0; i < Q::kPieces; ++i, from += 32 * Q::kPiece) take<Q::kPiece>(b.k1 + i * Q::kPiece / 4, from);
  from = slot + 32 * 2 * (DP / 8) + lane * Q::kVPiece;
#pragma unroll
  for (int i = 0; i < Q::kVPieces; ++i, from += 32 * Q::kVPiece) take<Q::kVPiece>(b.v + i * Q::kVPiece / 4, from);
  from = slot + 32 * (2 * (DP / 8) + DP / 4) + lane * 8;
  b.kp = *reinterpret_cast<const uint2*>(from);
  b.vp = *reinterpret_cast<const uint2*>(from + 32 * 8);
}

// Byte column b of O's tile t (16 columns): lane g holds columns 2 b and 2 b + 1.
template <int DP>
__device__ __forceinline__ int byte_column(int t, int g) {
  return DP >= 64 ? (t >> 2) * 32 + g * 4 + (t & 3) : g * 2 + t;
}

template <int DT, int DP, int NT, int kWarps>
struct Shape {
  static constexpr int kQ = DT == SA_REP_BFLOAT16 ? 1 : (DT == SA_REP_FLOAT16 ? 2 : 3);   // pieces of q
  static constexpr int kP = DT == SA_REP_FLOAT32 ? 3 : 2;                                 // pieces of p s_v
  static constexpr int kRows = 8 * NT;
  // registers of O, Q and a block in a lane: where two CTAs an SM would spill, one
  static constexpr int kHeld = NT * (DP / 4 + kQ * DP / 8) + DP / 8;
  static constexpr int kPerSm = (kHeld <= 96 ? 2 : 1) * (8 / kWarps);
  static constexpr int kPitch = DP + 4;   // a row of O in shared memory
  // the queues, later the warps' O; then m, l and factors of warps (and CTAs), m, l
  static constexpr int kQueues = kWarps * kDepth * Queue<DP>::kSlot;
  static constexpr int kJoin = kWarps * kRows * kPitch * 4;
  static constexpr int kFirst = kQueues > kJoin ? kQueues : kJoin;
  static constexpr int kSmem = kFirst + (3 * kWarps * kRows + 2 * kRows) * 4;
};

// How many entries of a list of pages count: those before the first that lies outside
// the table or is not above the one before it (reported), or is -1.
template <int kThreads>
__device__ __forceinline__ int listed_pages(const Kv4AttendArgs& a, const int32_t* list, int* shared) {
  if (threadIdx.x == 0) *shared = a.count;
  __syncthreads();
  for (int e = threadIdx.x; e < a.count; e += kThreads) {
    const int x = __ldg(list + e);
    if (x < 0 || x >= a.width || (e > 0 && x <= __ldg(list + e - 1))) atomicMin(shared, e);
  }
  __syncthreads();
  const int n = *shared;
  if (threadIdx.x == 0 && n < a.count && __ldg(list + n) != -1) report(a.status, kBadList, __ldg(list + n));
  __syncthreads();
  return n;
}

template <int DT, int DP, int NT, int kMode, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, (Shape<DT, DP, NT, kWarps>::kPerSm)) attend_kernel(const Kv4AttendArgs a) {
  using T = typename Elem<DT>::T;
  using S = Shape<DT, DP, NT, kWarps>;
  constexpr int kThreads = kWarps * 32;
  // codes of K and V enter the products plus 16, or, where the sums need the bits, less 8
  // (the weights are float32, whatever the inputs)
  constexpr int kOff = DT == SA_REP_FLOAT32 || kMode == kWeigh ? -8 : 16;
  constexpr int kOffV = DT == SA_REP_BFLOAT16 ? 16 : -8;
  constexpr int kKS = DP / 16;   // k steps of the first product, 16-column tiles of the second
  if (kMode == kPrefix || kMode == kWeigh) next_may_start();
  extern __shared__ __align__(16) uint8_t smem[];
  float* sm_o = reinterpret_cast<float*>(smem);                // [warps][rows][pitch]
  float* sm_m = reinterpret_cast<float*>(smem + S::kFirst);    // [warps][rows]
  float* sm_l = sm_m + kWarps * S::kRows;
  float* sm_f = sm_l + kWarps * S::kRows;
  float* part_m = sm_f + kWarps * S::kRows;                    // [rows]: this CTA's
  float* part_l = part_m + S::kRows;

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, cc = lane & 3;
  const int group = a.heads / a.c.heads;
  // kSelected: a query token's heads are a problem of their own; kPrefix: all requests are one
  const int rows = kMode == kSelected ? group : kMode == kPrefix ? a.requests * a.n * group : a.n * group;
  const int tiles = (rows + S::kRows - 1) / S::kRows;
  const int hk = blockIdx.y / tiles, row0 = (blockIdx.y % tiles) * S::kRows;
  const int r = kMode == kSelected ? blockIdx.z / a.n : kMode == kPrefix ? 0 : blockIdx.z;
  const int splits = gridDim.x;

  const int cap = a.width << a.c.page_shift;
  int length = max(kMode == kPrefix ? a.prefix_length[0] : a.lengths[r], 0);
  if (length > cap && threadIdx.x == 0) report(a.status, kMode == kPrefix ? kBadPrefix : kBadLength, r);
  // as int: positions lie below 2^31 - 1, so differences of two are less than the largest
  const int window = (int)min(a.window, (int64_t)2147483647);
  int sinks = (int)min(a.sinks, (int64_t)2147483647);
  if (kMode == kTail) sinks = max(sinks - max(a.prefix_length[0], 0), 0);   // those that are no prefix tokens
  int listed = 0;
  const int32_t* list = nullptr;
  if (kMode == kSelected) {
    length -= a.n - 1 - (int)(blockIdx.z % a.n);   // up to this query
    list = a.pages + ((int64_t)blockIdx.z * a.c.heads + hk) * a.count;
    listed = listed_pages<kThreads>(a, list, reinterpret_cast<int*>(sm_f));
  }
  // positions of this tile's rows (rows behind the last count as the last); -1: sees nothing
  auto position = [&](int row) {
    if (kMode == kSelected) return length - 1;
    if (kMode == kPrefix) {
      const int x = min(row0 + row, rows - 1) / group, q = x / a.n;
      const int own = max(a.lengths[q], 0) - a.n + (x - q * a.n);   // only a request's own tokens ask
      return own < 0 ? -1 : (int)min((int64_t)length + own, (int64_t)2147483646);
    }
    return length - a.n + min(row0 + row, rows - 1) / group;
  };
  int p_lo, p_hi;   // least and largest position of the tile's rows
  KeyRanges kr;
  int held[NT][2];  // kPrefix: positions of this lane's rows
  if (kMode == kPrefix) {
    int least = 2147483647, most = -1, seen = 2147483647;   // seen: the least that sees anything
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int p = held[nt][e] = position(nt * 8 + 2 * cc + e);
        least = min(least, p);
        most = max(most, p);
        if (p >= 0) seen = min(seen, p);
      }
    p_lo = __reduce_min_sync(0xffffffffu, least);
    p_hi = __reduce_max_sync(0xffffffffu, most);
    kr = key_ranges(__reduce_min_sync(0xffffffffu, seen), p_hi, min(length, cap), a.window, a.sinks);
    if (p_hi < 0) kr = KeyRanges{0, 0, 0};
  } else {
    p_lo = position(0), p_hi = position(S::kRows - 1);
    if (kMode == kWeigh) p_lo = length - a.n, p_hi = length - 1;   // the same blocks for every tile of rows
    kr = key_ranges(p_lo, p_hi, min(length, cap), a.window, sinks);
  }
  const int sink_blocks = (int)((kr.first + 15) >> 4);
  const int win_begin = max((int)(kr.begin >> 4), sink_blocks), win_end = (int)((kr.end + 15) >> 4);
  const int page_blocks = a.c.page_shift - 4;   // log2 of a page's blocks
  const int blocks = kMode == kSelected ? listed << page_blocks : sink_blocks + max(win_end - win_begin, 0);
  const float sc = a.scale * 1.4426950408889634f;   // log2(e): scores in base 2

  // block u of this warp is block first + u * step of the visible ones
  const int parts = kMode == kPrefix ? gridDim.z : 1, part = kMode == kPrefix ? blockIdx.z : 0;
  const int first = (part * splits + blockIdx.x) * kWarps + warp, step = parts * splits * kWarps;
  const int mine = first < blocks ? (blocks - first + step - 1) / step : 0;
  auto token_of = [&](int u) {
    const int v = first + u * step;
    if (kMode == kSelected) return (__ldg(list + (v >> page_blocks)) << a.c.page_shift) + ((v & ((1 << page_blocks) - 1)) << 4);
    return (v < sink_blocks ? v : win_begin + v - sink_blocks) << 4;
  };
  const int32_t* table = kMode == kPrefix ? a.prefix_table : a.tables + (int64_t)r * a.width;
  // page ids of the next 32 blocks, one a lane
  int page_of = 0;
  auto fetch_pages = [&](int u0) {
    const int u = u0 + lane;
    const int token = u < mine ? token_of(u) : 0;
    page_of = u < mine ? __ldg(table + (token >> a.c.page_shift)) : 0;
    if (kMode == kSelected && token > p_hi) {
      page_of = -1;   // behind the query
    } else if (u < mine && (page_of < 0 || page_of >= a.c.pages)) {
      report(a.status, kBadPage, page_of);
      page_of = -1;   // its tokens count as hidden
    }
  };
  const int page_mask = (1 << a.c.page_shift) - 1;
  const int page_step = a.c.heads << a.c.page_shift;   // cells of a page, all heads
  const int64_t cell0 = (int64_t)hk << a.c.page_shift;
  const Lanes at{a.c.k_codes + (cell0 + 2 * g) * (DP / 2) + cc * (DP / 8),
                 a.c.v_codes + (cell0 + 4 * cc) * (DP / 2) + g * (DP >= 64 ? 16 : 8),
                 reinterpret_cast<const uint8_t*>(a.c.k_params + 2 * (cell0 + 2 * g)),
                 reinterpret_cast<const uint8_t*>(a.c.v_params + 2 * (cell0 + 2 * g))};
  uint8_t* queue = smem + warp * kDepth * Queue<DP>::kSlot;
  const uint32_t queue_u32 = static_cast<uint32_t>(__cvta_generic_to_shared(queue));
  uint32_t sent = 0;   // bit of a slot: a block is in it
  auto send = [&](int u) {
    const int slot = u % kDepth;
    sent &= ~(1u << slot);
    if (u < mine) {
      if ((u & 31) == 0) fetch_pages(u);
      const int page = __shfl_sync(0xffffffffu, page_of, u & 31);
      if (page >= 0) {
        send_block<DP>(at, ((int64_t)page * page_step + (token_of(u) & page_mask)) * (DP / 2),
                       queue_u32 + slot * Queue<DP>::kSlot, lane);
        sent |= 1u << slot;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // the first blocks come in under the queries' set-up
  for (int u = 0; u < kDepth - 1; ++u) send(u);

  // Q: fragments of this lane's row g (of each n tile) and the sums of the rows 2 cc, 2 cc + 1
  uint32_t qf[NT][S::kQ][kKS][2];
  float qsum[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = row0 + nt * 8 + g;
    const bool in = row < rows;
    const int x = in ? row / group : 0, h = hk * group + (in ? row - x * group : 0);
    const int i = kMode == kSelected ? (int)(blockIdx.z % a.n) : kMode == kPrefix ? x % a.n : x;
    const int64_t of = kMode == kPrefix ? x / a.n : r;
    const T* q = static_cast<const T*>(a.q) + of * a.q_r + i * a.q_n + h * a.q_h;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kKS / 2; ++w) {
      float x[8];
      const int col = cc * (DP / 4) + w * 8;
      if (in && a.vec_q && col + 8 <= a.c.d) {
        load8(x, q + col);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = in && col + e < a.c.d ? to_f32(q[col + e]) : 0.0f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += x[e];
#pragma unroll
      for (int s = 0; s < S::kQ; ++s) {
        float hi[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          hi[e] = __bfloat162float(__float2bfloat16_rn(x[e]));
          x[e] -= hi[e];
        }
        qf[nt][s][2 * w][0] = pack_bf16(hi[0], hi[4]);
        qf[nt][s][2 * w][1] = pack_bf16(hi[1], hi[5]);
        qf[nt][s][2 * w + 1][0] = pack_bf16(hi[2], hi[6]);
        qf[nt][s][2 * w + 1][1] = pack_bf16(hi[3], hi[7]);
      }
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);   // row g's sum, in its four lanes
    qsum[nt][0] = __shfl_sync(0xffffffffu, sum, 8 * cc);
    qsum[nt][1] = __shfl_sync(0xffffffffu, sum, 8 * cc + 4);
  }

  float o[NT][kKS][4];
  float m[NT][2], l[NT][2], z[NT][2];   // of rows 2 cc and 2 cc + 1
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int t = 0; t < kKS; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[nt][t][e] = 0.0f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      m[nt][e] = -INFINITY;
      l[nt][e] = z[nt][e] = 0.0f;
    }
  }

  // off: what is added to a score before 2^x; the maximum is moved where a score passes kMove + kShift
  float off[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) off[nt][0] = off[nt][1] = INFINITY;   // no maximum yet: the first score moves it

  const int bound = kMode == kPrefix ? min(length, cap) : cap;   // no token stands there or behind
  // float32: the scores' sums are kept apart by size
  constexpr bool kApart = DT == SA_REP_FLOAT32;
  auto work = [&](const Block<DP>& b, int token, int u, auto whole) {
    constexpr bool kWhole = decltype(whole)::value;   // every row sees the whole block
    float s[NT][4], low[NT][4];   // low: the products of Q's lower pieces, added at the end
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][e] = low[nt][e] = 0.0f;
#pragma unroll
    for (int w = 0; w < kKS / 2; ++w) {
      uint32_t f[2][4] = {{codes<0, kOff>(b.k0[w]), codes<0, kOff>(b.k1[w]), codes<1, kOff>(b.k0[w]), codes<1, kOff>(b.k1[w])},
                          {codes<2, kOff>(b.k0[w]), codes<2, kOff>(b.k1[w]), codes<3, kOff>(b.k0[w]), codes<3, kOff>(b.k1[w])}};
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int q = 0; q < S::kQ; ++q)
            mma(kApart && q > 0 ? low[nt] : s[nt], f[half][0], f[half][1], f[half][2], f[half][3], qf[nt][q][2 * w + half][0],
                qf[nt][q][2 * w + half][1]);
    }
    const float2 ka = params(b.kp.x), kb = params(b.kp.y), va = params(b.vp.x), vb = params(b.vp.y);
    const float k_s[2] = {ka.x * sc, kb.x * sc}, k_x[2] = {fmaf(-(float)kOff, ka.x, ka.y) * sc, fmaf(-(float)kOff, kb.x, kb.y) * sc};
    const float v_s[2] = {va.x, vb.x}, v_x[2] = {fmaf(-(float)kOffV, va.x, va.y), fmaf(-(float)kOffV, vb.x, vb.y)};
    uint32_t on = 0;   // bit 4 nt + e: s[nt][e] is seen
    if (!kWhole) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = token + 2 * g + (e >> 1), p = kMode == kPrefix ? held[nt][e & 1] : position(nt * 8 + 2 * cc + (e & 1));
          if (j <= p && (p - j < window || j < sinks) && j < bound) on |= 1u << (4 * nt + e);
        }
    }
    bool move = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (kApart) s[nt][e] += low[nt][e];
        s[nt][e] = fmaf(k_s[e >> 1], s[nt][e], k_x[e >> 1] * qsum[nt][e & 1]);
        if (!kWhole) s[nt][e] = (on >> (4 * nt + e)) & 1u ? s[nt][e] : -INFINITY;
        move |= s[nt][e] + off[nt][e & 1] > kMove + kShift;
      }
    if (kMode == kWeigh) {   // the scores, for the weights: rows 2 cc and 2 cc + 1 of tokens 2 g and 2 g + 1
      float* to = a.scores + (((int64_t)r * a.c.heads + hk) * a.score_blocks + first + (int64_t)u * step) * 16 * a.score_rows;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int row = row0 + nt * 8 + 2 * cc;
        if (row < rows) {
          *reinterpret_cast<float2*>(to + (2 * g) * a.score_rows + row) = make_float2(s[nt][0], s[nt][1]);
          *reinterpret_cast<float2*>(to + (2 * g + 1) * a.score_rows + row) = make_float2(s[nt][2], s[nt][3]);
        }
      }
    }
    if (__any_sync(0xffffffffu, move)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(s[nt][e], s[nt][e + 2]);
#pragma unroll
          for (int d = 4; d < 32; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          if (top > m[nt][e] + kMove) {
            const float alpha = ex2(m[nt][e] - top);   // from -inf: 0
            m[nt][e] = top;
            off[nt][e] = kShift - top;
            l[nt][e] *= alpha;
            z[nt][e] *= alpha;
#pragma unroll
            for (int t = 0; t < kKS; ++t) {
              o[nt][t][e] *= alpha;
              o[nt][t][e + 2] *= alpha;
            }
          }
        }
    }
    uint32_t pf[NT][S::kP][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float ps[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // without a maximum yet nothing has been seen: every score is -inf (or NaN)
        const float p = ex2(kWhole || m[nt][e & 1] != -INFINITY ? s[nt][e] + off[nt][e & 1] : s[nt][e]);
        const bool seen = kWhole || ((on >> (4 * nt + e)) & 1u);   // hidden tokens' scales may be anything
        l[nt][e & 1] += p;
        z[nt][e & 1] = seen ? fmaf(p, v_x[e >> 1], z[nt][e & 1]) : z[nt][e & 1];
        ps[e] = seen ? p * v_s[e >> 1] : 0.0f;
      }
#pragma unroll
      for (int q = 0; q < S::kP; ++q) {
        const uint32_t x = pack_bf16(ps[0], ps[1]), y = pack_bf16(ps[2], ps[3]);
        pf[nt][q][0] = transpose8(x);
        pf[nt][q][1] = transpose8(y);
        if (q + 1 < S::kP) {
          ps[0] -= __uint_as_float(x << 16);
          ps[1] -= __uint_as_float(x & 0xffff0000u);
          ps[2] -= __uint_as_float(y << 16);
          ps[3] -= __uint_as_float(y & 0xffff0000u);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < kKS; ++t) {
      const uint32_t w = b.v[t];
      const uint32_t a0 = codes<0, kOffV>(w), a1 = codes<1, kOffV>(w), a2 = codes<2, kOffV>(w), a3 = codes<3, kOffV>(w);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float sum[4];
        mma_first(sum, a0, a1, a2, a3, pf[nt][S::kP - 1][0], pf[nt][S::kP - 1][1]);
#pragma unroll
        for (int q = S::kP - 2; q >= 0; --q) mma(sum, a0, a1, a2, a3, pf[nt][q][0], pf[nt][q][1]);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][t][e] += sum[e];
      }
    }
  };
  auto go = [&](const Block<DP>& b, int token, int u) {
    if (token + 15 <= p_lo && (p_hi - token < window || token + 16 <= sinks) && (kMode != kPrefix || token + 16 <= bound))
      work(b, token, u, std::true_type{});
    else
      work(b, token, u, std::false_type{});
  };

  for (int u = 0; u < mine; ++u) {
    send(u + kDepth - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
    if ((sent >> (u % kDepth)) & 1u) {
      Block<DP> b;
      take_block<DP>(b, queue + (u % kDepth) * Queue<DP>::kSlot, lane);
      go(b, token_of(u), u);
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();   // the queues' memory takes the outputs

  // join the warps
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = l[nt][e], y = z[nt][e];
#pragma unroll
      for (int d = 4; d < 32; d *= 2) {
        x += __shfl_xor_sync(0xffffffffu, x, d);
        y += __shfl_xor_sync(0xffffffffu, y, d);
      }
      const int row = nt * 8 + 2 * cc + e;
      if (g == 0) {
        sm_m[warp * S::kRows + row] = m[nt][e];
        sm_l[warp * S::kRows + row] = x;
      }
      float* to = sm_o + (warp * S::kRows + row) * S::kPitch;
#pragma unroll
      for (int t = 0; t < kKS; ++t) {
        const int col = 2 * byte_column<DP>(t, g);
        *reinterpret_cast<float2*>(to + col) = make_float2(o[nt][t][e] + y, o[nt][t][e + 2] + y);
      }
    }
  __syncthreads();
  if (threadIdx.x < S::kRows) {   // what each warp's sums count for
    const int row = threadIdx.x;
    float top = -INFINITY, total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm_m[w * S::kRows + row]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float mw = sm_m[w * S::kRows + row];
      const float f = mw == -INFINITY ? 0.0f : ex2(mw - top);
      sm_f[w * S::kRows + row] = f;
      total = fmaf(f, sm_l[w * S::kRows + row], total);
    }
    part_m[row] = top;
    part_l[row] = total;
  }
  __syncthreads();
  // warp 0's place takes the CTA's: each thread a row's four columns, warps in order
  const int valid = min(S::kRows, rows - row0);
  for (int x = threadIdx.x; x < valid * (DP / 4); x += kThreads) {
    const int row = x / (DP / 4), col = (x - row * (DP / 4)) * 4;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = sm_f[w * S::kRows + row];
      const float4 y = *reinterpret_cast<const float4*>(sm_o + (w * S::kRows + row) * S::kPitch + col);
      sum.x = fmaf(f, y.x, sum.x);
      sum.y = fmaf(f, y.y, sum.y);
      sum.z = fmaf(f, y.z, sum.z);
      sum.w = fmaf(f, y.w, sum.w);
    }
    *reinterpret_cast<float4*>(sm_o + row * S::kPitch + col) = sum;
  }
  cg::cluster_group cluster = cg::this_cluster();
  if (splits > 1)
    cluster.sync();
  else
    __syncthreads();
  // and the cluster's CTAs, each a share of the rows' four columns (where a prefix's parts are read or written,
  // neighbouring threads take neighbouring rows, as they stand there)
  constexpr bool kParts = kMode == kPrefix || kMode == kTail;
  if (kMode == kTail) previous_has_ended();
  const int share = (valid * (DP / 4) + splits - 1) / splits, share_end = min((int)(blockIdx.x + 1) * share, valid * (DP / 4));
  for (int x = blockIdx.x * share + threadIdx.x; x < share_end; x += kThreads) {
    const int row = kParts ? x % valid : x / (DP / 4), col = (kParts ? x / valid : x - row * (DP / 4)) * 4;
    float top = -INFINITY, total = 0.0f;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    auto add = [&](float f, const float4& o) {
      sum[0] = fmaf(f, o.x, sum[0]);
      sum[1] = fmaf(f, o.y, sum[1]);
      sum[2] = fmaf(f, o.z, sum[2]);
      sum[3] = fmaf(f, o.w, sum[3]);
    };
    for (int s = 0; s < splits; ++s) top = fmaxf(top, splits > 1 ? *cluster.map_shared_rank(part_m + row, s) : part_m[row]);
    for (int s = 0; s < splits; ++s) {
      const float ms = splits > 1 ? *cluster.map_shared_rank(part_m + row, s) : part_m[row];
      const float ls = splits > 1 ? *cluster.map_shared_rank(part_l + row, s) : part_l[row];
      const float* from = sm_o + row * S::kPitch + col;
      const float4 os = *reinterpret_cast<const float4*>(splits > 1 ? cluster.map_shared_rank(from, s) : from);
      const float f = ms == -INFINITY ? 0.0f : ex2(ms - top);
      add(f, os);
      total = fmaf(f, ls, total);
    }
    if (kMode == kPrefix) {   // unfinished: kTail joins the parts
      const int64_t of = (int64_t)part * a.c.heads + hk;
      reinterpret_cast<float4*>(a.part_o)[(of * (DP / 4) + (col >> 2)) * rows + row0 + row] = make_float4(sum[0], sum[1], sum[2], sum[3]);
      if (col == 0) a.part_ml[of * rows + row0 + row] = make_float2(top, total);
      continue;
    }
    if (kMode == kTail) {   // the prefix's parts (in before this loop), in order, kBatch of them on their way at a time
      constexpr int kBatch = 6;
      const int64_t all = (int64_t)a.requests * rows, at = (int64_t)r * rows + row0 + row;
      const int64_t ml_step = a.c.heads * all, o_step = ml_step * (DP / 4);
      const float2* from_ml = a.part_ml + hk * all + at;
      const float4* from_o = reinterpret_cast<const float4*>(a.part_o) + (hk * (DP / 4) + (col >> 2)) * all + at;
      for (int s0 = 0; s0 < a.parts; s0 += kBatch, from_ml += kBatch * ml_step, from_o += kBatch * o_step) {
        float2 ml[kBatch];
        float4 o[kBatch];
        float next = top;
#pragma unroll
        for (int s = 0; s < kBatch; ++s) {
          ml[s] = s0 + s < a.parts ? from_ml[s * ml_step] : make_float2(-INFINITY, 0.0f);
          o[s] = s0 + s < a.parts ? from_o[s * o_step] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int s = 0; s < kBatch; ++s) next = fmaxf(next, ml[s].x);
        const float f = top == -INFINITY ? 1.0f : ex2(top - next);   // nothing yet: zeros, or NaN that stays
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] *= f;
        total *= f;
#pragma unroll
        for (int s = 0; s < kBatch; ++s) {
          const float g = ml[s].x == -INFINITY ? 1.0f : ex2(ml[s].x - next);
          add(g, o[s]);
          total = fmaf(g, ml[s].y, total);
        }
        top = next;
      }
    }
    const int i = kMode == kSelected ? (int)(blockIdx.z % a.n) : (row0 + row) / group;
    const int h = hk * group + row0 + row - (kMode == kSelected ? 0 : i * group);
    T* out = static_cast<T*>(a.out) + (((int64_t)r * a.n + i) * a.heads + h) * a.c.d + col;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < a.c.d) out[e] = from_f32<T>(total == 0.0f ? 0.0f : sum[e] / total);
    // p = 2^(s + kShift - top) / total
    if (kMode == kWeigh && col == 0)
      a.score_ml[((int64_t)r * a.c.heads + hk) * a.score_rows + row0 + row] =
          make_float2(kShift - top, total == 0.0f ? 0.0f : 1.0f / total);
  }
  if (splits > 1) cluster.sync();   // nobody leaves while its shared memory is read
}

// Query rows of a key head, in one problem of the mode.
template <int kMode>
int64_t rows_of(const Kv4AttendArgs& a) {
  const int64_t group = a.heads / a.c.heads;
  return kMode == kSelected ? group : kMode == kPrefix ? a.requests * a.n * group : a.n * group;
}

template <int DT, int DP, int NT, int kMode, int kWarps = kMode == kPlain ? 8 : 4>
int launch_one(const Kv4AttendArgs& a, cudaStream_t s) {
  using S = Shape<DT, DP, NT, kWarps>;
  auto kern = attend_kernel<DT, DP, NT, kMode, kWarps>;
  static std::atomic<uint64_t> allowed{0};
  const int rc = allow_shared(kern, S::kSmem, allowed, "kv4 attend");
  if (rc) return rc;
  const int64_t y = a.c.heads * ceil_div(rows_of<kMode>(a), S::kRows);
  const int64_t z = kMode == kSelected ? (int64_t)a.requests * a.n : kMode == kPrefix ? a.parts : a.requests;
  if (y > 65535 || z > 65535) return set_error(SA_ERR_UNSUPPORTED, "kv4 attend: grid too large");
  const int64_t held = (int64_t)(kMode == kSelected ? std::min(a.count, a.width) : a.width) << a.c.page_shift;
  const int64_t longest = std::min<int64_t>(held, a.window + a.sinks + a.n);
  int splits = 1;   // CTAs per (request, key head)
  if (kMode == kPlain) {
    // while a warp keeps at least four blocks of the longest request the table allows, of
    // what window and first tokens show of it (8192 first tokens and a window of 64 of one
    // request: 65 us as one CTA, 20 as eight), and the grid has less than three rounds (the
    // batch above as it was at 212 us: 232 with six, 231 with one)
    while (splits < 8 && longest >= (int64_t)splits * 2 * kWarps * 16 * 4 && y * z * splits < 148 * S::kPerSm * 3) splits *= 2;
  } else {
    // while all run at once and a warp has half a block, or, in less than three rounds, it
    // keeps 32 (48 requests x 8 heads x 2048 selected tokens: 57 us as one, 64 as two, 70 as
    // four; three queries x 4 heads over 800: 16, 14, 12, 10 as eight; 32 requests of 10000
    // tokens with weights: 196, 158, 150, 154)
    auto more = [&](int64_t blocks, int64_t ctas) {
      return splits < 8 && 2 * longest >= splits * 2 * kWarps * 16 * blocks && y * z * splits * 2 <= ctas;
    };
    while (more(1, 148 * S::kPerSm) || more(64, 148 * S::kPerSm * 3)) splits *= 2;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)splits, (unsigned)y, (unsigned)z);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (splits > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = (unsigned)splits;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  if (kMode == kTail) {   // its launch, and its own tokens on SMs without a CTA of the prefix, beside that kernel
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
  if (e != cudaSuccess) return set_error(SA_ERR_CUDA, "kv4 attend_kernel: %s", cudaGetErrorString(e));
  return check_launch("kv4 attend_kernel");
}

// Two tiles of eight rows where the registers hold them and there are that many rows.
template <int DT, int DP, int kMode>
int launch_rows(const Kv4AttendArgs& a, cudaStream_t s) {
  if constexpr (DT != SA_REP_FLOAT32 && DP <= 128)
    if (rows_of<kMode>(a) > 8) return launch_one<DT, DP, 2, kMode>(a, s);
  return launch_one<DT, DP, 1, kMode>(a, s);
}

template <int DT, int kMode>
int launch_dim(const Kv4AttendArgs& a, cudaStream_t s) {
  if (a.c.dp == 32) return launch_rows<DT, 32, kMode>(a, s);
  if (a.c.dp == 64) return launch_rows<DT, 64, kMode>(a, s);
  if (a.c.dp == 128) return launch_rows<DT, 128, kMode>(a, s);
  return launch_rows<DT, 256, kMode>(a, s);
}

template <int kMode>
int launch_mode(const Kv4AttendArgs& a, cudaStream_t s) {
  if (a.dtype == SA_REP_FLOAT32) return launch_dim<SA_REP_FLOAT32, kMode>(a, s);
  if (a.dtype == SA_REP_FLOAT16) return launch_dim<SA_REP_FLOAT16, kMode>(a, s);
  return launch_dim<SA_REP_BFLOAT16, kMode>(a, s);
}

}  // namespace

}  // namespace sa
