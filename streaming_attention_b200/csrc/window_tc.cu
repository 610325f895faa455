// Attention with a sliding window and first tokens that stay visible, on the
// 5th-generation tensor cores (tcgen05 kind::f16, TMEM, TMA): float16 and
// bfloat16, head widths up to 128.
//
//   out_i = sum_j softmax_j(scale q_i.k_j) v_j,  j <= p_i and (j > p_i - window or j < sinks)
//
// Rows.  A query tile is 128 rows of S = Q K^T: 128 / G queries times G query
// heads of one key head (G the largest power of two that divides the group, up
// to 32), so that grouped heads share their key tiles and one new token of a
// group fills G rows.  A CTA holds two query tiles of consecutive queries.
//
// Columns.  The keys that a CTA's queries see are the first tokens [0, first)
// and the window [begin, end).  They are laid side by side on a virtual axis:
// columns 0 .. F - 1 are the first tokens (F = first rounded up to 16), column
// V >= F is key begin + V - F.  Tiles of 128 columns; the one that holds the
// seam is loaded in 16-row boxes, the others in one.  On that axis
//   visible(V) = V <= hi and (V >= hi - window + 1 or V < sk),  hi = p - begin + F
// with sk = first (the filling columns lie below every row's window), or, where
// window and first tokens touch, F = begin = 0 and sk = sinks.
//
// One CTA per SM works through query tile pairs (persistent: a pair's set-up,
// first loads and stores run under its neighbours' products; as one CTA per pair
// they took 40 % of the time).  Warps: 0 plans the pairs and loads (TMA), 1 and 2
// issue the products of query tile 0 and 1 (converged, one elected lane), 3..6
// and 7..10 are their softmax, one row per thread, a tile's 64 scores in
// registers (more, of 128 columns, spilled: beside 220 KB of shared memory that
// goes to L2).  TMEM: of each query tile two S of 64 columns and O of 128; P, in 16
// bits, overwrites the first half of its S.  A tile's issuer goes P V(j), S(j + 2),
// so that the next scores are there while a softmax runs (their commit says too
// that P V(j) has ended; one without scores behind it has a barrier of its own,
// since a parity wait must have seen each phase of its barrier before the next
// ends: scores' commits are all answered by a P, these by a later one); with one S of 128
// columns each waited for the other (32 heads x 8192 of 128, window 1024: 184 us, and
// 174 so, back to back; 188 us of a caller's time with cold caches, 129 GFLOP, 41 % of
// the measured GEMM rate; bound by that chain: tensor pipe and exponentials 40 % each).
//
// Where a dense call has few pairs and many keys, a pair's key tiles are dealt
// into parts that run as items of their own and are joined by join_kernel.
//
// Softmax in base 2 with a lazily moved maximum: m follows a tile's maximum
// only when that is more than kMove above it, so O is scaled rarely.  P is
// 2^(x - m + kShift): bfloat16 takes kShift = -24 (float32's range, so that
// 2^16 of the largest values still sum below float32's limit), float16 +6 (at
// most 2^14, and 2^-14, where float16 starts to lose bits, is 2^-20 of the
// row's usual largest).
//
// The matrix units truncate as they add, so a chain of products pulls O towards
// zero by up to 7e-8 of it a step of 16 keys: values of mean 1 came out 5.5e-4 low
// after 131072 keys.  Given a workspace, O goes to a sum in memory every kFold
// tiles (32768 keys, at most 1.4e-4) and starts from zero again.
//
// A product with a hidden key's value is 0 * v, NaN where v is NaN or infinite.
// Columns that come out non-finite are computed again by the row's warp from the
// visible keys alone (repair_row): what a query does not see cannot reach it.
// The bounded waits of the CTA's other warps are renewed as long as that goes on.
#include <cuda.h>
#include <math.h>

#include <algorithm>

#include "serving.cuh"
#include "tc_util.cuh"
#include "window_row.cuh"

namespace sa {

namespace {

using namespace tc;

constexpr int kRows = 128;     // rows of a query tile
constexpr int kCols = 64;      // keys of a key tile
constexpr int kSeam = 16;      // rows of a box of the seam tile
constexpr int kThreads = 352;
constexpr int kFold = 512;     // key tiles of a chain of products, where there is a workspace
constexpr int kFoldCtas = 148;
constexpr float kMove = 8.0f;

constexpr int kErrQ = 501, kErrFull = 502, kErrP = 503, kErrS = 504, kErrEmpty = 505, kErrO = 506, kErrDrain = 507,
              kErrPlan = 508;

struct WindowTcParams {
  WindowArgs a;
  int group, pack, blocks;   // query heads per key head, heads per tile, tiles of heads per key head
  int pack_log;              // pack = 1 << pack_log
  int rows_per_cta;          // queries of a CTA (2 * kRows / pack)
  int vec_out;               // out rows take 16-byte stores
  uint32_t tiles, items;     // query tile pairs of one tile of heads, and work items (pairs times splits) of all
  int splits;                // parts that a pair's keys are dealt into
  float* part;               // splits > 1: [row][split][pitch], O (not divided), m, l
  int pitch;
  float* sums;               // kLong: [cta][query tile][dv + 1][row], folded O and the maximum it goes by
  uint64_t wait_ns;
};

// Columns of one CTA on the virtual axis.
struct Columns {
  int first, fill, total;   // first tokens, rounded up to 16, all columns
  int sk;
  int64_t begin;
};

__device__ __forceinline__ Columns columns_of(int64_t p0, int64_t p1, int64_t m, int64_t window, int64_t sinks) {
  const KeyRanges r = key_ranges(p0, p1, m, window, sinks);
  Columns c;
  if (sinks >= r.begin) {
    c.first = c.fill = 0;
    c.begin = 0;
    c.sk = (int)min(sinks, (int64_t)2147483647);
  } else {
    c.first = (int)r.first;
    c.fill = (c.first + kSeam - 1) / kSeam * kSeam;
    c.begin = r.begin;
    c.sk = c.first;
  }
  c.total = (int)(r.end - c.begin) + c.fill;
  return c;
}

// A query tile pair, in shared memory: each role reads what it needs, so that
// nothing of it takes registers (or, worse, local memory) where it is not used.
struct PairPlan {
  int live;        // 0: no queries (skipped), -1: no pairs are left
  int b, hk, g0;   // request, key head, first query head of the tile within the group
  int q_row, nq;   // first query's row in q, queries
  int k_row, m;    // first key's row in k, keys of the request
  int p0;          // position of the first query
  int j0, tiles;   // first key tile, key tiles
  int split;
  int total, fill, sk;
  int base;        // column V >= fill is row base + V of k
  int hi;          // hi of the first query; query i's is hi + i
  int lo[2], last[2];   // columns that query tile t needs: lo[t] (or below sk) .. last[t]
};

__device__ __forceinline__ PairPlan plan_pair(const WindowTcParams& p, uint32_t item) {
  const WindowArgs& a = p.a;
  PairPlan c;
  const uint32_t whole = item / (uint32_t)p.splits;
  c.split = (int)(item - whole * p.splits);
  item = whole;
  const uint32_t y = item / p.tiles;
  int64_t tile;
  c.b = tile_request(a, item - y * p.tiles, p.rows_per_cta, &tile);
  const Request rq = request_of(a, c.b);
  const int64_t i0 = tile * p.rows_per_cta;
  c.live = tile >= 0 && i0 < rq.n;
  c.hk = y / p.blocks;
  c.g0 = (y % p.blocks) * p.pack;
  c.q_row = (int)(rq.q0 + i0);
  c.nq = (int)min((int64_t)p.rows_per_cta, rq.n - i0);
  c.k_row = (int)rq.k0;
  c.m = (int)rq.m;
  const int64_t p0 = rq.m - rq.n + i0;
  c.p0 = (int)p0;
  const Columns cols = columns_of(p0, p0 + c.nq - 1, rq.m, a.window, a.sinks);
  const int64_t all = (cols.total + kCols - 1) / kCols;
  c.j0 = (int)(all * c.split / p.splits);
  c.tiles = (int)(all * (c.split + 1) / p.splits) - c.j0;
  c.total = cols.total;
  c.fill = cols.fill;
  c.sk = cols.sk;
  c.base = (int)(rq.k0 + cols.begin) - cols.fill;
  c.hi = (int)(p0 - cols.begin) + cols.fill;
  const int tq = kRows >> p.pack_log, window = (int)min(a.window, (int64_t)1 << 30);
  c.last[0] = c.hi + min(tq, c.nq) - 1;
  c.last[1] = c.nq > tq ? c.hi + c.nq - 1 : -1;
  c.lo[0] = c.hi - window + 1;
  c.lo[1] = c.lo[0] + tq;
  return c;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Ties 32 loaded registers to this point of the program: what follows uses them
// after the wait that stands before.
__device__ __forceinline__ void tie32(float (&v)[32]) {
  asm volatile("" : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
               "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]));
  asm volatile("" : "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]),
               "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]),
               "+f"(v[31]));
}

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

// Two floats as 16-bit values, the first in the low half.
template <int DT>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if (DT == SA_REP_BFLOAT16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// The x lowest bits set (x may be anything).
__device__ __forceinline__ uint32_t low_bits(int x) {
  return x >= 32 ? 0xffffffffu : (x <= 0 ? 0u : (1u << x) - 1u);
}

// Hidden scores (bit 0) become -inf.
__device__ __forceinline__ void hide(float (&s)[32], uint32_t on) {
#pragma unroll
  for (int e = 0; e < 32; ++e) s[e] = (on >> e) & 1u ? s[e] : -INFINITY;
}

__device__ __forceinline__ float max32(const float (&s)[32]) {
  float t[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
  for (int e = 4; e < 32; ++e) t[e & 3] = fmaxf(t[e & 3], s[e]);
  return fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
}

// P of a chunk: 2^(s c2 + off), summed and, in 16 bits, stored to TMEM.  (A third
// of the exponentials as a polynomial on the FMA pipe, which a loop of softmax
// alone gains 15 % from, cost 3 % here: the loop waits more than it computes.)
template <int DT>
__device__ __forceinline__ void exp_chunk(float (&s)[32], uint64_t c22, uint64_t off2, uint64_t (&sum2)[2], uint32_t to) {
  uint32_t pk[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    float x, y;
    unpack2(fma2(pack2(s[2 * e], s[2 * e + 1]), c22, off2), x, y);
    x = ex2(x);
    y = ex2(y);
    sum2[e & 1] = add2(sum2[e & 1], pack2(x, y));
    pk[e] = pack16<DT>(x, y);
  }
  tmem_st16(to, pk);
}

// O of a row times alpha, in TMEM (rare: kept out of the way of the tile loop's code).
__device__ __noinline__ void scale_row(uint32_t to, int dv, float alpha) {
#pragma unroll 1
  for (int c = 0; c < dv; c += 16) {
    float o[16];
    tmem_ld16(to + c, o);
    tmem_wait_ld();
    uint32_t os[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) os[e] = __float_as_uint(o[e] * alpha);
    tmem_st16(to + c, os);
  }
  tmem_wait_st();
}

// A row's place in the folded sums: columns kRows apart, behind them the maximum
// that they go by.  (All from the thread's index: called rarely, it takes no registers elsewhere.)
__device__ __forceinline__ float* sums_of(float* sums, int dv) {
  const int warp = threadIdx.x >> 5, t = (warp - 3) >> 2;
  return sums + ((blockIdx.x * 2 + t) * (dv + 1)) * kRows + (warp & 3) * 32 + (threadIdx.x & 31);
}

// O of a row, in TMEM, times alpha; then, with `fold`, into its sum, and zero there.
__device__ __noinline__ void scale_fold_row(uint32_t to, int dv, float alpha, float m, float* sums, bool fold, bool first) {
  float* at = sums_of(sums, dv);
  const float before = first || !fold ? -INFINITY : at[dv * kRows];
  const float f = before == -INFINITY ? 0.0f : ex2(before - m);
#pragma unroll 1
  for (int c = 0; c < dv; c += 16) {
    float o[16];
    tmem_ld16(to + c, o);
    tmem_wait_ld();
    uint32_t os[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      o[e] *= alpha;
      os[e] = fold ? 0u : __float_as_uint(o[e]);
      if (fold && c + e < dv) at[(c + e) * kRows] = before == -INFINITY ? o[e] : fmaf(f, at[(c + e) * kRows], o[e]);
    }
    tmem_st16(to + c, os);
  }
  tmem_wait_st();
  if (fold) at[dv * kRows] = m;
}

// The sum of a row back to its O in TMEM.
__device__ __noinline__ void unfold_row(uint32_t to, int dv, float m, float* sums) {
  const float* at = sums_of(sums, dv);
  const float before = at[dv * kRows], f = before == -INFINITY ? 0.0f : ex2(before - m);
#pragma unroll 1
  for (int c = 0; c < dv; c += 16) {
    float o[16];
    tmem_ld16(to + c, o);
    tmem_wait_ld();
    uint32_t os[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) os[e] = __float_as_uint(c + e < dv ? fmaf(f, at[(c + e) * kRows], o[e]) : 0.0f);
    tmem_st16(to + c, os);
  }
  tmem_wait_st();
}

template <int DC, int VC>   // 64-column chunks of the head widths
struct Layout {
  static constexpr uint32_t kQ = DC * kRows * 128;                              // one query tile
  static constexpr uint32_t kTile = (DC > VC ? DC : VC) * kCols * 128;          // one K or V tile
  static constexpr uint32_t kSlot = 2 * kTile;                                  // a group of the ring
  static constexpr int kSlots = DC == 2 || VC == 2 ? 4 : 8;
  static constexpr uint32_t kRing = 2 * kQ;
  static constexpr uint32_t kPitch = 80;                                        // a row's 32 columns, staged
  static constexpr uint32_t kStage = kRing + kSlots * kSlot;
  static constexpr uint32_t kBars = kStage + 8 * 32 * kPitch;
  static constexpr uint32_t kBytes = kBars + (2 * kSlots + 20) * 8 + 16 + 2 * sizeof(PairPlan) + 1024;
  static_assert(kBytes <= 227 * 1024, "shared memory");
};

template <int DT, int DC, int VC, bool kLong>   // kLong: chains are folded (the code costs the others registers)
__global__ void __launch_bounds__(kThreads, 1)
window_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_ks, const __grid_constant__ CUtensorMap tm_kw,
                 const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_vs,
                 const __grid_constant__ CUtensorMap tm_vw, const __grid_constant__ WindowTcParams p) {
  using L = Layout<DC, VC>;
  using T = typename Elem<DT>::T;
  constexpr int kSlots = L::kSlots;
  constexpr float kShift = DT == SA_REP_BFLOAT16 ? -24.0f : 6.0f;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t* empty = full + kSlots;
  uint64_t* sfull = empty + kSlots;   // [2 query tiles][2 score buffers]
  uint64_t* pfull = sfull + 4;        // likewise
  uint64_t* ofull = pfull + 4;        // likewise: a P V that no scores follow in its buffer has ended
  uint64_t* qfull = ofull + 4;
  uint64_t* qempty = qfull + 1;
  uint64_t* plan_full = qempty + 1;       // [2]
  uint64_t* plan_empty = plan_full + 2;   // [2]
  uint64_t* drain = plan_empty + 2;       // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  int* abort_word = reinterpret_cast<int*>(tmem_slot + 1);
  PairPlan* plans = reinterpret_cast<PairPlan*>(tmem_slot + 4);   // [2]

  const WindowArgs& a = p.a;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 2);   // both issuers
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sfull[i], 1);
      mbar_init(&pfull[i], 4);
      mbar_init(&ofull[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&plan_full[i], 1);
      mbar_init(&plan_empty[i], 10);   // two issuers and eight softmax warps
      mbar_init(&drain[i], 1);
    }
    mbar_init(qfull, 1);
    mbar_init(qempty, 2);
    abort_word[0] = abort_word[1] = 0;   // [1] counts on while a warp repairs rows
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const Abort ab{abort_word, a.status, p.wait_ns, true};
  const uint32_t tS[2] = {tmem, tmem + 128}, tO[2] = {tmem + 256, tmem + 384};

  if (warp == 0) {
    // ------------------------------------------------------------ plans and loads
    if (lane == 0) {
      int u = 0, pairs = 0;   // ring loads and pairs so far
      bool ok = true;
#pragma unroll 1
      for (uint32_t item = blockIdx.x; ok; item += gridDim.x) {
        PairPlan c;
        c.live = -1;
        if (item < p.items) c = plan_pair(p, item);
        if (c.live == 0) continue;
        const int ps = pairs & 1;
        if (pairs >= 2 && !mbar_wait(&plan_empty[ps], ((pairs >> 1) - 1) & 1, ab, kErrPlan)) break;
        plans[ps] = c;
        mbar_arrive(&plan_full[ps]);
        if (c.live < 0) break;
        if (pairs >= 1 && !mbar_wait(qempty, (pairs - 1) & 1, ab, kErrEmpty)) break;
        ++pairs;
        const int kb = a.cu_q ? 0 : c.b, tq = kRows >> p.pack_log;
        if (c.tiles > 0) {
          mbar_arrive_expect_tx(qfull, 2 * L::kQ);
          for (int t = 0; t < 2; ++t)
            for (int j = 0; j < DC; ++j)
              tma_load_5d(smem + t * L::kQ + j * (kRows * 128), &tm_q, qfull, j * 64, c.g0, c.q_row + t * tq, c.hk, kb);
        } else {
          mbar_arrive(qfull);
        }
        // group 0: K of tiles 0 and 1; group g: V of tile g - 1 and K of tile g + 1
#pragma unroll 1
        for (int g = 0; c.tiles > 0 && g <= c.tiles; ++g, ++u) {
          const int s = u % kSlots;
          if (u >= kSlots && !mbar_wait(&empty[s], ((u / kSlots) - 1) & 1, ab, kErrEmpty)) {
            ok = false;
            break;
          }
          const int second = g == 0 ? 1 : g + 1;   // the key tile of the second half, if there is one
          const bool two = second < c.tiles;
          mbar_arrive_expect_tx(&full[s], ((g == 0 ? DC : VC) + (two ? DC : 0)) * kCols * 128);
#pragma unroll 1
          for (int half = 0; half < (two ? 2 : 1); ++half) {
            const bool isv = g > 0 && half == 0;
            const int v0 = (c.j0 + (half ? second : (g == 0 ? 0 : g - 1))) * kCols;
            uint8_t* dst = smem + L::kRing + s * L::kSlot + half * L::kTile;
#pragma unroll 1
            for (int j = 0; j < (isv ? VC : DC); ++j, dst += kCols * 128) {
              if (v0 >= c.fill) {
                tma_load_4d(dst, isv ? &tm_v : &tm_k, &full[s], j * 64, c.base + v0, c.hk, kb);
              } else if (c.fill == kSeam) {
                tma_load_4d(dst, isv ? &tm_vs : &tm_ks, &full[s], j * 64, c.k_row, c.hk, kb);
                tma_load_4d(dst + kSeam * 128, isv ? &tm_vw : &tm_kw, &full[s], j * 64, c.base + kSeam, c.hk, kb);
              } else {
#pragma unroll 1
                for (int r = 0; r < kCols; r += kSeam) {
                  const int v = v0 + r;
                  tma_load_4d(dst + r * 128, isv ? &tm_vs : &tm_ks, &full[s], j * 64,
                              v < c.fill ? c.k_row + v : c.base + v, c.hk, kb);
                }
              }
            }
          }
        }
      }
      // never leave with copies in flight
      for (int i = max(0, u - kSlots); i <= u; ++i) {
        if (i == u && pairs == 0) break;
        uint64_t* bar = i < u ? &full[i % kSlots] : qfull;
        const int parity = i < u ? (i / kSlots) & 1 : (pairs - 1) & 1;
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(bar, parity)) {
          if (globaltimer_ns() - t0 > 1000000000ull) {
            if (a.status) atomicCAS(a.status, 0, kErrDrain);
            break;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp <= 2) {
    // ------------------------------------------------------------ products of query tile t
    const int ksteps = (a.d + 15) >> 4;
    const uint32_t id_pv = idesc_f16(kRows, (a.dv + 15) & ~15, DT == SA_REP_BFLOAT16, false, true);
    const int t = warp - 1;
    const uint32_t q_smem = smem_u32(smem + t * L::kQ), ring = smem_u32(smem + L::kRing);
    int u = 0;                 // ring groups before this pair
    int count_p[2] = {0, 0};   // P tiles waited for in each buffer
    bool ok = true;
#pragma unroll 1
    for (int pair = 0; ok; ++pair) {
      ok = mbar_wait_warp_lazy(&plan_full[pair & 1], (pair >> 1) & 1, ab, kErrPlan);
      if (!ok) break;
      const PairPlan& c = plans[pair & 1];
      if (c.live < 0) break;
      const int tiles = c.tiles, total = c.total, sk = c.sk, lo = c.lo[t], last = c.last[t];
      const int start = c.j0 * kCols;
      auto needed = [&](int j) {
        const int v = start + j * kCols;
        return v <= last && (v + kCols > lo || v < sk);
      };
      // columns of tile j that a product takes: a multiple of 32
      auto width = [&](int j) { return min(kCols, (total - start - j * kCols + 31) & ~31); };
      // S of tile j into buffer j & 1 (called by one lane)
      auto scores = [&](int j) {
        const int group = u + (j < 2 ? 0 : j - 1);
        const uint64_t qd = sdesc_sw128(q_smem, 16, 1024);
        const uint64_t kd = sdesc_sw128(ring + (group % kSlots) * L::kSlot + (j == 0 ? 0 : L::kTile), 16, 1024);
        const uint32_t id_s = idesc_f16(kRows, width(j), DT == SA_REP_BFLOAT16, false, false);
        const uint32_t to = tS[t] + (j & 1) * kCols;
        // unrolled: descriptors that are constants apart stay in uniform registers
#pragma unroll
        for (int kk = 0; kk < DC * 4; ++kk)
          if (kk < ksteps)
            mma_f16_ss(to, qd + (uint64_t)(((kk >> 2) * (kRows * 128) + (kk & 3) * 32) >> 4),
                       kd + (uint64_t)(((kk >> 2) * (kCols * 128) + (kk & 3) * 32) >> 4), id_s, kk > 0 ? 1u : 0u);
      };
      __syncwarp();
      if (lane == 0) mbar_arrive(&plan_empty[pair & 1]);
      ok = mbar_wait_warp_lazy(qfull, pair & 1, ab, kErrQ);
      if (ok && tiles > 0) ok = mbar_wait_warp_lazy(&full[u % kSlots], (u / kSlots) & 1, ab, kErrFull);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll 1
        for (int j = 0; j < min(tiles, 2); ++j)
          if (needed(j)) {
            scores(j);
            mma_commit(&sfull[2 * t + j]);
          }
        if (tiles > 0) mma_commit(&empty[u % kSlots]);
        if (tiles <= 2) mma_commit(qempty);
      }
      __syncwarp();
      bool begun = false;
#pragma unroll 1
      for (int j = 0; j < tiles; ++j) {
        const int group = u + j + 1, buf = j & 1;
        const bool pv = needed(j), next = j + 2 < tiles && needed(j + 2);
        ok = mbar_wait_warp_lazy(&full[group % kSlots], (group / kSlots) & 1, ab, kErrFull);
        if (ok && pv) {
          ok = mbar_wait_warp_lazy(&pfull[2 * t + buf], count_p[buf] & 1, ab, kErrP);
          ++count_p[buf];
        }
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          if (pv) {
            const int steps = width(j) >> 4;
            const uint64_t vd = sdesc_sw128(ring + (group % kSlots) * L::kSlot, kCols * 128, 1024);
#pragma unroll
            for (int kk = 0; kk < kCols / 16; ++kk)
              if (kk < steps)
                mma_f16_ts(tO[t], tS[t] + buf * kCols + kk * 8, vd + (uint64_t)((kk * 16 * 128) >> 4), id_pv,
                           (begun || kk > 0) ? 1u : 0u);
          }
          if (next) scores(j + 2);
          // every commit to sfull is of scores, whose P the issuer waits for before the next; one to ofull
          // is waited for by the softmax before it makes the P of a later tile in the buffer
          if (next)
            mma_commit(&sfull[2 * t + buf]);
          else if (pv)
            mma_commit(&ofull[2 * t + buf]);
          mma_commit(&empty[group % kSlots]);
          if (j + 3 == tiles) mma_commit(qempty);   // the queries' last product is issued
        }
        __syncwarp();
        begun |= pv;
      }
      u += tiles > 0 ? tiles + 1 : 0;
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
  } else {
    // ------------------------------------------------------------ softmax rows
    zero_unwritten_rows<T>(a, p.rows_per_cta, threadIdx.x - 96, kThreads - 96, abort_word + 1);
    const int t = (warp - 3) >> 2;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int tq = kRows >> p.pack_log;                      // queries of a tile
    const int qi = t * tq + (row >> p.pack_log);             // query of the pair
    const uint32_t at = (uint32_t)(quarter * 32) << 16;
    const float c2 = a.scale * 1.4426950408889634f;          // log2(e); positive (window_tc_takes)
    uint8_t* stage = smem + L::kStage + (warp - 3) * 32 * L::kPitch;
    int count[2] = {0, 0}, ended[2] = {0, 0};   // commits waited for in each buffer: scores, P V alone
    bool ok = true;
#pragma unroll 1
    for (int pair = 0; ok; ++pair) {
      ok = mbar_wait_warp_lazy(&plan_full[pair & 1], (pair >> 1) & 1, ab, kErrPlan);
      if (!ok) break;
      const PairPlan& c = plans[pair & 1];
      if (c.live < 0) break;
      // rows behind the last query count as that query: they need no masks of their own
      const int hi = c.hi + min(qi, c.nq - 1);
      const int lo = hi - (int)min(a.window, (int64_t)1 << 30) + 1;
      const int tiles = c.tiles, total = c.total, sk = c.sk, tlo = c.lo[t], tlast = c.last[t], start = c.j0 * kCols;
      float m = -INFINITY, l = 0.0f;
      int done = 0;
      auto needed = [&](int j) {   // as the issuer's
        const int v = start + j * kCols;
        return j < tiles && v <= tlast && (v + kCols > tlo || v < sk);
      };
      // step j of the issuer: P V of tile j, then S of tile j + 2 into the same
      // buffer, then a commit; so the commit that brings S(j) says that P V of tile
      // j - 2 has ended; where there is no S(j), that P V has a commit of its own
#pragma unroll 1
      for (int j = 0; j < tiles + 2; ++j) {
        const int buf = j & 1;
        const bool here = needed(j);
        if (!here) {
          if (j < 2 || !needed(j - 2)) continue;
          ok = mbar_wait_warp_lazy(&ofull[2 * t + buf], ended[buf] & 1, ab, kErrO);
          if (!ok) break;
          ++ended[buf];
          continue;
        }
        ok = mbar_wait_warp_lazy(&sfull[2 * t + buf], count[buf] & 1, ab, kErrS);
        if (!ok) break;
        ++count[buf];
        tc_fence_after();
        // columns of a last, narrower tile that its product left out hold an earlier tile's numbers: hidden like others
        const int v0 = start + j * kCols, w = min(kCols, (total - v0 + 31) & ~31);
        const uint32_t ts = tS[t] + at + buf * kCols;
        // a tile that all rows of the warp see whole needs no mask
        const bool all_on = __all_sync(0xffffffffu, v0 + kCols - 1 <= hi && (v0 >= lo || v0 + kCols <= sk));
        float s0[32], s1[32];
        tmem_ld32(ts, s0);
        tmem_ld32(ts + 32, s1);
        tmem_wait_ld();
        tie32(s0);
        tie32(s1);
        if (!all_on) {
          auto seen = [&](int v) { return low_bits(hi - v + 1) & (~low_bits(lo - v) | low_bits(sk - v)) & low_bits(v0 + w - v); };
          hide(s0, seen(v0));
          hide(s1, seen(v0 + 32));
        }
        const float top = fmaxf(max32(s0), max32(s1)) * c2;
        const bool move = top > m + kMove;
        const bool fold = kLong && done > 0 && (done & (kFold - 1)) == 0;
        if (__any_sync(0xffffffffu, move) || fold) {
          const float to = move ? top : m;
          const float alpha = move ? ex2(m - to) : 1.0f;   // m = -inf: 0
          m = to;
          l *= alpha;
          if (done > 0) {
            // the product of the tile before may still run: its step's commit ends the wait (and is not used up)
            if (needed(j - 1)) {
              const bool more = needed(j + 1);
              ok = mbar_wait_warp_lazy(more ? &sfull[2 * t + (buf ^ 1)] : &ofull[2 * t + (buf ^ 1)],
                                       (more ? count[buf ^ 1] : ended[buf ^ 1]) & 1, ab, kErrO);
            }
            if (!ok) break;
            tc_fence_after();
            if (kLong)
              scale_fold_row(tO[t] + at, a.dv, alpha, m, p.sums, fold, done == kFold);
            else
              scale_row(tO[t] + at, a.dv, alpha);
          }
        }
        const float off = kShift - (m == -INFINITY ? 0.0f : m);
        const uint64_t off2 = pack2(off, off), c22 = pack2(c2, c2);
        uint64_t sum2[2] = {0, 0};
        exp_chunk<DT>(s0, c22, off2, sum2, ts);
        exp_chunk<DT>(s1, c22, off2, sum2, ts + 16);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&pfull[2 * t + buf]);
        float x0, x1, x2, x3;
        unpack2(sum2[0], x0, x1);
        unpack2(sum2[1], x2, x3);
        l += (x0 + x1) + (x2 + x3);
        ++done;
      }
      if (!ok) break;
      tc_fence_after();
      const int h0 = c.hk * p.group + c.g0, nq = c.nq;
      if (kLong && done > kFold) unfold_row(tO[t] + at, a.dv, m, p.sums);
      const int64_t obase = c.b * a.o_b + (int64_t)h0 * a.o_h + c.q_row * a.o_n;
      // 32 columns at a time pass through shared memory, so that neighbouring
      // lanes store neighbouring pieces of a row (16 bytes; the pitch keeps the
      // banks apart)
      T* out = static_cast<T*>(a.out) + obase;
      if (p.splits > 1) {   // this part's O, maximum and sum, for join_kernel
        const int64_t h = h0 + (row & (p.pack - 1)), r = (c.b * (int64_t)a.heads + h) * a.n + c.q_row + qi;
        float* to = p.part + (r * p.splits + c.split) * p.pitch;
#pragma unroll 1
        for (int c0 = 0; c0 < a.dv; c0 += 16) {
          float o[16];
          if (done > 0) {
            tmem_ld16(tO[t] + at + c0, o);
            tmem_wait_ld();
          }
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            if (qi < nq && c0 + e < p.pitch - 4)
              *reinterpret_cast<float4*>(to + c0 + e) =
                  done > 0 ? make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        if (qi < nq) *reinterpret_cast<float2*>(to + p.pitch - 4) = make_float2(m, l);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&plan_empty[pair & 1]);
        continue;
      }
      const float inv = 1.0f / l;
      bool fine = true;
#pragma unroll 1
      for (int c0 = 0; c0 < a.dv && t * tq < nq; c0 += 32) {
        float o[32];
        if (done > 0) {
          tmem_ld32(tO[t] + at + c0, o);
          tmem_wait_ld();
        }
        tie32(o);
        float big = 0.0f;
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          o[e] = l == 0.0f ? 0.0f : o[e] * inv;
          // 0 * x is 0, NaN where x is not finite
          big = c0 + e < a.dv ? fmaf(o[e], 0.0f, big) : big;
        }
        fine &= big == 0.0f;
#pragma unroll
        for (int e = 0; e < 32; e += 8)
          *reinterpret_cast<uint4*>(stage + lane * L::kPitch + e * 2) =
              make_uint4(pack16<DT>(o[e], o[e + 1]), pack16<DT>(o[e + 2], o[e + 3]), pack16<DT>(o[e + 4], o[e + 5]),
                         pack16<DT>(o[e + 6], o[e + 7]));
        __syncwarp();
        const int width = min(32, a.dv - c0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {   // 8 rows of four pieces
          const int r = i * 8 + (lane >> 2), piece = lane & 3;
          const int rr = quarter * 32 + r, rqi = t * tq + (rr >> p.pack_log);
          T* to = out + (int64_t)(rr & (p.pack - 1)) * a.o_h + rqi * a.o_n + c0 + piece * 8;
          if (rqi < nq && piece * 8 < width) {
            if (p.vec_out) {
              *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(stage + r * L::kPitch + piece * 16);
            } else {
#pragma unroll 1
              for (int e = 0; e < min(8, width - piece * 8); ++e)
                to[e] = *reinterpret_cast<const T*>(stage + r * L::kPitch + piece * 16 + e * 2);
            }
          }
        }
        __syncwarp();
      }
#pragma unroll 1
      for (unsigned left = __ballot_sync(0xffffffffu, qi < nq && !fine); left; left &= left - 1) {
        const int rr = quarter * 32 + __ffs(left) - 1, rqi = t * tq + (rr >> p.pack_log), g = rr & (p.pack - 1);
        repair_row<DT>(a, c.b * a.q_b + (int64_t)(h0 + g) * a.q_h + (c.q_row + rqi) * a.q_n,
                       c.b * a.k_b + (int64_t)c.hk * a.k_h + c.k_row * a.k_n,
                       c.b * a.v_b + (int64_t)c.hk * a.v_h + c.k_row * a.v_n, obase + (int64_t)g * a.o_h + rqi * a.o_n,
                       c.p0 + rqi, c.m, abort_word + 1);
      }
      tc_fence_before();   // O has been read: the next pair's products may overwrite it
      __syncwarp();
      if (lane == 0) mbar_arrive(&plan_empty[pair & 1]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of rows whose keys were split: a warp takes a row (query, head).
template <int DT>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ WindowTcParams p) {
  using T = typename Elem<DT>::T;
  const WindowArgs& a = p.a;
  const int lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (r >= (int64_t)a.batch * a.heads * a.n) return;
  const int64_t bh = r / a.n, i = r - bh * a.n, b = bh / a.heads, h = bh - b * a.heads;
  const float* part = p.part + r * p.splits * p.pitch;
  const float2 ml = lane < p.splits ? *reinterpret_cast<const float2*>(part + lane * p.pitch + p.pitch - 4)
                                    : make_float2(-INFINITY, 0.0f);
  float top = ml.x;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  const float f = ml.x == -INFINITY ? 0.0f : ex2(ml.x - top);
  float total = f * ml.y;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) total += __shfl_xor_sync(0xffffffffu, total, d);
  T* out = static_cast<T*>(a.out) + b * a.o_b + h * a.o_h + i * a.o_n;
  bool fine = true;
  for (int c0 = 0; c0 < a.dv; c0 += 32) {
    const int c = c0 + lane;
    float sum = 0.0f;
    for (int s = 0; s < p.splits; ++s) {
      const float fs = __shfl_sync(0xffffffffu, f, s);
      if (c < a.dv) sum = fmaf(fs, part[s * p.pitch + c], sum);
    }
    const float x = total == 0.0f ? 0.0f : sum / total;
    if (c < a.dv) {
      fine &= fabsf(x) < INFINITY;
      out[c] = from_f32<T>(x);
    }
  }
  if (!__all_sync(0xffffffffu, fine)) {
    const int64_t hk = h / p.group;
    __syncwarp();
    repair_row<DT>(a, b * a.q_b + h * a.q_h + i * a.q_n, b * a.k_b + hk * a.k_h, b * a.v_b + hk * a.v_h,
                   b * a.o_b + h * a.o_h + i * a.o_n, a.m - a.n + i, a.m, nullptr);
  }
}

// ---------------------------------------------------------------- host side

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static const EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      return reinterpret_cast<EncodeTiledFn>(p);
    return static_cast<EncodeTiledFn>(nullptr);
  }();
  return fn;
}

// A map of 16-bit elements, 128-byte swizzle, zeros outside.  dims[0] is the
// contiguous axis; strides (in elements) belong to dims[1..].  An axis of one
// entry may have any stride: it takes one that the encoder accepts.
int encode(CUtensorMap* map, bool bf16, const void* base, int rank, const int64_t* dims, const int64_t* strides,
           const int* box) {
  cuuint64_t gd[5], gs[4];
  cuuint32_t bx[5], es[5];
  for (int i = 0; i < rank; ++i) {
    gd[i] = (cuuint64_t)dims[i];
    bx[i] = (cuuint32_t)box[i];
    es[i] = 1;
    if (i > 0) gs[i - 1] = dims[i] > 1 ? (cuuint64_t)strides[i - 1] * 2 : 16;
  }
  const EncodeTiledFn enc = encode_fn();
  if (!enc) return set_error(SA_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  const CUresult r = enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank,
                         const_cast<void*>(base), gd, gs, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(SA_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return SA_OK;
}

template <int DT, int DC, int VC>
int launch_one(const CUtensorMap* maps, const WindowTcParams& p, dim3 grid, cudaStream_t s) {
  auto kern = p.sums ? window_tc_kernel<DT, DC, VC, true> : window_tc_kernel<DT, DC, VC, false>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Layout<DC, VC>::kBytes);
  if (e != cudaSuccess) return set_error(SA_ERR_CUDA, "window_tc smem attribute: %s", cudaGetErrorString(e));
  kern<<<grid, kThreads, Layout<DC, VC>::kBytes, s>>>(maps[0], maps[1], maps[2], maps[3], maps[4], maps[5], maps[6], p);
  return check_launch("window_tc_kernel");
}

template <int DT>
int launch_dims(const CUtensorMap* maps, const WindowTcParams& p, dim3 grid, cudaStream_t s) {
  if (p.a.d <= 64) return p.a.dv <= 64 ? launch_one<DT, 1, 1>(maps, p, grid, s) : launch_one<DT, 1, 2>(maps, p, grid, s);
  return p.a.dv <= 64 ? launch_one<DT, 2, 1>(maps, p, grid, s) : launch_one<DT, 2, 2>(maps, p, grid, s);
}

void shape_of(const WindowArgs& a, WindowTcParams& p) {
  p.group = a.heads / a.kv_heads;
  p.pack = 1;
  while (p.pack < 32 && p.group % (2 * p.pack) == 0) {
    p.pack *= 2;
    ++p.pack_log;
  }
  p.blocks = p.group / p.pack;
  p.rows_per_cta = 2 * kRows / p.pack;
}

int part_pitch(int dv) { return (dv + 3) / 4 * 4 + 4; }

bool aligned(const void* base, int64_t size1, int64_t s1, int64_t size2, int64_t s2, int64_t size3, int64_t s3) {
  const bool ok = ((uintptr_t)base & 15) == 0;
  auto fits = [](int64_t size, int64_t s) { return size <= 1 || (s > 0 && (s & 7) == 0 && s < ((int64_t)1 << 38)); };
  return ok && fits(size1, s1) && fits(size2, s2) && fits(size3, s3);
}

}  // namespace

// Whether the tensor-core kernel takes these tensors: 16-bit elements, head
// widths up to 128, rows on 16-byte borders (TMA), no repeated rows, and a positive
// scale (the running maximum is taken before the scale, and a hidden score, -inf,
// has to stay that when it is scaled).
bool window_tc_takes(const WindowArgs& a) {
  if (a.dtype == SA_REP_FLOAT32 || a.d > 128 || a.dv > 128 || a.m == 0 || a.m >= (1 << 30) || a.n >= (1 << 30) || !(a.scale > 0.0f)) return false;
  return aligned(a.q, a.n, a.q_n, a.heads, a.q_h, a.cu_q ? 1 : a.batch, a.q_b) &&
         aligned(a.k, a.m, a.k_n, a.kv_heads, a.k_h, a.cu_q ? 1 : a.batch, a.k_b) &&
         aligned(a.v, a.m, a.v_n, a.kv_heads, a.v_h, a.cu_q ? 1 : a.batch, a.v_b);
}

// Parts of each pair's keys, for a dense call whose pairs fill less than half of
// the SMs: at most 32 (a lane each in the join), at least four tiles to a part,
// from 48 tiles on, and where the tiles that a pair saves (1.3 us each, 0.9 with few
// rows) cost more than the parts (15 us for the join's launch and the workspace,
// 0.9 ns for each part's row of 128 columns, written and read).  32/8 heads of 128,
// whole and split: 1 query over 8192 keys 106 and 31 us, over 4096 59 and 26; 256
// over 4096 82 and 51; 512, in two parts, over 4096 82 and 90 (stays whole), over
// 8192 151 and 126; over 1024 keys 28 whole and 39.
int window_tc_splits(const WindowArgs& a, int64_t tiles) {
  if (a.cu_q) return 1;
  WindowTcParams p{};
  shape_of(a, p);
  const int64_t pairs = ceil_div(a.n, p.rows_per_cta) * a.batch * (a.heads / p.pack);
  const int64_t splits = std::min<int64_t>(std::min<int64_t>(148 / std::max<int64_t>(pairs, 1), tiles / 4), 32);
  if (splits < 2 || tiles < 48) return 1;
  const double saved = 1.3 * (double)tiles * (double)(splits - 1) / (double)splits;
  const double parts = (double)a.batch * a.heads * (double)a.n * (double)splits;
  return saved > 15.0 + 0.0009 / 132.0 * part_pitch(a.dv) * parts ? (int)splits : 1;
}

// What a call keeps in its workspace: the parts of split keys, then folded sums.
struct WindowTcSpace {
  int splits;
  size_t sums_at, bytes;   // folded sums, where bytes > sums_at
};
WindowTcSpace window_tc_space(const WindowArgs& a) {
  WindowTcParams p{};
  shape_of(a, p);
  // the most key tiles of a pair
  const int64_t rows = std::min<int64_t>(a.n, p.rows_per_cta), span = std::min<int64_t>(a.window, a.m) + rows;
  const int64_t tiles = ceil_div(std::min<int64_t>(a.m, span + std::min<int64_t>(a.sinks, a.m)), kCols);
  WindowTcSpace w{window_tc_splits(a, tiles), 0, 0};
  if (w.splits > 1) w.sums_at = ((size_t)a.batch * a.heads * a.n * w.splits * part_pitch(a.dv) * sizeof(float) + 255) & ~(size_t)255;
  w.bytes = w.sums_at;
  if (tiles / w.splits + 2 > kFold) w.bytes += (size_t)kFoldCtas * 2 * (a.dv + 1) * kRows * sizeof(float);
  return w;
}

size_t window_tc_bytes(const WindowArgs& a) { return window_tc_space(a).bytes; }

int launch_window_tc(const WindowArgs& a, void* workspace, size_t workspace_bytes, cudaStream_t s) {
  WindowTcParams p{};
  p.a = a;
  shape_of(a, p);
  p.vec_out = ((uintptr_t)a.out & 15) == 0 && (a.o_n & 7) == 0 && (a.o_h & 7) == 0 && (a.o_b & 7) == 0 &&
              (a.dv & 7) == 0;
  p.wait_ns = wait_limit_ns();
  p.pitch = part_pitch(a.dv);
  // without a workspace the keys are not split, nor sums folded
  const WindowTcSpace space = window_tc_space(a);
  const bool given = workspace && workspace_bytes >= space.bytes;
  p.splits = given ? space.splits : 1;
  p.part = static_cast<float*>(workspace);
  p.sums = given && space.bytes > space.sums_at ? reinterpret_cast<float*>(static_cast<char*>(workspace) + space.sums_at) : nullptr;
  const bool bf16 = a.dtype == SA_REP_BFLOAT16;
  const int64_t batch = a.cu_q ? 1 : a.batch;
  CUtensorMap maps[7];   // q; k in boxes of a tile, of the seam's 16 rows and of the rows behind them; v likewise
  const int64_t qd[5] = {a.d, p.group, a.n, a.kv_heads, batch};
  const int64_t qs[4] = {a.q_h, a.q_n, a.q_h * p.group, a.q_b};
  const int qb[5] = {64, p.pack, kRows / p.pack, 1, 1};
  int rc = encode(&maps[0], bf16, a.q, 5, qd, qs, qb);
  for (int i = 0; !rc && i < 6; ++i) {
    const bool isv = i >= 3;
    const int64_t kd[4] = {isv ? a.dv : a.d, a.m, a.kv_heads, batch};
    const int64_t ks[3] = {isv ? a.v_n : a.k_n, isv ? a.v_h : a.k_h, isv ? a.v_b : a.k_b};
    const int rows[3] = {kCols, kSeam, kCols - kSeam};
    const int kb[4] = {64, rows[i % 3], 1, 1};
    rc = encode(&maps[1 + i], bf16, isv ? a.v : a.k, 4, kd, ks, kb);
  }
  if (rc) return rc;
  const int64_t tiles = tile_count(a, p.rows_per_cta), items = tiles * (a.heads / p.pack) * p.splits;
  if (items > 2147483647LL) return set_error(SA_ERR_UNSUPPORTED, "window attention: grid too large");
  p.tiles = (uint32_t)tiles;
  p.items = (uint32_t)items;
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return set_error(SA_ERR_CUDA, "window_tc device query: %s", cudaGetErrorString(e));
  if (p.sums) sms = std::min(sms, kFoldCtas);
  dim3 grid((unsigned)(items < sms ? items : sms));
  rc = bf16 ? launch_dims<SA_REP_BFLOAT16>(maps, p, grid, s) : launch_dims<SA_REP_FLOAT16>(maps, p, grid, s);
  if (rc || p.splits == 1) return rc;
  const unsigned join = (unsigned)ceil_div((int64_t)a.batch * a.heads * a.n, 8);
  if (bf16)
    join_kernel<SA_REP_BFLOAT16><<<join, 256, 0, s>>>(p);
  else
    join_kernel<SA_REP_FLOAT16><<<join, 256, 0, s>>>(p);
  return check_launch("window join_kernel");
}

}  // namespace sa
