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
// Warps: 0 loads (TMA), 1 issues the products (converged, one elected lane),
// 2..5 and 6..9 are the softmax of query tile 0 and 1, one row per thread.
// TMEM: S0 S1 O0 O1 of 128 columns each; P, in 16 bits, overwrites the first
// half of its S.  The issue order per key tile is PV0 S0' PV1 S1', so that one
// tile's softmax runs under the other's products; the commit of S(j + 1) also
// says that PV(j) has ended, so that a row may then scale its O.
//
// Softmax in base 2 with a lazily moved maximum: m follows a tile's maximum
// only when that is more than kMove above it, so O is scaled rarely.  P is
// 2^(x - m + kShift): bfloat16 takes kShift = -24 (float32's range, so that
// 2^16 of the largest values still sum below float32's limit), float16 +6 (at
// most 2^14, and 2^-14, where float16 starts to lose bits, is 2^-20 of the
// row's usual largest).
//
// A product with a hidden key's value is 0 * v, NaN where v is NaN or infinite.
// Rows that come out non-finite are computed again by one thread from the
// visible keys alone (row_again): what a query does not see cannot reach it.
#include <cuda.h>
#include <math.h>

#include "serving.cuh"
#include "tc_util.cuh"

namespace sa {

namespace {

using namespace tc;

constexpr int kRows = 128;     // rows of a query tile
constexpr int kCols = 128;     // keys of a key tile
constexpr int kSeam = 16;      // rows of a box of the seam tile
constexpr int kThreads = 320;
constexpr float kMove = 8.0f;

constexpr int kErrQ = 501, kErrFull = 502, kErrP = 503, kErrS = 504, kErrEmpty = 505, kErrO = 506, kErrDrain = 507;

struct WindowTcParams {
  WindowArgs a;
  int group, pack, blocks;   // query heads per key head, heads per tile, tiles of heads per key head
  int rows_per_cta;          // queries of a CTA (2 * kRows / pack)
  int vec_out;               // out rows take 16-byte stores
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

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

// One output row from its visible keys alone, in float32 by one thread.
template <int DT>
__device__ __noinline__ void row_again(const WindowArgs& a, int64_t qoff, int64_t koff, int64_t voff, int64_t ooff,
                                       int64_t p, int64_t m) {
  using T = typename Elem<DT>::T;
  const T* q = static_cast<const T*>(a.q) + qoff;
  const T* k = static_cast<const T*>(a.k) + koff;
  const T* v = static_cast<const T*>(a.v) + voff;
  T* out = static_cast<T*>(a.out) + ooff;
  const KeyRanges kr = key_ranges(p, p, m, a.window, a.sinks);
  auto score = [&](int64_t j) {
    float x = 0.0f;
    for (int c = 0; c < a.d; ++c) x = fmaf(to_f32(q[c]), to_f32(k[j * a.k_n + c]), x);
    return x * a.scale;
  };
  float top = -INFINITY;
  bool nan = false;
  const int64_t count = kr.first + kr.end - kr.begin;
  for (int64_t u = 0; u < count; ++u) {
    const float x = score(u < kr.first ? u : kr.begin + u - kr.first);
    nan |= x != x;
    top = fmaxf(top, x);
  }
  top = nan ? NAN : (top == -INFINITY ? 0.0f : top);
  for (int c0 = 0; c0 < a.dv; c0 += 16) {
    float acc[16], l = 0.0f;
    for (int c = 0; c < 16; ++c) acc[c] = 0.0f;
    for (int64_t u = 0; u < count; ++u) {
      const int64_t j = u < kr.first ? u : kr.begin + u - kr.first;
      const float e = expf(score(j) - top) * 0x1p-24f;
      l += e;
      if (e != 0.0f)
        for (int c = 0; c < 16 && c0 + c < a.dv; ++c) acc[c] = fmaf(e, to_f32(v[j * a.v_n + c0 + c]), acc[c]);
    }
    for (int c = 0; c < 16 && c0 + c < a.dv; ++c) out[c0 + c] = from_f32<T>(l == 0.0f ? 0.0f : acc[c] / l);
  }
}

template <int DC, int VC>   // 64-column chunks of the head widths
struct Layout {
  static constexpr uint32_t kQ = DC * kRows * 128;                              // one query tile
  static constexpr uint32_t kSlot = (DC > VC ? DC : VC) * kCols * 128;          // one K or V tile
  static constexpr int kSlots = DC == 2 || VC == 2 ? 5 : 8;
  static constexpr uint32_t kRing = 2 * kQ;
  static constexpr uint32_t kBars = kRing + kSlots * kSlot;
  static constexpr uint32_t kBytes = kBars + (2 * kSlots + 8) * 8 + 16 + 1024;
  static_assert(kBytes <= 227 * 1024, "shared memory");
};

template <int DT, int DC, int VC>
__global__ void __launch_bounds__(kThreads, 1)
window_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_ks, const __grid_constant__ CUtensorMap tm_v,
                 const __grid_constant__ CUtensorMap tm_vs, const __grid_constant__ WindowTcParams p) {
  using L = Layout<DC, VC>;
  using T = typename Elem<DT>::T;
  constexpr int kSlots = L::kSlots;
  constexpr float kShift = DT == SA_REP_BFLOAT16 ? -24.0f : 6.0f;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t* empty = full + kSlots;
  uint64_t* sfull = empty + kSlots;   // [2]
  uint64_t* pfull = sfull + 2;        // [2]
  uint64_t* qfull = pfull + 2;
  uint64_t* ofull = qfull + 1;
  uint64_t* drain = ofull + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  int* abort_word = reinterpret_cast<int*>(tmem_slot + 1);

  const WindowArgs& a = p.a;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  int64_t tile;
  const int b = tile_request(a, blockIdx.x, p.rows_per_cta, &tile);
  const Request rq = request_of(a, b);
  const int64_t i0 = tile * p.rows_per_cta;
  if (tile < 0 || i0 >= rq.n) return;
  const int hk = blockIdx.y / p.blocks, g0 = (blockIdx.y % p.blocks) * p.pack;
  const int tq = kRows / p.pack;                               // queries of a tile
  const int nq = (int)min((int64_t)p.rows_per_cta, rq.n - i0);
  const int64_t p0 = rq.m - rq.n + i0;
  const Columns cols = columns_of(p0, p0 + nq - 1, rq.m, a.window, a.sinks);
  const int tiles = (cols.total + kCols - 1) / kCols;
  const int window = (int)min(a.window, (int64_t)1 << 30);
  // the columns that query tile t needs: below hi_t, and from lo_t on or below sk
  const int hi0 = (int)(p0 + min(tq, nq) - 1 - cols.begin) + cols.fill;
  const int hi1 = nq > tq ? (int)(p0 + nq - 1 - cols.begin) + cols.fill : -1;
  const int lo0 = (int)(p0 - cols.begin) + cols.fill - window + 1;
  const int lo1 = lo0 + tq;
  auto needed = [&](int t, int j) {
    const int v0 = j * kCols;
    return v0 <= (t ? hi1 : hi0) && (v0 + kCols > (t ? lo1 : lo0) || v0 < cols.sk);
  };
  // columns of tile j that a product takes: a multiple of 32
  auto width = [&](int j) { return min(kCols, (cols.total - j * kCols + 31) & ~31); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sfull[t], 1);
      mbar_init(&pfull[t], 4);
    }
    mbar_init(qfull, 1);
    mbar_init(ofull, 1);
    mbar_init(drain, 1);
    *abort_word = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const Abort ab{abort_word, a.status, p.wait_ns};
  const uint32_t tS[2] = {tmem, tmem + 128}, tO[2] = {tmem + 256, tmem + 384};

  if (warp == 0) {
    // ------------------------------------------------------------ loads
    if (lane == 0 && tiles > 0) {
      const int qb = a.cu_q ? 0 : b;
      mbar_arrive_expect_tx(qfull, 2 * L::kQ);
      for (int t = 0; t < 2; ++t)
        for (int c = 0; c < DC; ++c)
          tma_load_5d(smem + t * L::kQ + c * (kRows * 128), &tm_q, qfull, c * 64, g0, (int)(rq.q0 + i0) + t * tq, hk, qb);
      int issued = 0;
      for (int u = 0; u < 2 * tiles; ++u) {   // K of a tile, then its V
        const int s = u % kSlots, j = u >> 1;
        if (u >= kSlots && !mbar_wait(&empty[s], ((u / kSlots) - 1) & 1, ab, kErrEmpty)) break;
        const bool isv = u & 1;
        const int chunks = isv ? VC : DC;
        uint8_t* dst = smem + L::kRing + s * L::kSlot;
        mbar_arrive_expect_tx(&full[s], chunks * kCols * 128);
        const int v0 = j * kCols;
        if (v0 >= cols.fill) {
          const int row = (int)(rq.k0 + cols.begin) + v0 - cols.fill;
          for (int c = 0; c < chunks; ++c)
            tma_load_4d(dst + c * (kCols * 128), isv ? &tm_v : &tm_k, &full[s], c * 64, row, hk, qb);
        } else {
          for (int r = 0; r < kCols; r += kSeam) {
            const int v = v0 + r;
            const int row = (int)rq.k0 + (v < cols.fill ? v : (int)cols.begin + v - cols.fill);
            for (int c = 0; c < chunks; ++c)
              tma_load_4d(dst + c * (kCols * 128) + r * 128, isv ? &tm_vs : &tm_ks, &full[s], c * 64, row, hk, qb);
          }
        }
        ++issued;
      }
      // never leave with copies in flight
      for (int u = max(0, issued - kSlots); u <= issued; ++u) {
        uint64_t* bar = u < issued ? &full[u % kSlots] : qfull;
        const int parity = u < issued ? (u / kSlots) & 1 : 0;
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
  } else if (warp == 1) {
    // ------------------------------------------------------------ products
    if (tiles > 0) {
      bool ok = mbar_wait_warp(qfull, 0, ab, kErrQ);
      const int ksteps = (a.d + 15) >> 4;
      const uint32_t id_pv = idesc_f16(kRows, (a.dv + 15) & ~15, DT == SA_REP_BFLOAT16, false, true);
      int done[2] = {0, 0};   // products P V issued per query tile
      for (int j = 0; ok && j <= tiles; ++j) {
        const int us = 2 * j, uv = 2 * j - 1;   // ring positions of K(j) and V(j - 1)
        bool waited_k = false, waited_v = false;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (ok && j > 0 && needed(t, j - 1)) {
            if (!waited_v) ok = mbar_wait_warp(&full[uv % kSlots], (uv / kSlots) & 1, ab, kErrFull);
            waited_v = true;
            if (ok) ok = mbar_wait_warp(&pfull[t], done[t] & 1, ab, kErrP);
            if (ok) {
              tc_fence_after();
              const int steps = width(j - 1) >> 4;
              if (elect_one()) {
                const uint64_t vd = sdesc_sw128(smem_u32(smem + L::kRing + (uv % kSlots) * L::kSlot), kCols * 128, 1024);
                for (int kk = 0; kk < steps; ++kk)
                  mma_f16_ts(tO[t], tS[t] + kk * 8, vd + (uint64_t)((kk * 16 * 128) >> 4), id_pv,
                             (done[t] > 0 || kk > 0) ? 1u : 0u);
              }
              __syncwarp();
              ++done[t];
            }
          }
          if (ok && j < tiles && needed(t, j)) {
            if (!waited_k) ok = mbar_wait_warp(&full[us % kSlots], (us / kSlots) & 1, ab, kErrFull);
            waited_k = true;
            if (ok) {
              tc_fence_after();
              const uint32_t id_s = idesc_f16(kRows, width(j), DT == SA_REP_BFLOAT16, false, false);
              if (elect_one()) {
                const uint64_t qd = sdesc_sw128(smem_u32(smem + t * L::kQ), 16, 1024);
                const uint64_t kd = sdesc_sw128(smem_u32(smem + L::kRing + (us % kSlots) * L::kSlot), 16, 1024);
                for (int kk = 0; kk < ksteps; ++kk) {
                  const uint64_t at = (uint64_t)(((kk >> 2) * (kRows * 128) + (kk & 3) * 32) >> 4);
                  mma_f16_ss(tS[t], qd + at, kd + at, id_s, kk > 0 ? 1u : 0u);
                }
                mma_commit(&sfull[t]);
              }
              __syncwarp();
            }
          }
        }
        if (ok && elect_one()) {
          if (j > 0) mma_commit(&empty[uv % kSlots]);
          if (j < tiles) mma_commit(&empty[us % kSlots]);
        }
        __syncwarp();
      }
      if (ok && elect_one()) mma_commit(ofull);
      if (elect_one()) mma_commit(drain);
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(drain, 0)) {
        if (globaltimer_ns() - t0 > 2000000000ull) {
          if (a.status) atomicCAS(a.status, 0, kErrDrain);
          break;
        }
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------ softmax rows
    const int t = (warp - 2) >> 2;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int qi = t * tq + row / p.pack;                    // query of the CTA
    const int h = hk * p.group + g0 + (row & (p.pack - 1));
    const bool valid = qi < nq;
    const uint32_t at = (uint32_t)(quarter * 32) << 16;
    const int hi = valid ? (int)(p0 + qi - cols.begin) + cols.fill : -1;
    const int lo = hi - window + 1;
    const bool flip = a.scale < 0.0f;
    const float c2 = fabsf(a.scale) * 1.4426950408889634f;
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    int done = 0;
    for (int j = 0; ok && j < tiles; ++j) {
      if (!needed(t, j)) continue;
      if (!mbar_wait_warp(&sfull[t], done & 1, ab, kErrS)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int w = width(j), v0 = j * kCols;
      float s[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (c * 32 < w) tmem_ld32(tS[t] + at + c * 32, s[c]);
      tmem_wait_ld();
      if (flip) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e) s[c][e] = -s[c][e];
      }
      const bool all_on = v0 + w - 1 <= hi && (v0 >= lo || v0 + w <= cols.sk);
      if (!__all_sync(0xffffffffu, all_on)) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int vc = v0 + c * 32;
          const uint32_t on = low_bits(hi - vc + 1) & (~low_bits(lo - vc) | low_bits(cols.sk - vc));
#pragma unroll
          for (int e = 0; e < 32; ++e) s[c][e] = (on >> e) & 1u ? s[c][e] : -INFINITY;
        }
      }
      float tm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (c * 32 < w) {
#pragma unroll
          for (int e = 0; e < 32; ++e) tm[e & 3] = fmaxf(tm[e & 3], s[c][e]);
        }
      const float top = fmaxf(fmaxf(tm[0], tm[1]), fmaxf(tm[2], tm[3])) * c2;
      const bool move = top > m + kMove;
      if (__any_sync(0xffffffffu, move)) {
        const float to = move ? top : m;
        const float alpha = move ? ex2(m - to) : 1.0f;   // m = -inf: 0
        m = to;
        l *= alpha;
        if (done > 0) {   // the products of this row's earlier tiles have ended (sfull)
#pragma unroll
          for (int c = 0; c < VC * 2; ++c)
            if (c * 32 < a.dv) {
              float o[32];
              tmem_ld32(tO[t] + at + c * 32, o);
              tmem_wait_ld();
              uint32_t os[32];
#pragma unroll
              for (int e = 0; e < 32; ++e) os[e] = __float_as_uint(o[e] * alpha);
              tmem_st32(tO[t] + at + c * 32, os);
            }
        }
      }
      const float off = kShift - (m == -INFINITY ? 0.0f : m);
      const uint64_t off2 = pack2(off, off), c22 = pack2(c2, c2);
      uint64_t sum2[2] = {0, 0};
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (c * 32 < w) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float x, y;
            unpack2(fma2(pack2(s[c][2 * e], s[c][2 * e + 1]), c22, off2), x, y);
            x = ex2(x);
            y = ex2(y);
            sum2[e & 1] = add2(sum2[e & 1], pack2(x, y));
            pk[e] = pack16<DT>(x, y);
          }
          tmem_st16(tS[t] + at + c * 16, pk);
        }
      float x0, x1, x2, x3;
      unpack2(sum2[0], x0, x1);
      unpack2(sum2[1], x2, x3);
      l += (x0 + x1) + (x2 + x3);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&pfull[t]);
      ++done;
    }
    if (ok && tiles > 0 && done > 0) ok = mbar_wait_warp(ofull, 0, ab, kErrO);
    if (ok) {
      tc_fence_after();
      const int64_t ooff = b * a.o_b + (int64_t)h * a.o_h + (rq.q0 + i0 + qi) * a.o_n;
      T* orow = static_cast<T*>(a.out) + (valid ? ooff : 0);
      bool fine = true;
#pragma unroll
      for (int c = 0; c < VC * 2; ++c) {
        if (c * 32 >= a.dv) break;
        float o[32];
        if (done > 0) {
          tmem_ld32(tO[t] + at + c * 32, o);
          tmem_wait_ld();
        }
        const float inv = 1.0f / l;
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float x = l == 0.0f ? 0.0f : o[2 * e] * inv, y = l == 0.0f ? 0.0f : o[2 * e + 1] * inv;
          fine &= c * 32 + 2 * e >= a.dv || fabsf(x) < INFINITY;
          fine &= c * 32 + 2 * e + 1 >= a.dv || fabsf(y) < INFINITY;
          pk[e] = pack16<DT>(x, y);
        }
        if (valid) {
          if (p.vec_out && c * 32 + 32 <= a.dv) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              reinterpret_cast<uint4*>(orow + c * 32)[e] = make_uint4(pk[4 * e], pk[4 * e + 1], pk[4 * e + 2], pk[4 * e + 3]);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (c * 32 + e < a.dv) {
                const uint16_t bits = (uint16_t)(pk[e >> 1] >> (16 * (e & 1)));
                reinterpret_cast<uint16_t*>(orow)[c * 32 + e] = bits;
              }
          }
        }
      }
      if (valid && !fine)
        row_again<DT>(a, b * a.q_b + (int64_t)h * a.q_h + (rq.q0 + i0 + qi) * a.q_n,
                      b * a.k_b + (int64_t)hk * a.k_h + rq.k0 * a.k_n, b * a.v_b + (int64_t)hk * a.v_h + rq.k0 * a.v_n, ooff,
                      p0 + qi, rq.m);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
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
  auto kern = window_tc_kernel<DT, DC, VC>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Layout<DC, VC>::kBytes);
  if (e != cudaSuccess) return set_error(SA_ERR_CUDA, "window_tc smem attribute: %s", cudaGetErrorString(e));
  kern<<<grid, kThreads, Layout<DC, VC>::kBytes, s>>>(maps[0], maps[1], maps[2], maps[3], maps[4], p);
  return check_launch("window_tc_kernel");
}

template <int DT>
int launch_dims(const CUtensorMap* maps, const WindowTcParams& p, dim3 grid, cudaStream_t s) {
  if (p.a.d <= 64) return p.a.dv <= 64 ? launch_one<DT, 1, 1>(maps, p, grid, s) : launch_one<DT, 1, 2>(maps, p, grid, s);
  return p.a.dv <= 64 ? launch_one<DT, 2, 1>(maps, p, grid, s) : launch_one<DT, 2, 2>(maps, p, grid, s);
}

bool aligned(const void* base, int64_t size1, int64_t s1, int64_t size2, int64_t s2, int64_t size3, int64_t s3) {
  const bool ok = ((uintptr_t)base & 15) == 0;
  auto fits = [](int64_t size, int64_t s) { return size <= 1 || (s > 0 && (s & 7) == 0 && s < ((int64_t)1 << 38)); };
  return ok && fits(size1, s1) && fits(size2, s2) && fits(size3, s3);
}

}  // namespace

// Whether the tensor-core kernel takes these tensors: 16-bit elements, head
// widths up to 128, rows on 16-byte borders (TMA) and no repeated rows.
bool window_tc_takes(const WindowArgs& a) {
  if (a.dtype == SA_REP_FLOAT32 || a.d > 128 || a.dv > 128 || a.m == 0) return false;
  return aligned(a.q, a.n, a.q_n, a.heads, a.q_h, a.cu_q ? 1 : a.batch, a.q_b) &&
         aligned(a.k, a.m, a.k_n, a.kv_heads, a.k_h, a.cu_q ? 1 : a.batch, a.k_b) &&
         aligned(a.v, a.m, a.v_n, a.kv_heads, a.v_h, a.cu_q ? 1 : a.batch, a.v_b);
}

int launch_window_tc(const WindowArgs& a, cudaStream_t s) {
  WindowTcParams p{};
  p.a = a;
  p.group = a.heads / a.kv_heads;
  p.pack = 1;
  while (p.pack < 32 && p.group % (2 * p.pack) == 0) p.pack *= 2;
  p.blocks = p.group / p.pack;
  p.rows_per_cta = 2 * kRows / p.pack;
  p.vec_out = ((uintptr_t)a.out & 15) == 0 && (a.o_n & 7) == 0 && (a.o_h & 7) == 0 && (a.o_b & 7) == 0;
  p.wait_ns = wait_limit_ns();
  const bool bf16 = a.dtype == SA_REP_BFLOAT16;
  const int64_t batch = a.cu_q ? 1 : a.batch;
  CUtensorMap maps[5];
  const int64_t qd[5] = {a.d, p.group, a.n, a.kv_heads, batch};
  const int64_t qs[4] = {a.q_h, a.q_n, a.q_h * p.group, a.q_b};
  const int qb[5] = {64, p.pack, kRows / p.pack, 1, 1};
  int rc = encode(&maps[0], bf16, a.q, 5, qd, qs, qb);
  for (int i = 0; !rc && i < 4; ++i) {
    const bool isv = i >= 2;
    const int64_t kd[4] = {isv ? a.dv : a.d, a.m, a.kv_heads, batch};
    const int64_t ks[3] = {isv ? a.v_n : a.k_n, isv ? a.v_h : a.k_h, isv ? a.v_b : a.k_b};
    const int kb[4] = {64, i & 1 ? kSeam : kCols, 1, 1};
    rc = encode(&maps[1 + i], bf16, isv ? a.v : a.k, 4, kd, ks, kb);
  }
  if (rc) return rc;
  const int64_t tiles = tile_count(a, p.rows_per_cta);
  if (tiles > 2147483647LL || a.heads / p.pack > 65535) return set_error(SA_ERR_UNSUPPORTED, "window attention: grid too large");
  dim3 grid((unsigned)tiles, (unsigned)(a.heads / p.pack));
  return bf16 ? launch_dims<SA_REP_BFLOAT16>(maps, p, grid, s) : launch_dims<SA_REP_FLOAT16>(maps, p, grid, s);
}

}  // namespace sa
