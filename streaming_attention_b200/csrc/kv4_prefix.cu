// The queries of all requests over a prefix that they share, on the 5th-generation
// tensor cores (tcgen05 kind::f16, TMEM): float16 and bfloat16, head widths up to 128.
// What the prefix of a batch adds to each row: an unfinished sum, its maximum and total
// for kTail (kv4_attend.cuh), as kPrefix there, which takes the other types and few rows.
//
// A code less 8 is exact in bfloat16, so the products take codes and the rows' scales and
// least values stay outside, in float32.  With x = least + 8 scale,
//   score_j = s_k (Q K'^T)_j + x_k sum(Q),   O = (p s_v) V' + sum(p x_v),
// K', V' the centred codes.  Q is one bfloat16 piece (float16: two, exact), and so is p s_v
// (rounded to bfloat16, as the windowed attention's probabilities; float16: two pieces, 16 bits).
//
// A CTA holds two tiles of 128 query rows of one key head (a row: request, query, head)
// and a part of the prefix in tiles of 64 tokens; all rows see (nearly) all of it, so a
// decoded tile serves 256 rows.  Warps: 0..3 and 4..7 are the softmax of a row tile, one
// row a thread; 8..11 decode: 16 bytes of codes a load, two tiles ahead in registers, to
// swizzled tiles in shared memory; 12 and 13 issue the products of a row tile, one elected lane.
// TMEM: of each row tile two S of 64 columns and O; P overwrites its S.  The issuer goes
// P V(j), S(j + 2), so that scores are there while a softmax runs.
//
// Order inside the tiles.  A word of a key row holds eight columns' codes; one shift and
// two logical operations give those of columns i and i + 4, so K' and Q hold columns in the
// order 0 4 1 5 2 6 3 7.  A word of values holds four tokens of two columns, and gives tokens
// 0 and 2, 1 and 3: V' lies a column to a row, tokens in the order 0 2 1 3, and P's halves
// are packed to match.
#include <math.h>

#include <algorithm>

#include "kv4_attend.cuh"
#include "tc_util.cuh"

namespace sa {

namespace {

using namespace tc;

constexpr int kTileRows = 128;
constexpr int kTokens = 64;        // of a tile
constexpr int kRowTiles = 2;
constexpr int kSoftmax = kRowTiles * kTileRows;
constexpr int kDecoders = 128;
constexpr int kPrefixThreads = kSoftmax + kDecoders + kRowTiles * 32;

constexpr int kErrK = 521, kErrV = 522, kErrP = 523, kErrS = 524, kErrEmpty = 525, kErrO = 526, kErrDrain = 527;

struct PrefixParams {
  Kv4AttendArgs a;
  int rows;      // requests * n * group
  int vec_q;     // rows of q take 16-byte loads
  uint64_t wait_ns;
};

template <int DT, int DP>
struct PrefixLayout {
  static constexpr int kQ = DT == SA_REP_BFLOAT16 ? 1 : 2;   // pieces of q, and of p s_v
  static constexpr int kChunks = (DP + 63) / 64;             // of 64 columns: a row of 128 bytes
  static constexpr int kQPiece = kChunks * kTileRows * 128;
  static constexpr int kK = kChunks * kTokens * 128;
  static constexpr int kV = DP * 128;
  static constexpr int kKStages = kQ == 1 ? 4 : 3, kVStages = kQ == 1 ? 3 : 2;
  static constexpr int kKeys = kRowTiles * kQ * kQPiece;
  static constexpr int kValues = kKeys + kKStages * kK;
  static constexpr int kParams = kValues + kVStages * kV;    // of each V stage: 64 keys' and 64 values' scales and offsets
  static constexpr int kInfo = kParams + kVStages * kTokens * 16;   // and its blocks' first tokens, and whether all see all
  static constexpr int kBars = kInfo + kVStages * 32;
  static constexpr int kBytes = kBars + (2 * kKStages + 2 * kVStages + 12) * 8 + 32 + 1024;
  static_assert(kBytes <= 227 * 1024, "shared memory");
  static_assert(kValues % 1024 == 0 && kKeys % 1024 == 0, "swizzled tiles start on 1024 bytes");
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
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
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

// The x lowest bits set (x may be anything).
__device__ __forceinline__ uint32_t low_bits(int x) {
  return x >= 32 ? 0xffffffffu : (x <= 0 ? 0u : (1u << x) - 1u);
}

// 32 scores in base 2: s_k S + x_k sum(Q); params: {s, s', x, x'} of each pair of tokens.
__device__ __forceinline__ void finish_scores(float (&s)[32], const float4* params, uint64_t qsum2) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float4 k = params[e];
    unpack2(fma2(pack2(s[2 * e], s[2 * e + 1]), pack2(k.x, k.y), mul2(pack2(k.z, k.w), qsum2)), s[2 * e], s[2 * e + 1]);
  }
}

// P of 32 tokens: p = 2^(s + off), its sum, sum(p x_v), and p s_v in pieces to TMEM.
// Without kWhole, bit e of `on` says whether token e is seen: a hidden one's parameters may be anything.
template <int kP, bool kWhole>
__device__ __forceinline__ void exp_chunk(float (&s)[32], float off, const float4* params, uint32_t on, uint64_t& sum2,
                                          uint64_t& z2, uint32_t to) {
  uint32_t pk[kP][16];
  const uint64_t off2 = pack2(off, off);
#pragma unroll
  for (int g = 0; g < 8; ++g) {   // four tokens: pairs 0 2 and 1 3
    float ps[4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float4 v = params[2 * g + e];
      const int t = 4 * g + 2 * e;
      float x, y;
      unpack2(add2(pack2(s[t], s[t + 1]), off2), x, y);
      x = ex2(x);
      y = ex2(y);
      const uint64_t p2 = pack2(x, y);
      sum2 = add2(sum2, p2);
      if (kWhole) {
        z2 = fma2(p2, pack2(v.z, v.w), z2);
        unpack2(mul2(p2, pack2(v.x, v.y)), ps[2 * e], ps[2 * e + 1]);
      } else {
        const bool a = (on >> t) & 1u, b = (on >> (t + 1)) & 1u;
        z2 = fma2(p2, pack2(a ? v.z : 0.0f, b ? v.w : 0.0f), z2);
        unpack2(mul2(p2, pack2(a ? v.x : 0.0f, b ? v.y : 0.0f)), ps[2 * e], ps[2 * e + 1]);
      }
    }
#pragma unroll
    for (int q = 0; q < kP; ++q) {
      const uint32_t lo = pack_bf16(ps[0], ps[2]), hi = pack_bf16(ps[1], ps[3]);
      pk[q][2 * g] = lo;
      pk[q][2 * g + 1] = hi;
      if (q + 1 < kP) {
        ps[0] -= __uint_as_float(lo << 16);
        ps[2] -= __uint_as_float(lo & 0xffff0000u);
        ps[1] -= __uint_as_float(hi << 16);
        ps[3] -= __uint_as_float(hi & 0xffff0000u);
      }
    }
  }
#pragma unroll
  for (int q = 0; q < kP; ++q) tmem_st16(to + q * (kTokens / 2), pk[q]);
}

__device__ __forceinline__ float max32(const float (&s)[32]) {
  float t[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
  for (int e = 4; e < 32; ++e) t[e & 3] = fmaxf(t[e & 3], s[e]);
  return fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
}

template <int DT, int DP>
__global__ void __launch_bounds__(kPrefixThreads, 1) prefix_tc_kernel(const __grid_constant__ PrefixParams p) {
  using L = PrefixLayout<DT, DP>;
  using T = typename Elem<DT>::T;
  constexpr int kQ = L::kQ, kKStages = L::kKStages, kVStages = L::kVStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t* kempty = kfull + kKStages;
  uint64_t* vfull = kempty + kKStages;
  uint64_t* vempty = vfull + kVStages;
  uint64_t* sfull = vempty + kVStages;   // [row tile][score buffer]
  uint64_t* pfull = sfull + 4;           // likewise
  uint64_t* pvdone = pfull + 4;          // [row tile]: a P V has ended
  uint64_t* drain = pvdone + 2;          // [row tile]: every product has
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  int* abort_word = reinterpret_cast<int*>(tmem_slot + 1);
  int* range = abort_word + 2;           // least and largest position of the CTA's rows

  const Kv4AttendArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = blockIdx.x, parts = gridDim.x, row0 = blockIdx.y * kSoftmax, hk = blockIdx.z;
  const int group = a.heads / a.c.heads;
  const int live = p.rows - row0 > kTileRows ? 2 : 1;   // row tiles with rows
  if (threadIdx.x == 0) {
    for (int s = 0; s < kKStages; ++s) {
      mbar_init(&kfull[s], kDecoders / 32);
      mbar_init(&kempty[s], live);
    }
    for (int s = 0; s < kVStages; ++s) {
      mbar_init(&vfull[s], kDecoders / 32);
      mbar_init(&vempty[s], live);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sfull[i], 1);
      mbar_init(&pfull[i], 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&pvdone[i], 1);
      mbar_init(&drain[i], 1);
    }
    abort_word[0] = abort_word[1] = 0;
    range[0] = 2147483647;
    range[1] = -1;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 12) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  __syncthreads();
  const int cap = a.width << a.c.page_shift;
  const int length = max(a.prefix_length[0], 0), bound = min(length, cap);
  if (length > cap && threadIdx.x == 0) report(a.status, kBadPrefix, 0);
  // a softmax thread's row: where it stands, -1 where it sees nothing
  int position = -1;
  const int row = row0 + (int)threadIdx.x;
  if (threadIdx.x < kSoftmax) {
    if (row < p.rows) {
      const int x = row / group, q = x / a.n;
      const int own = max(a.lengths[q], 0) - a.n + (x - q * a.n);   // only a request's own tokens ask
      if (own >= 0) position = (int)min((int64_t)length + own, (int64_t)2147483646);
    }
    const int least = __reduce_min_sync(0xffffffffu, position < 0 ? 2147483647 : position);
    const int most = __reduce_max_sync(0xffffffffu, position);
    if (lane == 0) {
      atomicMin(&range[0], least);
      atomicMax(&range[1], most);
    }
  }
  // Q: eight columns at a time, in the order 0 4 1 5 2 6 3 7
  for (int x = threadIdx.x; x < live * kTileRows * (DP / 8); x += kPrefixThreads) {
    const int r = x / (DP / 8), c8 = x - r * (DP / 8), at = row0 + r;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    if (at < p.rows) {
      const int y = at / group, q = y / a.n;
      const T* from = static_cast<const T*>(a.q) + q * a.q_r + (y - q * a.n) * a.q_n + (int64_t)(hk * group + at - y * group) * a.q_h + c8 * 8;
      if (p.vec_q && c8 * 8 + 8 <= a.c.d) {
        load8(v, from);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c8 * 8 + e < a.c.d) v[e] = to_f32(from[e]);
      }
    }
    uint8_t* to = smem + (r / kTileRows) * kQ * L::kQPiece + (c8 >> 3) * (kTileRows * 128) + (r % kTileRows) * 128 +
                  (((c8 & 7) ^ (r & 7)) << 4);
#pragma unroll
    for (int q = 0; q < kQ; ++q) {
      uint4 w;
      w.x = pack_bf16(v[0], v[4]);
      w.y = pack_bf16(v[1], v[5]);
      w.z = pack_bf16(v[2], v[6]);
      w.w = pack_bf16(v[3], v[7]);
      *reinterpret_cast<uint4*>(to + q * L::kQPiece) = w;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] -= __bfloat162float(__float2bfloat16_rn(v[e]));
    }
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // the visible blocks of 16 tokens, and this part's tiles of four
  const int p_lo = range[0], p_hi = range[1];
  const int window = (int)min(a.window, (int64_t)2147483647), sinks = (int)min(a.sinks, (int64_t)2147483647);
  KeyRanges kr{0, 0, 0};
  if (p_hi >= 0) kr = key_ranges(p_lo, p_hi, bound, a.window, a.sinks);
  const int sink_blocks = (int)((kr.first + 15) >> 4);
  const int win_begin = max((int)(kr.begin >> 4), sink_blocks), win_end = (int)((kr.end + 15) >> 4);
  const int blocks = sink_blocks + max(win_end - win_begin, 0);
  const int all = (blocks + 3) >> 2;
  const int first = (int)((int64_t)all * part / parts), tiles = (int)((int64_t)all * (part + 1) / parts) - first;
  const Abort ab{abort_word, a.status, p.wait_ns};

  if (threadIdx.x < kSoftmax) {
    // ------------------------------------------------------------ softmax rows
    const int t = warp >> 2;
    if (t < live) {
      const uint32_t at = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t tO = tmem + 256 + t * 128 + at;
      float qsum = 0.0f;
      {
        const int r = threadIdx.x % kTileRows;
#pragma unroll 1
        for (int x = 0; x < kQ * (DP / 8); ++x) {
          const int q = x / (DP / 8), c8 = x - q * (DP / 8);
          const uint4 w = *reinterpret_cast<const uint4*>(smem + (t * kQ + q) * L::kQPiece + (c8 >> 3) * (kTileRows * 128) +
                                                          r * 128 + (((c8 & 7) ^ (r & 7)) << 4));
          const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) qsum += __uint_as_float(ws[e] << 16) + __uint_as_float(ws[e] & 0xffff0000u);
        }
      }
      const uint64_t qsum2 = pack2(qsum, qsum);
      float m = -INFINITY, l = 0.0f, z = 0.0f;
      bool ok = true;
#pragma unroll 1
      for (int j = 0; j < tiles; ++j) {
        const int buf = j & 1, vs = j % kVStages;
        ok = mbar_wait_warp_lazy(&vfull[vs], (j / kVStages) & 1, ab, kErrV);
        if (ok) ok = mbar_wait_warp_lazy(&sfull[2 * t + buf], (j >> 1) & 1, ab, kErrS);
        if (!ok) break;
        tc_fence_after();
        const float4* kp = reinterpret_cast<const float4*>(smem + L::kParams + vs * kTokens * 16);
        const float4* vp = kp + kTokens / 2;
        const int* info = reinterpret_cast<const int*>(smem + L::kInfo + vs * 32);
        const uint32_t ts = tmem + t * 128 + buf * kTokens + at;
        float s0[32], s1[32];
        tmem_ld32(ts, s0);
        tmem_ld32(ts + 32, s1);
        tmem_wait_ld();
        tie32(s0);
        tie32(s1);
        finish_scores(s0, kp, qsum2);
        finish_scores(s1, kp + 16, qsum2);
        uint32_t on0 = 0xffffffffu, on1 = 0xffffffffu;
        const bool whole = info[4] != 0;
        if (!whole) {
          // 16 tokens from info[b] on: j < bound and (j > position - window or j < sinks); j <= position always
          auto seen = [&](int b) {
            const int j0 = info[b];
            if (j0 < 0) return 0u;
            const uint32_t near = position - j0 < window ? 0xffffu : 0xffffu & ~low_bits(position - j0 - window + 1);
            return low_bits(bound - j0) & (near | low_bits(sinks - j0)) & 0xffffu;
          };
          on0 = seen(0) | seen(1) << 16;
          on1 = seen(2) | seen(3) << 16;
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            s0[e] = (on0 >> e) & 1u ? s0[e] : -INFINITY;
            s1[e] = (on1 >> e) & 1u ? s1[e] : -INFINITY;
          }
        }
        const float top = fmaxf(max32(s0), max32(s1));
        const bool move = top > m + kMove;
        if (__any_sync(0xffffffffu, move)) {
          const float to = move ? top : m;
          const float alpha = move ? ex2(m - to) : 1.0f;   // m = -inf: 0
          m = to;
          l *= alpha;
          z *= alpha;
          if (j > 0) {   // the product of the tile before may still run (that of the one before it ended before S(j))
            ok = mbar_wait_warp_lazy(&pvdone[t], (j - 1) & 1, ab, kErrO);
            if (!ok) break;
            tc_fence_after();
            scale_row(tO, DP, alpha);
          }
        }
        const float off = kShift - (m == -INFINITY ? 0.0f : m);
        uint64_t sum2 = 0, z2 = 0;
        if (whole) {
          exp_chunk<kQ, true>(s0, off, vp, on0, sum2, z2, ts);
          exp_chunk<kQ, true>(s1, off, vp + 16, on1, sum2, z2, ts + 16);
        } else {
          exp_chunk<kQ, false>(s0, off, vp, on0, sum2, z2, ts);
          exp_chunk<kQ, false>(s1, off, vp + 16, on1, sum2, z2, ts + 16);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&pfull[2 * t + buf]);
        float x, y;
        unpack2(sum2, x, y);
        l += x + y;
        unpack2(z2, x, y);
        z += x + y;
      }
      if (ok && tiles > 0) {
        // not pvdone: P V of the last tile but one may still run too, and a parity tells only neighbours apart
        ok = mbar_wait_warp_lazy(&drain[t], 0, ab, kErrO);
        tc_fence_after();
      }
      // this part's sums: [part][key head][columns / 4][row][4]
      const int64_t of = (int64_t)part * a.c.heads + hk;
      const bool some = ok && tiles > 0 && position >= 0 && m != -INFINITY;
      if (row < p.rows) a.part_ml[of * p.rows + row] = some || (position >= 0 && !(l == 0.0f)) ? make_float2(m, l) : make_float2(-INFINITY, 0.0f);
#pragma unroll 1
      for (int c = 0; c < DP; c += 16) {
        float o[16];
        if (tiles > 0) {
          tmem_ld16(tO + c, o);
          tmem_wait_ld();
          tie16(o);
        }
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          if (row < p.rows)
            *reinterpret_cast<float4*>(a.part_o + ((of * (DP / 4) + (c + e) / 4) * p.rows + row) * 4) =
                some ? make_float4(o[e] + z, o[e + 1] + z, o[e + 2] + z, o[e + 3] + z) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
      tc_fence_before();
    }
  } else if (threadIdx.x < kSoftmax + kDecoders) {
    // ------------------------------------------------------------ codes to tiles
    constexpr int kPieces = DP / 32;                               // 16-byte pieces of a key row
    constexpr int kKLoads = (kTokens * kPieces + kDecoders - 1) / kDecoders;
    const int d = threadIdx.x - kSoftmax;
    const int v_chunk = d & 7, v_quad = d >> 3;                    // 8 tokens, 8 columns (quad < DP / 8)
    const int64_t cell0 = (int64_t)hk << a.c.page_shift;
    const int64_t page_step = (int64_t)a.c.heads << a.c.page_shift;
    const int page_mask = (1 << a.c.page_shift) - 1;
    auto token_of = [&](int v) { return (v < sink_blocks ? v : win_begin + v - sink_blocks) << 4; };
    const float sc = a.scale * 1.4426950408889634f;
    // first token (-1: none) and page of 32 blocks, one a lane: eight tiles
    int token_l = -1, page_l = 0;
    auto fetch = [&](int j) {
      const int v = (first + j) * 4 + lane;
      token_l = -1;
      page_l = 0;
      if (v < blocks && lane < (tiles - j) * 4) {
        const int token = token_of(v), page = __ldg(a.prefix_table + (token >> a.c.page_shift));
        if (page < 0 || page >= a.c.pages) {
          if (d < 32) report(a.status, kBadPage, page);
        } else {
          token_l = token;
          page_l = page;
        }
      }
    };
    struct Raw {
      uint4 k[kKLoads], v[2];
      uint32_t kp, vp;
      int block;     // lane b < 4: first token of block b
    };
    auto load = [&](Raw& x, int j) {
      if ((j & 7) == 0) fetch(j);
      const int b0 = (j & 7) * 4;
      // a block's first cell in the cache, or that of any valid one where there is none
      auto cell_of = [&](int b) {
        const int token = __shfl_sync(0xffffffffu, token_l, b0 + b), page = __shfl_sync(0xffffffffu, page_l, b0 + b);
        return (int64_t)page * page_step + cell0 + (max(token, 0) & page_mask);
      };
      x.block = __shfl_sync(0xffffffffu, token_l, b0 + (lane & 3));
#pragma unroll
      for (int i = 0; i < kKLoads; ++i) {
        const int u = i * kDecoders + d, token = (u / (8 * kPieces)) * 8 + (u & 7), piece = (u >> 3) % kPieces;
        const int64_t cell = cell_of((token >> 4) & 3);
        if (token < kTokens)
          x.k[i] = __ldg(reinterpret_cast<const uint4*>(a.c.k_codes + (cell + (token & 15)) * (DP / 2)) + piece);
      }
      const int64_t vc = cell_of(v_chunk >> 1);
      if (v_quad < DP / 8) {
        const uint8_t* from = a.c.v_codes + (vc + (v_chunk & 1) * 8) * (DP / 2) + v_quad * 16;
        x.v[0] = __ldg(reinterpret_cast<const uint4*>(from));
        x.v[1] = __ldg(reinterpret_cast<const uint4*>(from + 4 * (DP / 2)));
      }
      const int64_t pc = cell_of((d >> 4) & 3) + (d & 15);
      if (d < kTokens) {
        x.kp = __ldg(reinterpret_cast<const uint32_t*>(a.c.k_params) + pc);
        x.vp = __ldg(reinterpret_cast<const uint32_t*>(a.c.v_params) + pc);
      }
    };
    bool ok = true;
    auto put = [&](const Raw& x, int j) {
      const int ks = j % kKStages, vs = j % kVStages;
      if (j >= kKStages) ok = mbar_wait_warp_lazy(&kempty[ks], ((j / kKStages) - 1) & 1, ab, kErrEmpty);
      if (!ok) return;
      uint8_t* kt = smem + L::kKeys + ks * L::kK;
#pragma unroll
      for (int i = 0; i < kKLoads; ++i) {
        const int u = i * kDecoders + d, token = (u / (8 * kPieces)) * 8 + (u & 7), piece = (u >> 3) % kPieces;
        if (token < kTokens) {
          const uint32_t ws[4] = {x.k[i].x, x.k[i].y, x.k[i].z, x.k[i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int c8 = piece * 4 + e;
            uint4 w;
            w.x = codes<0, -8>(ws[e]);
            w.y = codes<1, -8>(ws[e]);
            w.z = codes<2, -8>(ws[e]);
            w.w = codes<3, -8>(ws[e]);
            *reinterpret_cast<uint4*>(kt + (c8 >> 3) * (kTokens * 128) + token * 128 + (((c8 & 7) ^ (token & 7)) << 4)) = w;
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&kfull[ks]);
      if (j >= kVStages) ok = mbar_wait_warp_lazy(&vempty[vs], ((j / kVStages) - 1) & 1, ab, kErrEmpty);
      if (!ok) return;
      uint8_t* vt = smem + L::kValues + vs * L::kV;
      if (v_quad < DP / 8) {
        const uint32_t w0[4] = {x.v[0].x, x.v[0].y, x.v[0].z, x.v[0].w}, w1[4] = {x.v[1].x, x.v[1].y, x.v[1].z, x.v[1].w};
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          uint8_t* to = vt + (v_quad * 8 + 2 * b) * 128;
          *reinterpret_cast<uint4*>(to + ((v_chunk ^ (2 * b)) << 4)) =
              make_uint4(codes<0, -8>(w0[b]), codes<2, -8>(w0[b]), codes<0, -8>(w1[b]), codes<2, -8>(w1[b]));
          *reinterpret_cast<uint4*>(to + 128 + ((v_chunk ^ (2 * b + 1)) << 4)) =
              make_uint4(codes<1, -8>(w0[b]), codes<3, -8>(w0[b]), codes<1, -8>(w1[b]), codes<3, -8>(w1[b]));
        }
      }
      const int mine = __shfl_sync(0xffffffffu, x.block, (d >> 4) & 3);
      if (d < kTokens) {
        const bool in = mine >= 0 && mine + (d & 15) < bound;
        const float2 k = params(in ? x.kp : 0u), v = params(in ? x.vp : 0u);
        float* kp = reinterpret_cast<float*>(smem + L::kParams + vs * kTokens * 16) + (d >> 1) * 4 + (d & 1);
        kp[0] = k.x * sc;
        kp[2] = fmaf(8.0f, k.x, k.y) * sc;
        float* vp = kp + 2 * kTokens;
        vp[0] = v.x;
        vp[2] = fmaf(8.0f, v.x, v.y);
      }
      // whether every row that sees anything sees all 64 tokens
      const bool whole = __all_sync(0xffffffffu, x.block >= 0 && x.block + 16 <= bound && (p_hi - x.block < window || x.block + 16 <= sinks));
      if (d < 4) reinterpret_cast<int*>(smem + L::kInfo + vs * 32)[d] = x.block;
      if (d == 4) reinterpret_cast<int*>(smem + L::kInfo + vs * 32)[4] = whole;
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&vfull[vs]);
    };
    Raw x, y;
    if (tiles > 0) load(x, 0);
    if (tiles > 1) load(y, 1);
#pragma unroll 1
    for (int j = 0; j < tiles && ok; j += 2) {
      put(x, j);
      if (j + 2 < tiles) load(x, j + 2);
      if (j + 1 < tiles && ok) {
        put(y, j + 1);
        if (j + 3 < tiles) load(y, j + 3);
      }
    }
  } else {
    // ------------------------------------------------------------ products of row tile t
    const int t = warp - 12;
    if (t < live) {
      constexpr uint32_t id_s = idesc_f16(kTileRows, kTokens, true, false, false);
      constexpr uint32_t id_pv = idesc_f16(kTileRows, DP, true, false, false);
      const uint32_t q_smem = smem_u32(smem) + t * kQ * L::kQPiece, k_smem = smem_u32(smem + L::kKeys), v_smem = smem_u32(smem + L::kValues);
      const uint32_t tS = tmem + t * 128, tO = tmem + 256 + t * 128;
      auto scores = [&](int j) {   // by one lane
        const uint64_t kd = sdesc_sw128(k_smem + (j % kKStages) * L::kK, 16, 1024);
#pragma unroll
        for (int q = 0; q < kQ; ++q) {
          const uint64_t qd = sdesc_sw128(q_smem + q * L::kQPiece, 16, 1024);
#pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk)
            mma_f16_ss(tS + (j & 1) * kTokens, qd + (uint64_t)(((kk >> 2) * (kTileRows * 128) + (kk & 3) * 32) >> 4),
                       kd + (uint64_t)(((kk >> 2) * (kTokens * 128) + (kk & 3) * 32) >> 4), id_s, q > 0 || kk > 0 ? 1u : 0u);
        }
        mma_commit(&sfull[2 * t + (j & 1)]);
        mma_commit(&kempty[j % kKStages]);
      };
      bool ok = true;
#pragma unroll 1
      for (int j = 0; j < min(tiles, 2) && ok; ++j) {
        ok = mbar_wait_warp_lazy(&kfull[j % kKStages], (j / kKStages) & 1, ab, kErrK);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) scores(j);
        __syncwarp();
      }
#pragma unroll 1
      for (int j = 0; j < tiles && ok; ++j) {
        const int vs = j % kVStages;
        ok = mbar_wait_warp_lazy(&vfull[vs], (j / kVStages) & 1, ab, kErrV);
        if (ok) ok = mbar_wait_warp_lazy(&pfull[2 * t + (j & 1)], (j >> 1) & 1, ab, kErrP);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t vd = sdesc_sw128(v_smem + vs * L::kV, 16, 1024);
#pragma unroll
          for (int q = kQ - 1; q >= 0; --q)
#pragma unroll
            for (int kk = 0; kk < kTokens / 16; ++kk)
              mma_f16_ts(tO, tS + (j & 1) * kTokens + q * (kTokens / 2) + kk * 8, vd + (uint64_t)((kk * 32) >> 4), id_pv,
                         j > 0 || q < kQ - 1 || kk > 0 ? 1u : 0u);
          mma_commit(&pvdone[t]);
          mma_commit(&vempty[vs]);
        }
        __syncwarp();
        if (j + 2 < tiles) {
          ok = mbar_wait_warp_lazy(&kfull[(j + 2) % kKStages], ((j + 2) / kKStages) & 1, ab, kErrK);
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
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_dealloc(tmem, 512);
}

template <int DT, int DP>
int launch_prefix(const Kv4AttendArgs& a, int64_t rows, cudaStream_t s) {
  using L = PrefixLayout<DT, DP>;
  auto kern = prefix_tc_kernel<DT, DP>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes);
  if (e != cudaSuccess) return set_error(SA_ERR_CUDA, "kv4 prefix smem attribute: %s", cudaGetErrorString(e));
  PrefixParams p{};
  p.a = a;
  p.rows = (int)rows;
  p.vec_q = rows_aligned(a.q, elem_size(a.dtype), a.q_r | a.q_n, a.q_h);
  p.wait_ns = wait_limit_ns();
  const int64_t pairs = ceil_div(rows, kSoftmax);
  if (a.c.heads > 65535 || pairs > 65535) return set_error(SA_ERR_UNSUPPORTED, "kv4 prefix: grid too large");
  kern<<<dim3((unsigned)a.parts, (unsigned)pairs, (unsigned)a.c.heads), kPrefixThreads, L::kBytes, s>>>(p);
  return check_launch("kv4 prefix_tc_kernel");
}

}  // namespace

bool kv4_prefix_tc_takes(const Kv4AttendArgs& a, int64_t rows) {
  return a.dtype != SA_REP_FLOAT32 && a.c.dp <= 128 && rows > 32;
}

// Parts of the prefix, each a CTA for every pair of row tiles and key head: as many as
// fill the GPU, of two tiles at least.
int kv4_prefix_tc_parts(const Kv4AttendArgs& a, int64_t rows) {
  const int64_t longest = std::min<int64_t>((int64_t)a.prefix_width << a.c.page_shift, a.window + a.sinks + a.n);
  const int64_t ctas = ceil_div(rows, kSoftmax) * a.c.heads;
  return (int)std::max<int64_t>(1, std::min(148 / ctas, ceil_div(longest, 2 * kTokens)));
}

int launch_kv4_prefix_tc(const Kv4AttendArgs& a, int64_t rows, cudaStream_t s) {
  const bool b = a.dtype == SA_REP_BFLOAT16;
  if (a.c.dp == 32) return b ? launch_prefix<SA_REP_BFLOAT16, 32>(a, rows, s) : launch_prefix<SA_REP_FLOAT16, 32>(a, rows, s);
  if (a.c.dp == 64) return b ? launch_prefix<SA_REP_BFLOAT16, 64>(a, rows, s) : launch_prefix<SA_REP_FLOAT16, 64>(a, rows, s);
  return b ? launch_prefix<SA_REP_BFLOAT16, 128>(a, rows, s) : launch_prefix<SA_REP_FLOAT16, 128>(a, rows, s);
}

}  // namespace sa
