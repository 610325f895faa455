// Eviction: requests longer than `limit` keep `keep` tokens of each key head -- the
// first ones, the newest ones and, between, those of the largest weights (of equal ones
// the lowest) -- moved up in their order to the request's first places, in place.
//
// One CTA per (request, key head).  Its weights stand in shared memory (as whole numbers of
// the same order) while the border between kept and dropped ones is found by three passes
// over their digits and a scan in order turns them into the list of what is kept.  Token
// j's new place is no higher than j, so places are filled from the first on, a chunk at a
// time: all of a chunk is read before any of it is written, and what later chunks read lies
// behind, so the next chunks are on their way while one is written.
//
// 48 requests of 4000..8000 tokens to 2048, 8 key heads of 128: 97 us (215 MB, 33 us):
// the barriers between loads and stores, and the instructions that turn four tokens'
// bytes into a word.  With one chunk of 64 on its way and byte loads 298; with digits of 8
// bits and a list made by all warps in step 127.  One CTA per (request, key head) leaves most of the GPU idle where
// requests are few: one of 16000 tokens to 4000 takes 106 us with the return of its pages, one of 100000 to 8000 643.
#include <algorithm>

#include "kv4.cuh"

namespace sa {

namespace {

constexpr int kThreads = 384;
constexpr int kWarps = kThreads / 32;
constexpr int kChunk = 96;   // tokens moved at a time: of width 128, two units a thread
constexpr int kAhead = 3;    // chunks on their way
constexpr int kLoads = 8;    // weights on their way, a thread
constexpr int kDigits = 2048;
static_assert(3 * kChunk <= kThreads, "a thread moves one of a token's single words");
static_assert(kDigits % 8 == 0 && kDigits / 8 <= kThreads && kDigits / 8 % 32 == 0, "eight digits a thread, in whole warps");

// A weight as a whole number of the same order; NaN is the largest.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.0f);   // -0 becomes 0
  return b >> 31 ? ~b : b | 0x80000000u;
}

template <int DP>
__global__ void __launch_bounds__(kThreads, 3) evict_kernel(const Kv4EvictArgs a) {
  constexpr int bytes = DP / 2;                                      // of a row's codes
  constexpr int kSide = kChunk * bytes / 16;                         // 16-byte units of a chunk's keys, or of its values
  constexpr int kUnits = (2 * kSide + kThreads - 1) / kThreads;      // of a thread
  constexpr int kRing = kAhead + 3;
  __shared__ int64_t src[kRing][kChunk], dst[kRing][kChunk];   // of chunks' tokens: cells they come from and go to
  __shared__ int count_of[kDigits];
  __shared__ int warp_sum[kDigits / 256];
  __shared__ int part[2][kWarps];
  __shared__ int digit, below;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int h = blockIdx.x, r = blockIdx.y;
  const int shift = a.c.page_shift, mask = (1 << shift) - 1;
  const int cap = a.width << shift;
  const int whole = max(a.lengths[r], 0), length = min(whole, cap);
  if (whole > cap && h == 0 && tid == 0) report(a.status, kBadLength, r);
  const int32_t* table = a.tables + (int64_t)r * a.width;
  int32_t* kept = a.kept + ((int64_t)r * a.c.heads + h) * a.keep;
  if (length <= a.limit) {
    for (int j = tid; j < a.keep; j += kThreads) kept[j] = j < length ? j : -1;
    return;
  }
  // the place of token j of this head, -1 without a page
  auto cell = [&](int j) -> int64_t {
    const int page = __ldg(table + (j >> shift));
    if (page < 0 || page >= a.c.pages) return -1;
    return (((int64_t)page * a.c.heads + h) << shift) + (j & mask);
  };
  // the weights' order, then (in the same memory) the list; what does not fit is read where it stands
  extern __shared__ uint32_t held[];
  const int fits = min(a.fits, length);
  auto key_of = [&](int j) {
    const int64_t at = cell(j);
    return at < 0 ? 0u : order_of(a.weights[at]);
  };
  for (int j = tid; j < fits; j += kThreads * kLoads) {
    uint32_t k[kLoads];
#pragma unroll
    for (int x = 0; x < kLoads; ++x) k[x] = j + x * kThreads < fits ? key_of(j + x * kThreads) : 0u;
#pragma unroll
    for (int x = 0; x < kLoads; ++x)
      if (j + x * kThreads < fits) held[j + x * kThreads] = k[x];
  }
  auto key = [&](int j) { return j < fits ? held[j] : key_of(j); };
  __syncthreads();
  for (int row = tid; row << shift < length; row += kThreads)
    if (h == 0 && (table[row] < 0 || table[row] >= a.c.pages)) report(a.status, kBadPage, table[row]);
  const int begin = a.first, end = length - a.last, want = a.keep - a.first - a.last;
  uint32_t border = 0, top = 0;
  int ties = want;
  // digits of 11, 11 and 10 bits: a weight's exponent alone would send most of them to a few counters
  for (int at = 21; want > 0; at = at > 11 ? at - 11 : 0) {
    const uint32_t digits = at == 0 ? 1023u : 2047u;
    for (int x = tid; x < kDigits; x += kThreads) count_of[x] = 0;
    __syncthreads();
    for (int j = begin + tid; j < end; j += kThreads) {
      const uint32_t k = key(j);
      if ((k & top) == border) atomicAdd(&count_of[(k >> at) & digits], 1);
    }
    __syncthreads();
    // eight digits a thread, from the top, and the sums before them
    int sum = 0, upto = 0;
    if (tid < kDigits / 8) {
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += count_of[kDigits - 1 - 8 * tid - e];
      upto = sum;
#pragma unroll
      for (int x = 1; x < 32; x *= 2) {
        const int y = __shfl_up_sync(0xffffffffu, upto, x);
        if (lane >= x) upto += y;
      }
      if (lane == 31) warp_sum[warp] = upto;
    }
    __syncthreads();
    if (tid < kDigits / 8) {
      for (int w = 0; w < warp; ++w) upto += warp_sum[w];
      int before = upto - sum;
      if (before < ties && ties <= upto)
        for (int e = 0; e < 8; ++e) {
          const int c = count_of[kDigits - 1 - 8 * tid - e];
          if (before + c >= ties) {
            digit = kDigits - 1 - 8 * tid - e;
            below = before;
            break;
          }
          before += c;
        }
    }
    __syncthreads();
    border |= (uint32_t)digit << at;
    top |= digits << at;
    ties -= below;
    const bool all = count_of[digit] == ties;   // the whole digit is kept
    __syncthreads();
    if (all || at == 0) break;
  }
  // the list, in order: each warp counts what stays of a run of tokens, and, when all have, writes it
  const int run = (((length + kWarps - 1) / kWarps) + 31) & ~31, run_end = min((warp + 1) * run, length);
  auto stays = [&](int j, bool& over, bool& same) {
    const bool fixed = j < begin || j >= end;
    const uint32_t k = fixed || j >= run_end ? 0u : key(j) & top;
    over = j < run_end && (fixed || (want > 0 && k > border));
    same = j < run_end && !fixed && want > 0 && k == border;
  };
  int overs = 0, equal = 0;
  for (int j0 = warp * run; j0 < run_end; j0 += 32) {
    bool over, same;
    stays(j0 + lane, over, same);
    overs += __popc(__ballot_sync(0xffffffffu, over));
    equal += __popc(__ballot_sync(0xffffffffu, same));
  }
  if (lane == 0) {
    part[0][warp] = overs;
    part[1][warp] = equal;
  }
  __syncthreads();
  int at = 0;
  equal = 0;
  for (int w = 0; w < warp; ++w) {
    at += part[0][w];
    equal += part[1][w];
  }
  at += min(equal, ties);   // of the equal ones the first `ties` stay
  for (int j0 = warp * run; j0 < run_end; j0 += 32) {
    bool over, same;
    stays(j0 + lane, over, same);
    const unsigned all_over = __ballot_sync(0xffffffffu, over), all_same = __ballot_sync(0xffffffffu, same);
    const unsigned before = (1u << lane) - 1;
    const int s = equal + __popc(all_same & before);
    if (over || (same && s < ties)) kept[at + __popc(all_over & before) + min(s, ties) - min(equal, ties)] = j0 + lane;
    at += __popc(all_over) - min(equal, ties);
    equal += __popc(all_same);
    at += min(equal, ties);
  }
  __syncthreads();
  for (int j = tid; j < min(fits, a.keep); j += kThreads) held[j] = kept[j];   // the weights are done with
  __syncthreads();
  // the tokens, a chunk of new places at a time
  const int which = tid / kChunk, js = tid - which * kChunk;   // keys' parameters, values', weights
  auto cells = [&](int j0) {
    if (tid >= kChunk || j0 >= a.keep) return;
    const int j = j0 + tid, at = j0 / kChunk % kRing;
    int64_t from = -1, to = -1;
    if (j < ((a.keep + 3) & ~3)) {   // places behind `keep` in its word of values take what they hold
      to = cell(j);
      from = j < a.keep ? cell(j < fits ? (int)held[j] : kept[j]) : to;
    }
    src[at][tid] = from;
    dst[at][tid] = to;
  };
  struct Part {
    uint4 w[kUnits];
    uint32_t single;
  };
  // unit u: 16 bytes of a key row, or, behind those, four tokens' bytes of four column pairs
  auto load = [&](Part& c, int j0) {
    if (j0 >= a.keep) return;
    const int64_t* from = src[j0 / kChunk % kRing];
#pragma unroll
    for (int x = 0; x < kUnits; ++x) {
      const int u = x * kThreads + tid;
      c.w[x] = make_uint4(0, 0, 0, 0);
      if (u < kSide) {
        const int j = u / (bytes / 16);
        if (from[j] >= 0) c.w[x] = *reinterpret_cast<const uint4*>(a.c.k_codes + from[j] * bytes + u % (bytes / 16) * 16);
      } else if (u < 2 * kSide) {
        const int v = u - kSide, j = v / (bytes / 4) * 4, b = v % (bytes / 4) * 4;
        uint4 t[4];
        int byte[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int64_t f = from[j + e];
          t[e] = f < 0 ? make_uint4(0, 0, 0, 0) : *reinterpret_cast<const uint4*>(a.c.v_codes + (f & ~3ll) * bytes + b * 4);
          byte[e] = (int)(f & 3);
        }
        const uint32_t lo = byte[0] | (4 + byte[1]) << 4, hi = byte[2] | (4 + byte[3]) << 4;
        auto join = [&](uint32_t p, uint32_t q, uint32_t r, uint32_t s) {
          return __byte_perm(__byte_perm(p, q, lo), __byte_perm(r, s, hi), 0x5410);
        };
        c.w[x] = make_uint4(join(t[0].x, t[1].x, t[2].x, t[3].x), join(t[0].y, t[1].y, t[2].y, t[3].y),
                            join(t[0].z, t[1].z, t[2].z, t[3].z), join(t[0].w, t[1].w, t[2].w, t[3].w));
      }
    }
    c.single = 0;
    if (which < 3 && j0 + js < a.keep && from[js] >= 0)
      c.single = which == 0   ? reinterpret_cast<const uint32_t*>(a.c.k_params)[from[js]]
                 : which == 1 ? reinterpret_cast<const uint32_t*>(a.c.v_params)[from[js]]
                              : __float_as_uint(a.weights[from[js]]);
  };
  auto store = [&](const Part& c, int j0) {
    if (j0 >= a.keep) return;
    const int64_t* from = src[j0 / kChunk % kRing];
    const int64_t* to = dst[j0 / kChunk % kRing];
#pragma unroll
    for (int x = 0; x < kUnits; ++x) {
      const int u = x * kThreads + tid;
      if (u < kSide) {
        const int j = u / (bytes / 16);
        if (j0 + j < a.keep && to[j] >= 0 && from[j] >= 0)
          *reinterpret_cast<uint4*>(a.c.k_codes + to[j] * bytes + u % (bytes / 16) * 16) = c.w[x];
      } else if (u < 2 * kSide) {
        const int v = u - kSide, j = v / (bytes / 4) * 4, b = v % (bytes / 4) * 4;
        if (to[j] >= 0) *reinterpret_cast<uint4*>(a.c.v_codes + to[j] * bytes + b * 4) = c.w[x];
      }
    }
    if (which < 3 && j0 + js < a.keep && to[js] >= 0) {
      if (which == 0) reinterpret_cast<uint32_t*>(a.c.k_params)[to[js]] = c.single;
      if (which == 1) reinterpret_cast<uint32_t*>(a.c.v_params)[to[js]] = c.single;
      if (which == 2) a.weights[to[js]] = __uint_as_float(c.single);
    }
  };
  int begun = 0;   // the first tokens are where they were: the list ascends
  while (begun + kChunk <= a.keep) {
    const int last = begun + kChunk - 1;
    if ((last < fits ? (int)held[last] : kept[last]) != last) break;
    begun += kChunk;
  }
  // A barrier stands between a chunk's loads and its stores, and behind what says where it goes: of round i,
  // chunk i + kAhead + 1's cells, chunk i + kAhead's loads, barrier, chunk i's stores.
  Part parts[kAhead + 1];
#pragma unroll
  for (int x = 0; x <= kAhead; ++x) cells(begun + x * kChunk);
  __syncthreads();
#pragma unroll
  for (int x = 0; x < kAhead; ++x) load(parts[x], begun + x * kChunk);
  for (int j0 = begun; j0 < a.keep; j0 += (kAhead + 1) * kChunk) {
#pragma unroll
    for (int x = 0; x <= kAhead; ++x) {
      const int j1 = j0 + x * kChunk;
      cells(j1 + (kAhead + 1) * kChunk);
      load(parts[(x + kAhead) % (kAhead + 1)], j1 + kAhead * kChunk);
      __syncthreads();
      store(parts[x], j1);
    }
  }
  __syncthreads();
  // whoever stands in the places behind starts from zero
  for (int j = a.keep + tid; j < (((int64_t)length + mask) & ~(int64_t)mask); j += kThreads) {
    const int64_t to = cell(j);
    if (to >= 0) a.weights[to] = 0.0f;
  }
}

// Tokens whose weights shared memory holds: 64 KB, beside 17.5 of the CTA's own.  Three CTAs an SM while the table
// allows up to 14800 tokens, two above.
constexpr int kFits = 16384;

template <int DP>
int launch_evict(const Kv4EvictArgs& a, cudaStream_t s) {
  static std::atomic<uint64_t> allowed{0};
  const int rc = allow_shared(evict_kernel<DP>, kFits * 4, allowed, "kv4 evict");
  if (rc) return rc;
  evict_kernel<DP><<<dim3((unsigned)a.c.heads, (unsigned)a.requests), kThreads, a.fits * 4, s>>>(a);
  return check_launch("kv4 evict_kernel");
}

}  // namespace

int launch_kv4_evict(const Kv4EvictArgs& a, cudaStream_t s) {
  Kv4EvictArgs b = a;
  b.fits = (int)std::min<int64_t>((int64_t)a.width << a.c.page_shift, kFits);
  if (a.c.dp == 32) return launch_evict<32>(b, s);
  if (a.c.dp == 64) return launch_evict<64>(b, s);
  return a.c.dp == 128 ? launch_evict<128>(b, s) : launch_evict<256>(b, s);
}

}  // namespace sa
