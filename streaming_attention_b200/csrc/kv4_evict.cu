// Eviction: requests longer than `limit` keep `keep` tokens of each key head -- the
// first ones, the newest ones and, between, those of the largest weights (of equal ones
// the lowest) -- moved up in their order to the request's first places, in place.
//
// One CTA per (request, key head).  The border between kept and dropped weights is found
// by four passes over their digits; a scan in order then writes the list of what is kept.
// Token j's new place is no higher than j, so places are filled from the first on, a
// chunk at a time: all of a chunk is read before any of it is written, and what later
// chunks read lies behind.
#include <algorithm>

#include "kv4.cuh"

namespace sa {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kChunk = 64;   // tokens moved at a time
constexpr int kMaxRow = 128;                                            // bytes of a row's codes
constexpr int kPieces = kChunk * (kMaxRow / 16) / kThreads;             // 16-byte pieces of keys, a thread
constexpr int kWords = kChunk / 4 * kMaxRow / kThreads;                 // words of values, a thread
static_assert(kPieces * kThreads == kChunk * (kMaxRow / 16) && kWords * kThreads == kChunk / 4 * kMaxRow, "whole shares");
static_assert(3 * kChunk <= kThreads, "a thread moves one of a token's single words");

// A weight as a whole number of the same order; NaN is the largest.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.0f);   // -0 becomes 0
  return b >> 31 ? ~b : b | 0x80000000u;
}

__global__ void __launch_bounds__(kThreads) evict_kernel(const Kv4EvictArgs a) {
  __shared__ int count_of[256];
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
    const int page = table[j >> shift];
    if (page < 0 || page >= a.c.pages) return -1;
    return (((int64_t)page * a.c.heads + h) << shift) + (j & mask);
  };
  auto key = [&](int j) {
    const int64_t at = cell(j);
    return at < 0 ? 0u : order_of(a.weights[at]);
  };
  for (int row = tid; row << shift < length; row += kThreads)
    if (h == 0 && (table[row] < 0 || table[row] >= a.c.pages)) report(a.status, kBadPage, table[row]);
  const int begin = a.first, end = length - a.last, want = a.keep - a.first - a.last;
  uint32_t border = 0, top = 0;
  int ties = want;
  for (int at = 24; at >= 0 && want > 0; at -= 8) {
    if (tid < 256) count_of[tid] = 0;
    __syncthreads();
    for (int j = begin + tid; j < end; j += kThreads) {
      const uint32_t k = key(j);
      if ((k & top) == border) atomicAdd(&count_of[(k >> at) & 255], 1);
    }
    __syncthreads();
    if (warp == 0) {   // a lane eight digits, from the top
      int sum = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += count_of[255 - 8 * lane - e];
      int upto = sum;
#pragma unroll
      for (int x = 1; x < 32; x *= 2) {
        const int y = __shfl_up_sync(0xffffffffu, upto, x);
        if (lane >= x) upto += y;
      }
      int before = upto - sum;
      if (before < ties && ties <= upto)
        for (int e = 0; e < 8; ++e) {
          const int c = count_of[255 - 8 * lane - e];
          if (before + c >= ties) {
            digit = 255 - 8 * lane - e;
            below = before;
            break;
          }
          before += c;
        }
    }
    __syncthreads();
    border |= (uint32_t)digit << at;
    top |= 255u << at;
    ties -= below;
    const bool all = count_of[digit] == ties;   // the whole digit is kept
    __syncthreads();
    if (all) break;
  }
  // the list, in order
  int at = 0, equal = 0;
  for (int j0 = 0; j0 < length; j0 += kThreads) {
    const int j = j0 + tid;
    const bool fixed = j < begin || (j >= end && j < length);
    const uint32_t k = j >= begin && j < end ? key(j) & top : 0;
    const bool over = fixed || (j >= begin && j < end && want > 0 && k > border);
    const bool same = j >= begin && j < end && want > 0 && k == border;
    const unsigned overs = __ballot_sync(0xffffffffu, over), sames = __ballot_sync(0xffffffffu, same);
    if (lane == 0) {
      part[0][warp] = __popc(overs);
      part[1][warp] = __popc(sames);
    }
    __syncthreads();
    const unsigned before = (1u << lane) - 1;
    int o = __popc(overs & before), s = equal + __popc(sames & before), o_all = 0, s_all = 0;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) {
      if (x < warp) o += part[0][x], s += part[1][x];
      o_all += part[0][x];
      s_all += part[1][x];
    }
    // of the equal ones before this one, no more than `ties` were taken
    if (over || (same && s < ties)) kept[at + o + min(s, ties) - min(equal, ties)] = j;
    at += o_all + min(equal + s_all, ties) - min(equal, ties);
    equal += s_all;
    __syncthreads();
  }
  // the tokens, a chunk of new places at a time
  const int bytes = a.c.dp >> 1, pieces = bytes >> 4;
  for (int j0 = 0; j0 < a.keep; j0 += kChunk) {
    const int n = min(kChunk, a.keep - j0);
    if (kept[j0 + n - 1] == j0 + n - 1) continue;   // all where they were: kept[] ascends
    uint4 keys[kPieces];
    uint32_t values[kWords], single = 0;
#pragma unroll
    for (int x = 0; x < kPieces; ++x) {
      const int p = x * kThreads + tid, j = p / pieces;
      if (j < n) {
        const int64_t from = cell(kept[j0 + j]);
        if (from >= 0) keys[x] = reinterpret_cast<const uint4*>(a.c.k_codes + from * bytes)[p - j * pieces];
      }
    }
    // a word holds four tokens' bytes: of places behind `keep`, what they hold
#pragma unroll
    for (int x = 0; x < kWords; ++x) {
      const int p = x * kThreads + tid, j4 = p / bytes * 4, b = p - j4 / 4 * bytes;
      uint32_t w = 0;
      if (j4 < n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int64_t from = cell(j4 + e < n ? kept[j0 + j4 + e] : j0 + j4 + e);
          if (from < 0) continue;
          w |= (uint32_t)a.c.v_codes[(from & ~3ll) * bytes + b * 4 + (from & 3)] << (8 * e);
        }
      }
      values[x] = w;
    }
    const int which = tid / kChunk, js = tid - which * kChunk;   // keys' parameters, values', weights
    if (which < 3 && js < n) {
      const int64_t from = cell(kept[j0 + js]);
      if (from >= 0)
        single = which == 0   ? reinterpret_cast<const uint32_t*>(a.c.k_params)[from]
                 : which == 1 ? reinterpret_cast<const uint32_t*>(a.c.v_params)[from]
                              : __float_as_uint(a.weights[from]);
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < kPieces; ++x) {
      const int p = x * kThreads + tid, j = p / pieces;
      if (j < n) {
        const int64_t to = cell(j0 + j);
        if (to >= 0 && cell(kept[j0 + j]) >= 0) reinterpret_cast<uint4*>(a.c.k_codes + to * bytes)[p - j * pieces] = keys[x];
      }
    }
#pragma unroll
    for (int x = 0; x < kWords; ++x) {
      const int p = x * kThreads + tid, j4 = p / bytes * 4, b = p - j4 / 4 * bytes;
      if (j4 < n) {
        const int64_t to = cell(j0 + j4);
        if (to >= 0) *reinterpret_cast<uint32_t*>(a.c.v_codes + to * bytes + b * 4) = values[x];
      }
    }
    if (which < 3 && js < n) {
      const int64_t to = cell(j0 + js);
      if (to >= 0) {
        if (which == 0) reinterpret_cast<uint32_t*>(a.c.k_params)[to] = single;
        if (which == 1) reinterpret_cast<uint32_t*>(a.c.v_params)[to] = single;
        if (which == 2) a.weights[to] = __uint_as_float(single);
      }
    }
    __syncthreads();
  }
  // whoever stands in the places behind starts from zero
  for (int j = a.keep + tid; j < (((int64_t)length + mask) & ~(int64_t)mask); j += kThreads) {
    const int64_t to = cell(j);
    if (to >= 0) a.weights[to] = 0.0f;
  }
}

}  // namespace

int launch_kv4_evict(const Kv4EvictArgs& a, cudaStream_t s) {
  if (a.requests > 65535) return set_error(SA_ERR_UNSUPPORTED, "kv4 evict: more than 65535 requests in one call");
  evict_kernel<<<dim3((unsigned)a.c.heads, (unsigned)a.requests), kThreads, 0, s>>>(a);
  return check_launch("kv4 evict_kernel");
}

}  // namespace sa
