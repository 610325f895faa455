// Which pages of a long request a query reads: bounds of each page's keys, a score of
// every page from them, and the pages of the largest scores.
//
// Bounds of a page (of one key head): the least and the largest value of each column
// over the tokens it holds, in bfloat16, [pages, heads, 2, dp] (columns behind d: 0).
//
// Score of page w for the group of query heads that reads key head h:
//   score_w = sum over heads, columns of max(q_c low_c, q_c high_c)
//           = sum_c up_c high_c + down_c low_c,  up = sum of the heads' max(q, 0), down of min(q, 0),
// no less than the sum of the heads' scores of any token of the page (but for the
// bounds' rounding), at the price of one product of 2 d terms for the whole group.
// The second line is the first where bounds are finite; beside an infinite one it has 0 times
// infinity for a side that no head uses.  What is not finite is computed by the first line.
// The sums are float64: products of 16-bit queries with bounds are exact and their sums nearly so, and which pages are
// chosen hardly depends on the order of adding (scores have to agree to some 2^-50; float32 queries' products are rounded there).
//
// 48 requests of 12000..24000 tokens, 8 key heads of 128, pages of 64, 32 chosen: 25 us
// (52 MB of bounds, 8 us): latency, of six rounds of loads and five of digits; one page a
// warp at a time took 51, with every load waited for.
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>

#include "kv4.cuh"

namespace sa {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// Minimum and maximum that keep NaN.
__device__ __forceinline__ float least_of(float x, float y) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float most_of(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}

// A CTA per (touched page, head) at a time: a lane holds eight columns (a word of codes) of
// every (32 / words of a row)-th token of its warp's, kBatch loads on their way at a time;
// the warps join through shared memory.  (48 requests' newest pages of 64 tokens x 8 heads, 3.4 MB: 10 us,
// latency; as one warp a page, with four loads, 25: the chain of a lane's tokens.)
constexpr int kBoundWarps = 4;
constexpr int kBatch = 8;

__global__ void __launch_bounds__(kBoundWarps * 32) bounds_kernel(const Kv4BoundsArgs a) {
  __shared__ float joined[kBoundWarps][2][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = blockIdx.y;
  const int cap = a.width << a.c.page_shift;
  const int whole = max(a.lengths[r], 0), length = min(whole, cap);
  if (whole > cap && blockIdx.x == 0 && threadIdx.x == 0) report(a.status, kBadLength, r);
  const int from = whole - min(max(a.fresh[r], 0), whole);   // tokens [from, length) are new
  if (from >= length) return;
  const int first = from >> a.c.page_shift, last = (length - 1) >> a.c.page_shift;
  const int words = a.c.dp >> 3, word = lane & (words - 1), sub = lane / words, step = kBoundWarps * (32 / words);
  const int64_t units = (int64_t)(last - first + 1) * a.c.heads;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int row = first + (int)(u / a.c.heads), h = (int)(u % a.c.heads);
    const int page = a.tables[(int64_t)r * a.width + row];
    if (page < 0 || page >= a.c.pages) {
      if (h == 0 && threadIdx.x == 0) report(a.status, kBadPage, page);
      continue;
    }
    const int held = min(length - (row << a.c.page_shift), 1 << a.c.page_shift);
    const int64_t cell = (page * (int64_t)a.c.heads + h) << a.c.page_shift;
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(a.c.k_codes + cell * (a.c.dp >> 1)) + word;
    const uint32_t* params = reinterpret_cast<const uint32_t*>(a.c.k_params + 2 * cell);
    float low[8], high[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) low[e] = INFINITY, high[e] = -INFINITY;
    const int t0 = warp * (32 / words) + sub;
    for (int b = 0; b < held; b += kBatch * step) {
      uint32_t w[kBatch], p[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int t = min(b + t0 + i * step, held - 1);   // the last token again changes nothing
        w[i] = codes[(int64_t)t * words];
        p[i] = params[t];
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const float scale = __uint_as_float(p[i] << 16), least = __uint_as_float(p[i] & 0xffff0000u);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = fmaf((float)((w[i] >> (4 * e)) & 15u), scale, least);
          low[e] = least_of(low[e], x);
          high[e] = most_of(high[e], x);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      for (int d = words; d < 32; d *= 2) {
        low[e] = least_of(low[e], __shfl_xor_sync(0xffffffffu, low[e], d));
        high[e] = most_of(high[e], __shfl_xor_sync(0xffffffffu, high[e], d));
      }
    if (sub == 0)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        joined[warp][0][word * 8 + e] = low[e];
        joined[warp][1][word * 8 + e] = high[e];
      }
    __syncthreads();
    __nv_bfloat16* to = a.bounds + (page * (int64_t)a.c.heads + h) * 2 * a.c.dp;
    for (int c = threadIdx.x; c < a.c.dp; c += kBoundWarps * 32) {
      float x = joined[0][0][c], y = joined[0][1][c];
#pragma unroll
      for (int w = 1; w < kBoundWarps; ++w) {
        x = least_of(x, joined[w][0][c]);
        y = most_of(y, joined[w][1][c]);
      }
      to[c] = __float2bfloat16_rn(c < a.c.d ? x : 0.0f);
      to[a.c.dp + c] = __float2bfloat16_rn(c < a.c.d ? y : 0.0f);
    }
    __syncthreads();
  }
}

// A score as a whole number of the same order; NaN is the largest.
__device__ __forceinline__ uint64_t order_of(double x) {
  if (x != x) return ~0ull;
  const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);   // -0 becomes 0
  return b >> 63 ? ~b : b | (1ull << 63);
}

// A lane's columns of a row of bounds.
template <int N>
struct Columns {
  static constexpr int kWords = N > 1 ? N / 2 : 1;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {
    if constexpr (N == 8) {
      const uint4 x = *reinterpret_cast<const uint4*>(p);
      w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else if constexpr (N == 4) {
      const uint2 x = *reinterpret_cast<const uint2*>(p);
      w[0] = x.x, w[1] = x.y;
    } else if constexpr (N == 2) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ float get(int e) const {
    return __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
  }
};

// A lane's columns of a page's score by the definition, head by head: where the short form is not finite (rare).
template <typename T, int N>
__device__ __forceinline__ double score_by_heads(const T* q, int64_t q_h, int group, int columns, const Columns<N>& low,
                                                 const Columns<N>& high) {
  double sum = 0.0;
#pragma unroll
  for (int e = 0; e < N; ++e)
#pragma unroll 1
    for (int h = 0; e < columns && h < group; ++h) {
      const double x = to_f32(q[h * q_h + e]), at_low = x * (double)low.get(e), at_high = x * (double)high.get(e);
      sum += at_low != at_low ? at_low : (at_low > at_high ? at_low : at_high);   // (a NaN of either side stays)
    }
  return sum;
}

// Whether a number is no finite one.
__device__ __forceinline__ bool endless(double x) { return (__double2hiint(x) & 0x7ff00000) == 0x7ff00000; }

constexpr int kPages = 8;   // that a warp scores at a time

// A cluster of CTAs scores the pages of one (query token, key head); its first CTA
// then picks the largest scores by their digits and writes them in ascending order.
template <int DT, int DP>
__global__ void __launch_bounds__(kThreads, 3) select_kernel(const Kv4SelectArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int kCols = DP / 32;   // columns of a lane
  extern __shared__ __align__(16) uint64_t keys[];   // [width]: of the pages between first and last
  __shared__ double up[DP], down[DP];
  __shared__ int count_of[256];
  __shared__ int part[2][kWarps];
  __shared__ int digit, below;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int hk = blockIdx.y, r = blockIdx.z / a.n, i = blockIdx.z % a.n;
  const int group = a.heads / a.c.heads;
  const int cap = a.width << a.c.page_shift;
  const int whole = max(a.lengths[r], 0);
  if (whole > cap && tid == 0) report(a.status, kBadLength, r);
  const int length = min(whole, cap) - (a.n - 1 - i);   // up to this query
  const int pages = length > 0 ? (length + (1 << a.c.page_shift) - 1) >> a.c.page_shift : 0;
  int32_t* out = a.out + ((int64_t)blockIdx.z * a.c.heads + hk) * a.count;
  if (pages <= a.count) {   // all of them
    if (blockIdx.x == 0)
      for (int e = tid; e < a.count; e += kThreads) out[e] = e < pages ? e : -1;
    return;
  }
  const int middle = pages - a.first - a.last, want = a.count - a.first - a.last;
  cg::cluster_group cluster = cg::this_cluster();
  if (want > 0) {
    for (int c = tid; c < DP; c += kThreads) {
      double x = 0.0, y = 0.0;
      if (c < a.c.d)
        for (int e = 0; e < group; ++e) {
          const double q = to_f32(static_cast<const T*>(a.q)[r * a.q_r + i * a.q_n + (int64_t)(hk * group + e) * a.q_h + c]);
          x += q > 0.0 || q != q ? q : 0.0;
          y += q < 0.0 ? q : 0.0;
        }
      up[c] = x;
      down[c] = y;
    }
    if (gridDim.x > 1)
      cluster.sync();   // the first CTA has begun: its shared memory may be written
    else
      __syncthreads();
    double u[kCols], d[kCols];
#pragma unroll
    for (int e = 0; e < kCols; ++e) {
      u[e] = up[lane * kCols + e];
      d[e] = down[lane * kCols + e];
    }
    uint64_t* to = gridDim.x > 1 ? cluster.map_shared_rank(keys, 0) : keys;
    const int32_t* table = a.tables + (int64_t)r * a.width + a.first;
    // eight pages of a warp at a time, all their loads on their way
    const int step = gridDim.x * kWarps * kPages;
    int page = 0;
    Columns<kCols> low[kPages], high[kPages];
    auto fetch = [&](int w0) {
      const int mine = w0 + (lane & (kPages - 1));
      page = mine < middle ? __ldg(table + mine) : 0;
      const bool bad = page < 0 || page >= a.c.pages;
      if (bad && lane < kPages) report(a.status, kBadPage, page);
      if (bad) page = -1;
    };
    bool odd = false;   // a share of a score that is not finite
    const int begin = (blockIdx.x * kWarps + warp) * kPages;
    if (begin < middle) fetch(begin);
    for (int w0 = begin; w0 < middle; w0 += step) {
#pragma unroll
      for (int x = 0; x < kPages; ++x) {
        const int id = max(__shfl_sync(0xffffffffu, page, x), 0);
        const __nv_bfloat16* b = a.bounds + (id * (int64_t)a.c.heads + hk) * 2 * DP + lane * kCols;
        low[x].load(b);
        high[x].load(b + DP);
      }
      const int here = page;
      if (w0 + step < middle) fetch(w0 + step);
      double score[kPages];
#pragma unroll
      for (int x = 0; x < kPages; ++x) {
        score[x] = 0.0;
#pragma unroll
        for (int e = 0; e < kCols; ++e) {
          score[x] = fma(u[e], (double)high[x].get(e), score[x]);
          score[x] = fma(d[e], (double)low[x].get(e), score[x]);
        }
        odd |= endless(score[x]);
      }
      // sums over the lanes: each halving keeps half of the pages, so that in the end four lanes have one page's
#pragma unroll
      for (int n = kPages / 2, x = 16; n >= 1; n /= 2, x /= 2) {
        const bool upper = lane & x;
#pragma unroll
        for (int i = 0; i < n; ++i) {
          const double give = upper ? score[i] : score[i + n], keep = upper ? score[i + n] : score[i];
          score[i] = keep + __shfl_xor_sync(0xffffffffu, give, x);
        }
      }
      score[0] += __shfl_xor_sync(0xffffffffu, score[0], 2);
      score[0] += __shfl_xor_sync(0xffffffffu, score[0], 1);
      const int x = lane >> 2;   // bit 4 chose among pages 0..3 and 4..7, and so on
      const bool none = __shfl_sync(0xffffffffu, here, x) < 0;
      if ((lane & 3) == 0 && w0 + x < middle) to[w0 + x] = order_of(none ? -INFINITY : score[0]);
    }
    if (__any_sync(0xffffffffu, odd)) {   // again, a page at a time, those scores alone
      const T* q = static_cast<const T*>(a.q) + r * a.q_r + i * a.q_n + (int64_t)hk * group * a.q_h + lane * kCols;
      for (int w = begin; w < middle; w = (w & (kPages - 1)) == kPages - 1 ? w + 1 - kPages + step : w + 1) {
        const int id = __ldg(table + w);
        if (id < 0 || id >= a.c.pages) continue;
        const __nv_bfloat16* b = a.bounds + (id * (int64_t)a.c.heads + hk) * 2 * DP + lane * kCols;
        Columns<kCols> l, h;
        l.load(b);
        h.load(b + DP);
        double score = 0.0;
#pragma unroll
        for (int e = 0; e < kCols; ++e) {
          score = fma(u[e], (double)h.get(e), score);
          score = fma(d[e], (double)l.get(e), score);
        }
        odd = endless(score);
        if (!__any_sync(0xffffffffu, odd)) continue;
        if (odd) score = score_by_heads<T>(q, a.q_h, group, a.c.d - lane * kCols, l, h);
#pragma unroll
        for (int x = 16; x >= 1; x /= 2) score += __shfl_xor_sync(0xffffffffu, score, x);
        if (lane == 4 * (w & (kPages - 1))) to[w] = order_of(score);   // the lane that wrote it above
      }
    }
  }
  if (gridDim.x > 1)
    cluster.sync();
  else
    __syncthreads();
  if (blockIdx.x != 0) return;
  // the want-th largest key, digit by digit: `border`, of whose equals `ties` are taken
  uint64_t border = 0, mask = 0;
  int ties = want;
  for (int shift = 56; shift >= 0 && want > 0; shift -= 8) {
    count_of[tid] = 0;
    __syncthreads();
    for (int w = tid; w < middle; w += kThreads)
      if ((keys[w] & mask) == border) atomicAdd(&count_of[(keys[w] >> shift) & 255], 1);
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
    border |= (uint64_t)digit << shift;
    mask |= 255ull << shift;
    ties -= below;
    const bool all = count_of[digit] == ties;   // the whole digit is taken
    __syncthreads();
    if (all) break;
  }
  // ascending: the first pages, those picked between, the last
  for (int e = tid; e < a.first; e += kThreads) out[e] = e;
  for (int e = tid; e < a.last; e += kThreads) out[a.first + want + e] = pages - a.last + e;
  int at = a.first, equal = 0;
  for (int w0 = 0; w0 < middle && want > 0; w0 += kThreads) {
    const int w = w0 + tid;
    const uint64_t k = w < middle ? keys[w] & mask : 0;
    const bool over = w < middle && k > border, same = w < middle && k == border;
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
    if (over || (same && s < ties)) out[at + o + min(s, ties) - min(equal, ties)] = a.first + w;
    at += o_all + min(equal + s_all, ties) - min(equal, ties);
    equal += s_all;
    __syncthreads();
  }
}

template <int DT, int DP>
int launch_select(const Kv4SelectArgs& a, cudaStream_t s) {
  auto kern = select_kernel<DT, DP>;
  const int64_t z = (int64_t)a.requests * a.n;
  if (z > 65535 || a.c.heads > 65535) return set_error(SA_ERR_UNSUPPORTED, "kv4 select: grid too large");
  const size_t smem = (size_t)a.width * 8;
  static std::atomic<uint64_t> allowed{0};
  const int rc = allow_shared(kern, kSelectMaxPages * 8, allowed, "kv4 select");
  if (rc) return rc;
  int splits = 1;   // while a warp keeps eight pages and CTAs are few
  while (splits < 8 && a.width >= splits * 2 * kWarps * kPages && z * a.c.heads * splits < 148) splits *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)splits, (unsigned)a.c.heads, (unsigned)z);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  // An ordinary launch, behind all of the stream: what a caller put there before may write q, lengths or tables, or
  // still read the memory that `selected` lies in, and whether that kernel lets others start early is not known here.
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
  if (e != cudaSuccess) return set_error(SA_ERR_CUDA, "kv4 select_kernel: %s", cudaGetErrorString(e));
  return check_launch("kv4 select_kernel");
}

template <int DT>
int launch_select_dim(const Kv4SelectArgs& a, cudaStream_t s) {
  if (a.c.dp == 32) return launch_select<DT, 32>(a, s);
  if (a.c.dp == 64) return launch_select<DT, 64>(a, s);
  if (a.c.dp == 128) return launch_select<DT, 128>(a, s);
  return launch_select<DT, 256>(a, s);
}

}  // namespace

int launch_kv4_bounds(const Kv4BoundsArgs& a, cudaStream_t s) {
  // CTAs that share a request's pages: enough for the GPU when requests are few, and one for
  // each head of a page
  const int64_t most = (int64_t)a.width * a.c.heads;
  const int64_t x = std::min(most, std::max<int64_t>(ceil_div(148 * 8, a.requests), a.c.heads));
  if (a.requests > 65535) return set_error(SA_ERR_UNSUPPORTED, "kv4 bounds: more than 65535 requests in one call");
  bounds_kernel<<<dim3((unsigned)x, (unsigned)a.requests), kBoundWarps * 32, 0, s>>>(a);
  return check_launch("kv4 bounds_kernel");
}

int launch_kv4_select(const Kv4SelectArgs& a, int dtype, cudaStream_t s) {
  if (dtype == SA_REP_FLOAT32) return launch_select_dim<SA_REP_FLOAT32>(a, s);
  if (dtype == SA_REP_FLOAT16) return launch_select_dim<SA_REP_FLOAT16>(a, s);
  return launch_select_dim<SA_REP_BFLOAT16>(a, s);
}

}  // namespace sa
