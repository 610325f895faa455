// Page tables, slots and positions from request lengths, and the return of a
// request's pages.
//
//   after[r]   = lengths[r] + new[r],   offsets = exclusive sum of new
//   fresh(r)   = ceil(after[r] / P) - ceil(lengths[r] / P)  pages, in request order, from the end of the free list
//   packed token t of request r: position = lengths[r] + t - offsets[r],
//                         slot = tables[r][position / P] * P + position % P
//
// One launch.  Every CTA sums all requests' (new, fresh) pairs into shared
// memory (a request costs 8 bytes there; the redundant sum costs less than a
// second launch), then handles a run of new tokens: it finds a token's request
// by binary search over the sums, and the token that opens a page writes the
// page's entry of the table.  The first CTA writes what there is one of per
// request.  24 requests' next tokens: 6.2 us; 1000 prompts of up to 400 tokens: 9.4 us,
// both latency (a round of sums, a search, the table's and the list's loads).
#include "serving.cuh"

namespace sa {

namespace {

constexpr int kPlanThreads = 1024;              // a batch of 1000 requests is summed in one round (256 threads: 13 us)
constexpr int kPlanTokens = 2 * kPlanThreads;   // per CTA
constexpr int kPlanMaxRequests = 16384;

struct PlanArgs {
  const int32_t* lengths;
  const int32_t* fresh;   // new tokens per request
  int32_t* tables;
  const int32_t* free_pages;
  const int32_t* free_count;
  int32_t* lengths_out;
  int32_t* offsets;
  int32_t* positions;
  int32_t* slots;
  int32_t* free_out;
  int* status;
  int requests, width, free_size, max_tokens, page_shift;
  int per_request;   // > 0: token i of request r stands at r * per_request + i, not packed
  int prompts;       // new tokens of requests that hold some are reported
};

__device__ __forceinline__ int64_t pages_of(int64_t tokens, int shift, int width) {
  return min((tokens + (1 << shift) - 1) >> shift, (int64_t)width);
}

// The page that entry `row` of a request's table takes, the first of the new ones
// being `had`: nth from the end of the `have` free ones, `before` taken by the
// requests before; -1 where there is none.
__device__ __forceinline__ int32_t fresh_page(const PlanArgs& a, int have, int before, int64_t row, int64_t had) {
  const int64_t at = (int64_t)have - 1 - before - (row - had);
  if (at < 0) return -1;
  const int32_t page = a.free_pages[at];
  if (page >= 0 && page < a.free_size) return page;
  report(a.status, kBadPage, page);
  return -1;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  int32_t* sum_new = plan_smem;                       // [requests + 1], exclusive
  int32_t* sum_pages = plan_smem + a.requests + 1;    // [requests + 1]
  __shared__ long long part_new[kPlanThreads / 32];
  __shared__ int part_pages[kPlanThreads / 32];
  __shared__ long long carry_new;
  __shared__ int carry_pages;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool first = blockIdx.x == 0;
  if (tid == 0) {
    carry_new = 0;
    carry_pages = 0;
  }
  __syncthreads();
  for (int r0 = 0; r0 < a.requests; r0 += kPlanThreads) {
    const int r = r0 + tid;
    int64_t len = 0, add = 0;
    if (r < a.requests) {
      len = max(a.lengths[r], 0);
      add = max(a.fresh[r], 0);
      if (first) {
        if (len + add > ((int64_t)a.width << a.page_shift)) report(a.status, kBadLength, r);
        if (a.per_request > 0 && add > a.per_request) report(a.status, kNoRows, add);
        if (a.prompts && len > 0 && add > 0) report(a.status, kHeld, r);
        a.lengths_out[r] = (int32_t)min(len + add, (int64_t)2147483647);
      }
    }
    const int pages = (int)(pages_of(len + add, a.page_shift, a.width) - pages_of(len, a.page_shift, a.width));
    long long x = add;
    int y = pages;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long xo = __shfl_up_sync(0xffffffffu, x, o);
      const int yo = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) {
        x += xo;
        y += yo;
      }
    }
    if (lane == 31) {
      part_new[warp] = x;
      part_pages[warp] = y;
    }
    __syncthreads();
    // the warps before: each lane takes one, summed by shuffles
    long long xb = lane < warp ? part_new[lane] : 0;
    int yb = lane < warp ? part_pages[lane] : 0;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
      xb += __shfl_xor_sync(0xffffffffu, xb, o);
      yb += __shfl_xor_sync(0xffffffffu, yb, o);
    }
    x += carry_new + xb;
    y += carry_pages + yb;
    if (r < a.requests) {
      sum_new[r] = (int32_t)min(x - (long long)add, 2147483647LL);
      sum_pages[r] = y - pages;
    }
    __syncthreads();
    if (tid == kPlanThreads - 1) {
      carry_new = x;
      carry_pages = y;
    }
    __syncthreads();
  }
  const int total = (int)min(carry_new, 2147483647LL);
  if (tid == 0) {
    sum_new[a.requests] = total;
    sum_pages[a.requests] = carry_pages;
  }
  __syncthreads();
  // the list holds free_count entries, of which the last is taken first
  const int have = min(max(a.free_count[0], 0), a.free_size);
  if (first) {
    for (int r = tid; r <= a.requests; r += kPlanThreads) a.offsets[r] = sum_new[r];
    if (tid == 0) {
      const int taken = sum_pages[a.requests];
      a.free_out[0] = max(have - taken, 0);
      if (taken > have) report(a.status, kNoPages, taken);
      if (a.per_request == 0 && total > a.max_tokens) report(a.status, kNoRows, total);
    }
  }
  const int mask = (1 << a.page_shift) - 1;
  for (int j = 0; j < kPlanTokens / kPlanThreads; ++j) {
    const int64_t t = (int64_t)blockIdx.x * kPlanTokens + j * kPlanThreads + tid;
    if (t >= a.max_tokens) break;
    int32_t position = -1, slot = -1;
    int lo = 0;
    int64_t nth = t;   // which of its request's new tokens
    if (a.per_request > 0) {
      lo = (int)(t / a.per_request);
      nth = t - (int64_t)lo * a.per_request;
    } else if (t < total) {
      int hi = a.requests - 1;   // the last request whose offset is <= t
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (sum_new[mid] <= t)
          lo = mid;
        else
          hi = mid - 1;
      }
      nth = t - sum_new[lo];
    }
    if (lo < a.requests && nth < sum_new[lo + 1] - sum_new[lo]) {
      const int64_t len = max(a.lengths[lo], 0);
      const int64_t pos = len + nth;
      const int64_t row = pos >> a.page_shift;
      position = (int32_t)pos;
      if (row < a.width) {
        const int64_t had = pages_of(len, a.page_shift, a.width);
        int32_t page;
        if (row < had) {
          page = a.tables[(int64_t)lo * a.width + row];
          if (page < -1 || page >= a.free_size) report(a.status, kBadPage, page);   // -1: taken when none was free
        } else {
          page = fresh_page(a, have, sum_pages[lo], row, had);
          if ((pos & mask) == 0) a.tables[(int64_t)lo * a.width + row] = page;
        }
        if (page >= 0 && page < a.free_size) slot = (page << a.page_shift) | (int32_t)(pos & mask);
      }
    }
    a.positions[t] = position;
    a.slots[t] = slot;
  }
  // pages that are opened by tokens without a row: they are taken, so they are entered too
  for (int64_t r = (int64_t)blockIdx.x * kPlanThreads + tid; r < a.requests; r += (int64_t)gridDim.x * kPlanThreads) {
    const int64_t add = a.fresh[r];
    const int64_t rows = a.per_request > 0 ? a.per_request : max((int64_t)a.max_tokens - sum_new[r], (int64_t)0);
    if (add <= rows) continue;
    const int64_t len = max(a.lengths[r], 0), had = pages_of(len, a.page_shift, a.width);
    const int64_t from = (len + rows + mask) >> a.page_shift;   // the first that no token with a row opens
    for (int64_t row = max(had, from); row < pages_of(len + add, a.page_shift, a.width); ++row)
      a.tables[r * a.width + row] = fresh_page(a, have, sum_pages[r], row, had);
  }
}

// Returns the pages of the requests whose `drop` is not 0 to the end of the
// free list, in request order, and empties their rows of the table, whole: entries
// behind the pages a request holds are of nobody's (a plan whose lengths were not
// taken over leaves some) and go nowhere.  One CTA: it runs when a request ends.
__global__ void __launch_bounds__(kPlanThreads)
release_kernel(int32_t* lengths, int32_t* tables, const uint8_t* drop, int32_t* free_pages, int32_t* free_count,
               int requests, int width, int free_size, int page_shift, int* status) {
  __shared__ int part[kPlanThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int64_t at = min(max(free_count[0], 0), free_size);
  __syncthreads();
  for (int r = 0; r < requests; ++r) {
    if (!drop[r]) continue;
    const int64_t held = pages_of(max(lengths[r], 0), page_shift, width);
    for (int64_t c = held + tid; c < width; c += kPlanThreads) tables[(int64_t)r * width + c] = -1;
    for (int64_t c0 = 0; c0 < held; c0 += kPlanThreads) {
      const int64_t c = c0 + tid;
      int32_t page = -1;
      if (c < held) {
        page = tables[(int64_t)r * width + c];
        tables[(int64_t)r * width + c] = -1;
        if (page < -1 || page >= free_size) {
          report(status, kBadPage, page);
          page = -1;
        }
      }
      const unsigned on = __ballot_sync(0xffffffffu, page >= 0);
      if (lane == 0) part[warp] = __popc(on);
      __syncthreads();
      int before = 0, all = 0;
      for (int w = 0; w < kPlanThreads / 32; ++w) {
        if (w < warp) before += part[w];
        all += part[w];
      }
      const int64_t to = at + before + __popc(on & ((1u << lane) - 1));
      if (page >= 0) {
        if (to < free_size)
          free_pages[to] = page;
        else
          report(status, kNoRows, to);
      }
      at = min(at + all, (int64_t)free_size);
      __syncthreads();
    }
    __syncthreads();
    if (tid == 0) lengths[r] = 0;
  }
  if (tid == 0) free_count[0] = (int)at;
}

}  // namespace

int launch_plan_pages(const int32_t* lengths, const int32_t* fresh, int32_t* tables, const int32_t* free_pages,
                      const int32_t* free_count, int requests, int width, int free_size, int page_shift,
                      int max_tokens, int per_request, int prompts, int32_t* lengths_out, int32_t* offsets, int32_t* positions,
                      int32_t* slots, int32_t* free_out, int* status, cudaStream_t s) {
  if (requests > kPlanMaxRequests)
    return set_error(SA_ERR_UNSUPPORTED, "page plan: more than %d requests", kPlanMaxRequests);
  const PlanArgs a{lengths, fresh,     tables, free_pages, free_count, lengths_out, offsets,    positions,
                   slots,   free_out,  status, requests,   width,      free_size,   max_tokens, page_shift,
                   per_request, prompts};
  const size_t smem = (size_t)(requests + 1) * 8;
  if (smem > 48 * 1024) {
    const cudaError_t e =
        cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (kPlanMaxRequests + 1) * 8);
    if (e != cudaSuccess) return set_error(SA_ERR_CUDA, "page plan smem attribute: %s", cudaGetErrorString(e));
  }
  const int64_t ctas = max_tokens > 0 ? ceil_div(max_tokens, kPlanTokens) : 1;
  plan_kernel<<<(unsigned)ctas, kPlanThreads, smem, s>>>(a);
  return check_launch("plan_kernel");
}

int launch_release_pages(int32_t* lengths, int32_t* tables, const uint8_t* drop, int32_t* free_pages,
                         int32_t* free_count, int requests, int width, int free_size, int page_shift, int* status,
                         cudaStream_t s) {
  release_kernel<<<1, kPlanThreads, 0, s>>>(lengths, tables, drop, free_pages, free_count, requests, width, free_size,
                                            page_shift, status);
  return check_launch("release_kernel");
}

}  // namespace sa
