// Shared by the serving kernels (windowed attention, the 4-bit cache, page
// plans, norm + rotation): element types, the visible key ranges of a sliding
// window with first tokens, and the error word.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "sa_common.cuh"

namespace sa {

// Codes of the error word that name bad contents of device-side index arrays
// (the kernels skip what they point at); sa_serving_status reports them as
// SA_ERR_INVALID_ARG.
constexpr int kBadPage = 400;     // a page id outside the cache
constexpr int kBadSlot = 401;     // a slot outside the cache
constexpr int kBadLength = 402;   // a request longer than its row of the page table
constexpr int kBadOffsets = 403;  // offsets that are not monotone or leave the tensors
constexpr int kNoPages = 404;     // the list of free pages ran out
constexpr int kNoRows = 405;      // more new tokens than the outputs hold
constexpr int kHeld = 406;        // a prompt for a request that holds tokens

__device__ __forceinline__ void report(int* status, int code, long long index) {
  if (status && atomicCAS(status, 0, code) == 0) *reinterpret_cast<volatile long long*>(status + 2) = index;
}

// Element types (the SA_REP_* codes).
template <int DT>
struct Elem;
template <>
struct Elem<SA_REP_FLOAT32> {
  using T = float;
};
template <>
struct Elem<SA_REP_FLOAT16> {
  using T = __half;
};
template <>
struct Elem<SA_REP_BFLOAT16> {
  using T = __nv_bfloat16;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ uint16_t from_f32<uint16_t>(float) {   // bits of 0 alone
  return 0;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) {
  return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// Eight elements of a row, 16-byte aligned (32 bytes of float32).
template <typename T>
__device__ __forceinline__ void load8(float (&x)[8], const T* p) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *(reinterpret_cast<const float4*>(p) + 1);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    union {
      uint4 w;
      T e[8];
    } u;
    u.w = *reinterpret_cast<const uint4*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(u.e[i]);
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *(reinterpret_cast<float4*>(p) + 1) = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    union {
      uint4 w;
      T e[8];
    } u;
#pragma unroll
    for (int i = 0; i < 8; ++i) u.e[i] = from_f32<T>(x[i]);
    *reinterpret_cast<uint4*>(p) = u.w;
  }
}
// Whether every row of a tensor with these strides starts on a 16-byte border.
__host__ inline bool rows_aligned(const void* p, int elem, int64_t s0, int64_t s1) {
  return (((uintptr_t)p | (uintptr_t)(s0 * elem) | (uintptr_t)(s1 * elem)) & 15) == 0;
}

__host__ inline int elem_size(int dtype) { return dtype == SA_REP_FLOAT32 ? 4 : 2; }

// What the window kernels take.  Strides are in elements.  Dense: request b's
// rows start at b * *_b.  Packed (cu_q != nullptr): *_b is 0, n and m are the
// tensors' row counts and request b's rows are cu_q[b] .. cu_q[b + 1].
struct WindowArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  int64_t q_b, q_h, q_n, k_b, k_h, k_n, v_b, v_h, v_n, o_b, o_h, o_n;
  int batch, heads, kv_heads;
  int64_t n, m;
  int d, dv;
  int64_t window;   // keys p - window + 1 .. p of the query at position p
  int64_t sinks;    // and keys 0 .. sinks - 1
  float scale;
  int dtype;
  const int32_t* cu_q;
  const int32_t* cu_k;
  int* status;
  int zero_behind;   // packed: write zeros to the rows that no request writes
};

// Packed: whether request b's offsets are out of order or out of range.  Such a
// request counts as empty.
__device__ __forceinline__ bool offsets_refused(const WindowArgs& a, int64_t b) {
  const int64_t q0 = a.cu_q[b], q1 = a.cu_q[b + 1], k0 = a.cu_k[b], k1 = a.cu_k[b + 1];
  return q0 < 0 || q1 < q0 || q1 > a.n || k0 < 0 || k1 < k0 || k1 > a.m;
}

// One request of a (dense or packed) batch: first rows and row counts.
struct Request {
  int64_t q0, k0, n, m;
};

__device__ __forceinline__ Request request_of(const WindowArgs& a, int b) {
  if (!a.cu_q) return Request{0, 0, a.n, a.m};
  if (offsets_refused(a, b)) return Request{0, 0, 0, 0};
  const int64_t q0 = a.cu_q[b], k0 = a.cu_k[b];
  return Request{q0, k0, a.cu_q[b + 1] - q0, a.cu_k[b + 1] - k0};
}

// Tile t of a batch of query tiles of `rows` rows.  Dense: t = b * tiles + i.
// Packed: request b owns tiles cu_q[b] / rows + b onwards -- a start that is
// strictly monotone in b and leaves room for its ceil(n_b / rows) tiles, so a
// binary search over cu_q finds the request and the grid needs no request's
// length: n / rows + batch tiles in all.
__device__ __forceinline__ int tile_request(const WindowArgs& a, int64_t t, int rows, int64_t* tile) {
  if (!a.cu_q) {
    const uint32_t per = (uint32_t)((a.n + rows - 1) / rows), u = (uint32_t)t;   // the grid has less than 2^31 tiles
    *tile = u % per;
    return (int)(u / per);
  }
  int lo = 0, hi = a.batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((int64_t)max(a.cu_q[mid], 0) / rows + mid <= t)
      lo = mid;
    else
      hi = mid - 1;
  }
  *tile = t - ((int64_t)max(a.cu_q[lo], 0) / rows + lo);
  return lo;
}
__host__ inline int64_t tile_count(const WindowArgs& a, int rows) {
  return a.cu_q ? a.n / rows + a.batch : ceil_div(a.n, rows) * a.batch;
}

// Packed: reports the requests whose offsets are refused and writes zeros to the
// rows of out that no request writes, `tile_rows` rows to a query tile:
// - those before the first offset and behind the largest, dealt out to the grid's
//   threads (whole warps, `threads` of each CTA, this one the `thread`-th);
// - those between a refused request's offsets, by the CTA that finds it;
// - where an offset steps back, the tiles that tile_request then gives to another
//   request, likewise.
// Offsets go from the first to the last of them in steps, and a step back passes
// rows that one forward has passed before: so that is every row.  (Rows that two
// steps forward pass hold one's result or the other's, or zeros.)  `beat` as in
// repair_row.
template <typename T>
__device__ __forceinline__ void zero_unwritten_rows(const WindowArgs& a, int tile_rows, int64_t thread, int64_t threads,
                                                    int* beat) {
  if (!a.cu_q) return;
  const int64_t cta = blockIdx.x + (int64_t)blockIdx.y * gridDim.x, ctas = (int64_t)gridDim.x * gridDim.y;
  const int64_t width = (int64_t)a.heads * a.dv;
  const int lane = threadIdx.x & 31;
  auto zero = [&](int64_t first, int64_t e) {   // element e of the rows from `first` on
    const int64_t r = e / width, rest = e - r * width, h = rest / a.dv;
    static_cast<T*>(a.out)[h * a.o_h + (first + r) * a.o_n + rest - h * a.dv] = from_f32<T>(0.0f);
  };
  auto zero_rows = [&](int64_t x, int64_t y) {   // by this CTA
    int turn = 0;
    for (int64_t e = thread; e < (y - x) * width; e += threads) {
      zero(x, e);
      if (beat && (++turn & 1023) == 0) atomicAdd(beat, 1);
    }
  };
  bool back = false;
  for (int64_t b0 = cta; b0 < a.batch; b0 += 32 * ctas) {
    const int64_t b = b0 + lane * ctas;
    const bool bad = b < a.batch && offsets_refused(a, b);
    if (bad) report(a.status, kBadOffsets, b);
#pragma unroll 1
    for (unsigned left = __ballot_sync(0xffffffffu, bad); a.zero_behind && left; left &= left - 1) {
      const int64_t at = b0 + (__ffs(left) - 1) * ctas;
      const int64_t x = a.cu_q[at], y = a.cu_q[at + 1];
      back |= y < x;
      zero_rows(max(x, (int64_t)0), min(y, a.n));
    }
  }
  if (!a.zero_behind) return;
#pragma unroll 1
  for (int b = 0; back && b < a.batch; ++b) {
    const Request r = request_of(a, b);
    const int64_t first = r.q0 / tile_rows + b, tiles = (r.n + tile_rows - 1) / tile_rows;
    if (beat) atomicAdd(beat, 1);
#pragma unroll 1
    for (int64_t i0 = 0; i0 < tiles; i0 += 32) {
      int64_t tile;
      const bool lost = i0 + lane < tiles && tile_request(a, first + i0 + lane, tile_rows, &tile) != b;
#pragma unroll 1
      for (unsigned left = __ballot_sync(0xffffffffu, lost); left; left &= left - 1) {
        const int64_t x = (i0 + __ffs(left) - 1) * tile_rows;
        zero_rows(r.q0 + x, r.q0 + min(x + tile_rows, r.n));
      }
    }
  }
  const int64_t lead = min(max((int64_t)a.cu_q[0], (int64_t)0), a.n);
  int64_t behind = min(max((int64_t)a.cu_q[a.batch], lead), a.n);
  if (behind < a.n) {   // behind the largest of them, should that not be the last
    int top = 0;
    for (int b = lane; b <= a.batch; b += 32) top = max(top, a.cu_q[b]);
    behind = min(max(behind, (int64_t)__reduce_max_sync(0xffffffffu, top)), a.n);
  }
  for (int64_t e = cta * threads + thread; e < (lead + a.n - behind) * width; e += ctas * threads)
    zero(e < lead * width ? 0 : behind - lead, e);
}

// The keys that any of the queries at positions p0 .. p1 sees, as two ranges:
// first tokens [0, first) and window [begin, end); first <= begin.
struct KeyRanges {
  int64_t first, begin, end;
};
__host__ __device__ inline KeyRanges key_ranges(int64_t p0, int64_t p1, int64_t m, int64_t window, int64_t sinks) {
  KeyRanges r;
  r.end = p1 + 1 < m ? p1 + 1 : m;
  if (r.end < 0) r.end = 0;
  r.begin = p0 - window + 1 > 0 ? p0 - window + 1 : 0;
  if (r.begin > r.end) r.begin = r.end;
  r.first = sinks < r.begin ? sinks : r.begin;
  return r;
}

int launch_window_simt(const WindowArgs& a, cudaStream_t s);
bool window_tc_takes(const WindowArgs& a);
size_t window_tc_bytes(const WindowArgs& a);
int launch_window_tc(const WindowArgs& a, void* workspace, size_t workspace_bytes, cudaStream_t s);
size_t window_tf32_bytes(int64_t batch, int heads, int kv_heads, int64_t n, int64_t m, int d, int dv, int64_t window,
                         int64_t sinks);
int window_tf32_run(const WindowArgs& a, void* workspace, size_t workspace_bytes, cudaStream_t s);

}  // namespace sa
