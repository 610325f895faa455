// C ABI of the serving operators (declared in include/streaming_attention.h):
// argument checks, then one launch (two where a join is needed).  Every size is
// checked here; the contents of device-side index arrays (offsets, slots, page
// tables, lengths) are checked in the kernels, which skip what is out of range
// and record it in the error word of sa_serving_status.
#include <stddef.h>
#include <stdlib.h>
#include <string.h>

#include <algorithm>

#include "kv4.cuh"
#include "serving.cuh"

namespace sa {

int launch_plan_pages(const int32_t* lengths, const int32_t* fresh, int32_t* tables, const int32_t* free_pages,
                      const int32_t* free_count, int requests, int width, int free_size, int page_shift,
                      int max_tokens, int per_request, int prompts, int32_t* lengths_out, int32_t* offsets, int32_t* positions,
                      int32_t* slots, int32_t* free_out, int* status, cudaStream_t s);
int launch_release_pages(int32_t* lengths, int32_t* tables, const uint8_t* drop, int32_t* free_pages,
                         int32_t* free_count, int requests, int width, int free_size, int page_shift, int* status,
                         cudaStream_t s);
int prepare_shrink_requests(int requests);
int launch_shrink_requests(int32_t* lengths, int32_t* tables, int32_t* free_pages, int32_t* free_count, int32_t* dropped,
                           int requests, int width, int free_size, int page_shift, int keep, int limit, int* status,
                           cudaStream_t s);
int launch_rotary(const void* q, const void* k, void* q_out, void* k_out, const int32_t* positions,
                  const void* q_weight, const void* k_weight, const double* frequencies, const int64_t* strides,
                  int64_t tokens, int heads, int kv_heads, int d, int half, float eps, int interleaved,
                  int zero_skipped, int dtype, cudaStream_t s);

namespace {

// The error word: one per device, zero at load, set by the first kernel that
// finds something wrong and cleared when it is read.  Its index is stored as 8
// bytes behind it (report), so the type carries the alignment.
struct alignas(16) StatusWord {
  int code[2];
  long long index;
};
static_assert(alignof(StatusWord) % alignof(long long) == 0 && offsetof(StatusWord, index) == 2 * sizeof(int), "report() stores the index as one 8-byte word");
__device__ StatusWord g_serving_status;

// (where it lies is asked once for each device: 1 us)
int* status_word() {
  static std::atomic<int*> words[64];
  int device = -1;
  if (cudaGetDevice(&device) != cudaSuccess) {
    cudaGetLastError();
    return nullptr;
  }
  if (device >= 0 && device < 64)
    if (int* known = words[device].load(std::memory_order_relaxed)) return known;
  void* p = nullptr;
  if (cudaGetSymbolAddress(&p, g_serving_status) != cudaSuccess) {
    cudaGetLastError();
    return nullptr;
  }
  if (device >= 0 && device < 64) words[device].store(static_cast<int*>(p), std::memory_order_relaxed);
  return static_cast<int*>(p);
}

int check_dtype(int dtype) {
  if (dtype != SA_REP_FLOAT32 && dtype != SA_REP_FLOAT16 && dtype != SA_REP_BFLOAT16)
    return set_error(SA_ERR_INVALID_ARG, "dtype must be float32, float16 or bfloat16");
  return SA_OK;
}

int check_heads(int heads, int kv_heads) {
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0)
    return set_error(SA_ERR_INVALID_ARG, "the query heads must be a positive multiple of the key heads");
  return SA_OK;
}

// A window (0: without end) and first tokens, held where sums with positions
// (below 2^31) cannot pass 64 bits.
int64_t window_of(int64_t window) { return window > 0 ? std::min(window, (int64_t)1 << 40) : (int64_t)1 << 40; }
int64_t sinks_of(int64_t sinks) { return std::min(sinks, (int64_t)1 << 40); }

// Whether [b, h, n, width] with these strides is contiguous; an axis of one entry may have any.
bool contiguous(int64_t b, int64_t s_b, int64_t h, int64_t s_h, int64_t n, int64_t s_n, int64_t width) {
  return (n <= 1 || s_n == width) && (h <= 1 || s_h == n * width) && (b <= 1 || s_b == h * n * width);
}

int page_shift_of(int page_size) {
  for (int s = 4; s <= 8; ++s)
    if (page_size == 1 << s) return s;
  return -1;
}

// A head width filled up to 32, 64, 128 or 256.
int padded_dim(int d) {
  int dp = 32;
  while (dp < d) dp *= 2;
  return dp;
}

int check_cache(Kv4Cache* c, const void* k_codes, const void* k_params, const void* v_codes, const void* v_params,
                int64_t pages, int heads, int page_size, int d) {
  if (pages <= 0 || heads <= 0) return set_error(SA_ERR_INVALID_ARG, "the cache needs at least one page and one head");
  if (d <= 0 || d > SA_MAX_DIM) return set_error(SA_ERR_INVALID_ARG, "the cache's head width must lie in [1, %d]", SA_MAX_DIM);
  const int shift = page_shift_of(page_size);
  if (shift < 0) return set_error(SA_ERR_INVALID_ARG, "page_size must be 16, 32, 64, 128 or 256");
  if (pages > (2147483647LL >> shift)) return set_error(SA_ERR_UNSUPPORTED, "the cache holds 2^31 tokens or more");
  if (!k_codes || !k_params || !v_codes || !v_params) return set_error(SA_ERR_INVALID_ARG, "null cache pointer");
  if (((uintptr_t)k_codes | (uintptr_t)k_params | (uintptr_t)v_codes | (uintptr_t)v_params) & 15)
    return set_error(SA_ERR_INVALID_ARG, "the cache's tensors must be 16-byte aligned");
  *c = Kv4Cache{(uint8_t*)k_codes, (__nv_bfloat16*)k_params, (uint8_t*)v_codes, (__nv_bfloat16*)v_params,
                pages, heads, d, padded_dim(d), shift};
  return SA_OK;
}

int check_tables(int requests, int width, int page_shift) {
  if (requests < 0 || width < 0) return set_error(SA_ERR_INVALID_ARG, "sizes must be non-negative");
  if (requests > 65535) return set_error(SA_ERR_UNSUPPORTED, "more than 65535 requests in one call");
  if (((int64_t)width << page_shift) > 2147483647LL)
    return set_error(SA_ERR_UNSUPPORTED, "a row of the page table covers 2^31 tokens or more");
  return SA_OK;
}

// The sizes of an attention over the cache.
int attend_sizes(Kv4AttendArgs* a, int kv_heads, int page_size, int requests, int n, int heads, int width, int64_t window,
                 int64_t sinks) {
  int rc = check_heads(heads, kv_heads);
  if (rc) return rc;
  const int shift = page_shift_of(page_size);
  if (shift < 0) return set_error(SA_ERR_INVALID_ARG, "page_size must be 16, 32, 64, 128 or 256");
  if (requests < 0 || n < 0 || width < 0) return set_error(SA_ERR_INVALID_ARG, "sizes must be non-negative");
  if (window < 0 || sinks < 0) return set_error(SA_ERR_INVALID_ARG, "window and sinks must be non-negative");
  if ((int64_t)n * heads > 65535) return set_error(SA_ERR_UNSUPPORTED, "more than 65535 query rows per request");
  rc = check_tables(requests, width, shift);
  if (rc) return rc;
  a->c.heads = kv_heads;
  a->c.page_shift = shift;
  a->requests = requests;
  a->n = n;
  a->heads = heads;
  a->width = width;
  a->window = window_of(window);
  a->sinks = sinks_of(sinks);
  return SA_OK;
}

int attend_args(Kv4AttendArgs* a, const void* k_codes, const void* k_params, const void* v_codes, const void* v_params,
                int64_t pages, int kv_heads, int page_size, int d, const void* q, void* out, const int64_t* strides,
                const int32_t* tables, const int32_t* lengths, int requests, int n, int heads, int width, int64_t window,
                int64_t sinks, float scale, int dtype) {
  int rc = check_dtype(dtype);
  if (!rc) rc = check_cache(&a->c, k_codes, k_params, v_codes, v_params, pages, kv_heads, page_size, d);
  if (!rc) rc = attend_sizes(a, kv_heads, page_size, requests, n, heads, width, window, sinks);
  if (rc || requests == 0 || n == 0) return rc;
  if (!q || !out || !strides || !lengths || (width > 0 && !tables)) return set_error(SA_ERR_INVALID_ARG, "null pointer");
  a->q = q;
  a->out = out;
  a->q_r = strides[0];
  a->q_n = strides[1];
  a->q_h = strides[2];
  a->vec_q = rows_aligned(q, elem_size(dtype), strides[0] | strides[1], strides[2]);
  a->tables = tables;
  a->lengths = lengths;
  a->scale = scale;
  a->dtype = dtype;
  a->status = status_word();
  return SA_OK;
}

// The prefix's table, and the rows of all requests over it.
int prefix_sizes(Kv4AttendArgs* a, int prefix_width) {
  if (prefix_width < 0) return set_error(SA_ERR_INVALID_ARG, "sizes must be non-negative");
  if (((int64_t)prefix_width << a->c.page_shift) > 2147483647LL)
    return set_error(SA_ERR_UNSUPPORTED, "the prefix's table covers 2^31 tokens or more");
  if ((int64_t)a->requests * a->n * a->heads > 400000)
    return set_error(SA_ERR_UNSUPPORTED, "more than 400000 query rows over one prefix");
  a->prefix_width = prefix_width;
  return SA_OK;
}

// Entries that a CTA's threads take in turns, in steps of 31 bits that may pass the last entry by a CTA's width.
constexpr int kMostCounted = 1 << 30;

int check_workspace(const void* workspace, size_t have, size_t want) {
  if (want == 0) return SA_OK;
  if (!workspace || have < want) return set_error(SA_ERR_WORKSPACE, "the workspace has %zu bytes, %zu are needed", have, want);
  if ((uintptr_t)workspace & 255) return set_error(SA_ERR_WORKSPACE, "the workspace must be 256-byte aligned");
  return SA_OK;
}

int plan_pages(const int32_t* lengths, const int32_t* fresh, int32_t* tables, const int32_t* free_pages,
               const int32_t* free_count, int requests, int width, int free_size, int page_size, int max_tokens,
               int per_request, int prompts, int32_t* lengths_out, int32_t* offsets, int32_t* positions, int32_t* slots,
               int32_t* free_out, void* stream) {
  const int shift = page_shift_of(page_size);
  if (shift < 0) return set_error(SA_ERR_INVALID_ARG, "page_size must be 16, 32, 64, 128 or 256");
  if (requests < 0 || width < 0 || free_size < 0 || max_tokens < 0 || per_request < 0)
    return set_error(SA_ERR_INVALID_ARG, "sizes must be non-negative");
  if (per_request > 0 && (int64_t)requests * per_request != max_tokens)
    return set_error(SA_ERR_INVALID_ARG, "max_tokens must be requests * per_request");
  if ((int64_t)requests * width > 2147483647LL || free_size > (2147483647 >> shift))
    return set_error(SA_ERR_UNSUPPORTED, "the page table or the cache is too large");
  if (!offsets || !free_out || !free_count || (requests > 0 && (!lengths || !fresh || !lengths_out)) ||
      (requests > 0 && width > 0 && !tables) || (free_size > 0 && !free_pages) ||
      (max_tokens > 0 && (!positions || !slots)))
    return set_error(SA_ERR_INVALID_ARG, "null pointer");
  return launch_plan_pages(lengths, fresh, tables, free_pages, free_count, requests, width, free_size, shift,
                           max_tokens, per_request, prompts, lengths_out, offsets, positions, slots, free_out, status_word(),
                           (cudaStream_t)stream);
}

}  // namespace
}  // namespace sa

using namespace sa;

extern "C" {

int sa_serving_status(void* stream) {
  int* word = status_word();
  if (!word) return set_error(SA_ERR_CUDA, "no serving error word on this device");
  int64_t got[2] = {0, 0};
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e = cudaMemcpyAsync(got, word, sizeof(got), cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e != cudaSuccess) return set_error(SA_ERR_CUDA, "serving status read: %s", cudaGetErrorString(e));
  int code = 0;
  memcpy(&code, got, sizeof(int));
  if (code == 0) return SA_OK;
  e = cudaMemsetAsync(word, 0, sizeof(got), s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e != cudaSuccess) return set_error(SA_ERR_CUDA, "serving status reset: %s", cudaGetErrorString(e));
  const long long at = (long long)got[1];
  switch (code) {
    case kBadPage: return set_error(SA_ERR_INVALID_ARG, "page %lld lies outside the cache", at);
    case kBadSlot: return set_error(SA_ERR_INVALID_ARG, "the slot of token %lld lies outside the cache", at);
    case kBadLength: return set_error(SA_ERR_INVALID_ARG, "request %lld is longer than its row of the page table", at);
    case kBadOffsets: return set_error(SA_ERR_INVALID_ARG, "the offsets of request %lld are out of order or out of range", at);
    case kNoPages: return set_error(SA_ERR_INVALID_ARG, "%lld pages wanted, more than are free", at);
    case kHeld: return set_error(SA_ERR_INVALID_ARG, "request %lld holds tokens already, which its prompt does not see", at);
    case kBadList: return set_error(SA_ERR_INVALID_ARG, "entry %lld of a list of pages is not above the one before, or leaves the table", at);
    case kBadPrefix: return set_error(SA_ERR_INVALID_ARG, "the prefix is longer than its table (request %lld asked first)", at);
    case kNoRows: return set_error(SA_ERR_INVALID_ARG, "%lld entries, more than the output holds", at);
    default: break;
  }
  if (code >= kCheckFirst && code <= kCheckLast)
    return set_error(SA_ERR_DEVICE_CHECK, "device check %d failed at index %lld", code, at);
  return set_error(SA_ERR_TIMEOUT, "a bounded device-side wait gave up (wait code %d)", code);
}

int sa_window_attention_workspace_size(int batch, int heads, int kv_heads, int64_t n, int64_t m, int d, int dv,
                                       int64_t window, int64_t sinks, int dtype, size_t* bytes) {
  if (!bytes) return set_error(SA_ERR_INVALID_ARG, "null output pointer");
  int rc = check_dtype(dtype);
  if (!rc) rc = check_heads(heads, kv_heads);
  if (rc) return rc;
  if (batch < 0 || n < 0 || m < 0 || d <= 0 || dv <= 0 || window < 0 || sinks < 0) return set_error(SA_ERR_INVALID_ARG, "bad sizes");
  *bytes = 0;
  if (batch == 0 || n == 0 || m < n) return SA_OK;
  if (dtype == SA_REP_FLOAT32) {
    *bytes = window_tf32_bytes(batch, heads, kv_heads, n, m, d, dv, window, sinks_of(sinks));
  } else if (d <= 128 && dv <= 128) {
    WindowArgs a{};
    a.batch = batch;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.n = n;
    a.m = m;
    a.dv = dv;
    a.window = window_of(window);
    a.sinks = sinks_of(sinks);
    *bytes = window_tc_bytes(a);
  }
  return SA_OK;
}

int sa_window_attention(const void* q, const void* k, const void* v, void* out, const int64_t* strides, int batch,
                        int heads, int kv_heads, int64_t n, int64_t m, int d, int dv, int64_t window, int64_t sinks,
                        float scale, int dtype, const int32_t* cu_q, const int32_t* cu_k, int zero_behind, void* workspace,
                        size_t workspace_bytes, void* stream) {
  int rc = check_dtype(dtype);
  if (!rc) rc = check_heads(heads, kv_heads);
  if (rc) return rc;
  if (batch < 0 || n < 0 || m < 0) return set_error(SA_ERR_INVALID_ARG, "batch, n and m must be non-negative");
  if (d <= 0 || d > SA_MAX_DIM || dv <= 0 || dv > SA_MAX_VALUE_DIM)
    return set_error(SA_ERR_INVALID_ARG, "head widths must lie in [1, %d]", SA_MAX_DIM);
  if (window < 0 || sinks < 0) return set_error(SA_ERR_INVALID_ARG, "window and sinks must be non-negative");
  if (n > 2147483647LL || m > 2147483647LL) return set_error(SA_ERR_UNSUPPORTED, "more than 2^31 - 1 rows");
  if ((cu_q == nullptr) != (cu_k == nullptr)) return set_error(SA_ERR_INVALID_ARG, "cu_q and cu_k come together");
  if (!cu_q && m < n) return set_error(SA_ERR_INVALID_ARG, "fewer keys than queries");
  if (batch == 0 || n == 0) return SA_OK;
  if (!q || !out || !strides || (m > 0 && (!k || !v))) return set_error(SA_ERR_INVALID_ARG, "null pointer");
  const WindowArgs a{q,          k,          v,          out,        strides[0], strides[1], strides[2],  strides[3],
                     strides[4], strides[5], strides[6], strides[7], strides[8], strides[9], strides[10], strides[11],
                     batch,      heads,      kv_heads,   n,          m,          d,          dv,
                     window_of(window), sinks_of(sinks), scale, dtype, cu_q, cu_k, status_word(), zero_behind};
  const char* simt = getenv("SA_FORCE_SIMT");
  if (window_tc_takes(a) && !(simt && simt[0] == '1')) return launch_window_tc(a, workspace, workspace_bytes, (cudaStream_t)stream);
  // float32 on the tensor cores: contiguous tensors and a workspace
  if (dtype == SA_REP_FLOAT32 && !cu_q && workspace && a.status && contiguous(batch, a.q_b, heads, a.q_h, n, a.q_n, d) &&
      contiguous(batch, a.k_b, kv_heads, a.k_h, m, a.k_n, d) && contiguous(batch, a.v_b, kv_heads, a.v_h, m, a.v_n, dv) &&
      contiguous(batch, a.o_b, heads, a.o_h, n, a.o_n, dv) &&
      window_tf32_bytes(batch, heads, kv_heads, n, m, d, dv, window, sinks_of(sinks)) > 0)
    return window_tf32_run(a, workspace, workspace_bytes, (cudaStream_t)stream);
  return launch_window_simt(a, (cudaStream_t)stream);
}

int sa_plan_kv_pages(const int32_t* lengths, const int32_t* fresh, int32_t* tables, const int32_t* free_pages,
                     const int32_t* free_count, int requests, int width, int free_size, int page_size, int max_tokens,
                     int per_request, int32_t* lengths_out, int32_t* offsets, int32_t* positions, int32_t* slots, int32_t* free_out,
                     void* stream) {
  return plan_pages(lengths, fresh, tables, free_pages, free_count, requests, width, free_size, page_size, max_tokens,
                    per_request, 0, lengths_out, offsets, positions, slots, free_out, stream);
}

int sa_plan_kv_prompts(const int32_t* lengths, const int32_t* fresh, int32_t* tables, const int32_t* free_pages,
                       const int32_t* free_count, int requests, int width, int free_size, int page_size, int max_tokens,
                       int32_t* lengths_out, int32_t* offsets, int32_t* positions, int32_t* slots, int32_t* free_out,
                       void* stream) {
  return plan_pages(lengths, fresh, tables, free_pages, free_count, requests, width, free_size, page_size, max_tokens, 0,
                    1, lengths_out, offsets, positions, slots, free_out, stream);
}

int sa_release_kv_pages(int32_t* lengths, int32_t* tables, const uint8_t* drop, int32_t* free_pages,
                        int32_t* free_count, int requests, int width, int free_size, int page_size, void* stream) {
  const int shift = page_shift_of(page_size);
  if (shift < 0) return set_error(SA_ERR_INVALID_ARG, "page_size must be 16, 32, 64, 128 or 256");
  if (requests < 0 || width < 0 || free_size < 0) return set_error(SA_ERR_INVALID_ARG, "sizes must be non-negative");
  if (requests == 0) return SA_OK;
  if (!lengths || !drop || !free_count || (width > 0 && !tables) || (free_size > 0 && !free_pages)) return set_error(SA_ERR_INVALID_ARG, "null pointer");
  return launch_release_pages(lengths, tables, drop, free_pages, free_count, requests, width, free_size, shift,
                              status_word(), (cudaStream_t)stream);
}

int sa_qk_norm_rotary(const void* q, const void* k, void* q_out, void* k_out, const int32_t* positions,
                      const void* q_weight, const void* k_weight, const double* frequencies, const int64_t* strides,
                      int64_t tokens, int heads, int kv_heads, int d, int half, float eps, int interleaved,
                      int zero_skipped, int dtype, void* stream) {
  int rc = check_dtype(dtype);
  if (rc) return rc;
  if (tokens < 0 || heads < 0 || kv_heads < 0 || heads + kv_heads == 0)
    return set_error(SA_ERR_INVALID_ARG, "at least one head is needed");
  if (d <= 0 || d > SA_MAX_DIM) return set_error(SA_ERR_INVALID_ARG, "the head width must lie in [1, %d]", SA_MAX_DIM);
  if (half < 0 || 2 * half > d) return set_error(SA_ERR_INVALID_ARG, "more rotated columns than the head has");
  if (tokens == 0) return SA_OK;
  if (!strides || !positions || (heads > 0 && (!q || !q_out)) || (kv_heads > 0 && (!k || !k_out)) ||
      (half > 0 && !frequencies))
    return set_error(SA_ERR_INVALID_ARG, "null pointer");
  return launch_rotary(q, k, q_out, k_out, positions, q_weight, k_weight, frequencies, strides, tokens, heads, kv_heads,
                       d, half, eps, interleaved, zero_skipped, dtype, (cudaStream_t)stream);
}

int sa_kv4_append(void* k_codes, void* k_params, void* v_codes, void* v_params, int64_t pages, int heads,
                  int page_size, int d, const void* k, const void* v, const int64_t* strides, const int32_t* slots,
                  int64_t tokens, int dtype, void* stream) {
  Kv4AppendArgs a{};
  int rc = check_dtype(dtype);
  if (!rc) rc = check_cache(&a.c, k_codes, k_params, v_codes, v_params, pages, heads, page_size, d);
  if (rc) return rc;
  if (tokens < 0) return set_error(SA_ERR_INVALID_ARG, "tokens must be non-negative");
  if (tokens == 0) return SA_OK;
  if (!k || !v || !strides || !slots) return set_error(SA_ERR_INVALID_ARG, "null pointer");
  a.k = k;
  a.v = v;
  a.k_t = strides[0];
  a.k_h = strides[1];
  a.v_t = strides[2];
  a.v_h = strides[3];
  a.slots = slots;
  a.tokens = tokens;
  a.status = status_word();
  return launch_kv4_append(a, dtype, (cudaStream_t)stream);
}

int sa_kv4_read(const void* k_codes, const void* k_params, const void* v_codes, const void* v_params, int64_t pages,
                int heads, int page_size, int d, void* k, void* v, const int32_t* slots, int64_t tokens, int dtype,
                void* stream) {
  Kv4ReadArgs a{};
  int rc = check_dtype(dtype);
  if (!rc) rc = check_cache(&a.c, k_codes, k_params, v_codes, v_params, pages, heads, page_size, d);
  if (rc) return rc;
  if (tokens < 0) return set_error(SA_ERR_INVALID_ARG, "tokens must be non-negative");
  if (tokens == 0) return SA_OK;
  if (!k || !v || !slots) return set_error(SA_ERR_INVALID_ARG, "null pointer");
  a.k = k;
  a.v = v;
  a.slots = slots;
  a.tokens = tokens;
  a.status = status_word();
  return launch_kv4_read(a, dtype, (cudaStream_t)stream);
}

int sa_kv4_attend(const void* k_codes, const void* k_params, const void* v_codes, const void* v_params, int64_t pages,
                  int kv_heads, int page_size, int d, const void* q, void* out, const int64_t* strides,
                  const int32_t* tables, const int32_t* lengths, int requests, int n, int heads, int width,
                  int64_t window, int64_t sinks, float scale, int dtype, void* stream) {
  Kv4AttendArgs a{};
  const int rc = attend_args(&a, k_codes, k_params, v_codes, v_params, pages, kv_heads, page_size, d, q, out, strides,
                             tables, lengths, requests, n, heads, width, window, sinks, scale, dtype);
  if (rc || requests == 0 || n == 0) return rc;
  return launch_kv4_attend(a, (cudaStream_t)stream);
}

int sa_kv4_attend_pages(const void* k_codes, const void* k_params, const void* v_codes, const void* v_params, int64_t pages,
                        int kv_heads, int page_size, int d, const void* q, void* out, const int64_t* strides,
                        const int32_t* tables, const int32_t* lengths, const int32_t* selected, int count, int requests, int n,
                        int heads, int width, float scale, int dtype, void* stream) {
  Kv4AttendArgs a{};
  const int rc = attend_args(&a, k_codes, k_params, v_codes, v_params, pages, kv_heads, page_size, d, q, out, strides,
                             tables, lengths, requests, n, heads, width, 0, 0, scale, dtype);
  if (rc) return rc;
  if (count < 0) return set_error(SA_ERR_INVALID_ARG, "sizes must be non-negative");
  if (count > kMostCounted) return set_error(SA_ERR_UNSUPPORTED, "count must not pass 2^30");
  if ((int64_t)requests * n > 65535) return set_error(SA_ERR_UNSUPPORTED, "more than 65535 queries in one call");
  if (requests == 0 || n == 0) return SA_OK;
  if (count > 0 && !selected) return set_error(SA_ERR_INVALID_ARG, "null pointer");
  a.pages = selected;
  a.count = count;
  return launch_kv4_attend_pages(a, (cudaStream_t)stream);
}

int sa_kv4_attend_weigh_workspace_size(int kv_heads, int page_size, int requests, int n, int heads, int width, int64_t window,
                                       int64_t sinks, size_t* bytes) {
  if (!bytes) return set_error(SA_ERR_INVALID_ARG, "null output pointer");
  Kv4AttendArgs a{};
  const int rc = attend_sizes(&a, kv_heads, page_size, requests, n, heads, width, window, sinks);
  if (rc) return rc;
  *bytes = kv4_weigh_bytes(a);
  return SA_OK;
}

int sa_kv4_attend_weigh(const void* k_codes, const void* k_params, const void* v_codes, const void* v_params, int64_t pages,
                        int kv_heads, int page_size, int d, const void* q, void* out, const int64_t* strides,
                        const int32_t* tables, const int32_t* lengths, int requests, int n, int heads, int width,
                        int64_t window, int64_t sinks, float scale, int dtype, float* weights, void* workspace,
                        size_t workspace_bytes, void* stream) {
  Kv4AttendArgs a{};
  const int rc = attend_args(&a, k_codes, k_params, v_codes, v_params, pages, kv_heads, page_size, d, q, out, strides,
                             tables, lengths, requests, n, heads, width, window, sinks, scale, dtype);
  if (rc || requests == 0 || n == 0) return rc;
  if (!weights) return set_error(SA_ERR_INVALID_ARG, "null pointer");
  const int bad = check_workspace(workspace, workspace_bytes, kv4_weigh_bytes(a));
  if (bad) return bad;
  a.weights = weights;
  return launch_kv4_attend_weigh(a, workspace, (cudaStream_t)stream);
}

int sa_kv4_reset_weights(float* weights, int64_t pages, int kv_heads, int page_size, const int32_t* slots, int64_t tokens,
                         void* stream) {
  const int shift = page_shift_of(page_size);
  if (shift < 0) return set_error(SA_ERR_INVALID_ARG, "page_size must be 16, 32, 64, 128 or 256");
  if (pages <= 0 || kv_heads <= 0) return set_error(SA_ERR_INVALID_ARG, "the cache needs at least one page and one head");
  if (tokens < 0) return set_error(SA_ERR_INVALID_ARG, "tokens must be non-negative");
  if (tokens == 0) return SA_OK;
  if (!weights || !slots) return set_error(SA_ERR_INVALID_ARG, "null pointer");
  return launch_kv4_reset_weights(weights, slots, tokens, pages, kv_heads, shift, status_word(), (cudaStream_t)stream);
}

int sa_kv4_attend_shared_workspace_size(int kv_heads, int page_size, int d, int requests, int n, int heads, int prefix_width,
                                        int64_t window, int64_t sinks, int dtype, size_t* bytes) {
  if (!bytes) return set_error(SA_ERR_INVALID_ARG, "null output pointer");
  Kv4AttendArgs a{};
  int rc = check_dtype(dtype);
  if (!rc) rc = attend_sizes(&a, kv_heads, page_size, requests, n, heads, 0, window, sinks);
  if (!rc) rc = prefix_sizes(&a, prefix_width);
  if (rc) return rc;
  if (d <= 0 || d > SA_MAX_DIM) return set_error(SA_ERR_INVALID_ARG, "the cache's head width must lie in [1, %d]", SA_MAX_DIM);
  a.c.dp = padded_dim(d);
  a.dtype = dtype;
  *bytes = kv4_shared_bytes(a);
  return SA_OK;
}

int sa_kv4_attend_shared(const void* k_codes, const void* k_params, const void* v_codes, const void* v_params, int64_t pages,
                         int kv_heads, int page_size, int d, const void* q, void* out, const int64_t* strides,
                         const int32_t* prefix_table, const int32_t* prefix_length, int prefix_width, const int32_t* tables,
                         const int32_t* lengths, int requests, int n, int heads, int width, int64_t window, int64_t sinks,
                         float scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  Kv4AttendArgs a{};
  int rc = attend_args(&a, k_codes, k_params, v_codes, v_params, pages, kv_heads, page_size, d, q, out, strides, tables,
                       lengths, requests, n, heads, width, window, sinks, scale, dtype);
  if (!rc) rc = prefix_sizes(&a, prefix_width);
  if (rc || requests == 0 || n == 0) return rc;
  if (!prefix_length || (prefix_width > 0 && !prefix_table)) return set_error(SA_ERR_INVALID_ARG, "null pointer");
  rc = check_workspace(workspace, workspace_bytes, kv4_shared_bytes(a));
  if (rc) return rc;
  a.prefix_table = prefix_table;
  a.prefix_length = prefix_length;
  return launch_kv4_attend_shared(a, workspace, (cudaStream_t)stream);
}

int sa_kv4_page_bounds(const void* k_codes, const void* k_params, const void* v_codes, const void* v_params, int64_t pages,
                       int kv_heads, int page_size, int d, void* bounds, const int32_t* tables, const int32_t* lengths,
                       const int32_t* fresh, int requests, int width, void* stream) {
  Kv4BoundsArgs a{};
  int rc = check_cache(&a.c, k_codes, k_params, v_codes, v_params, pages, kv_heads, page_size, d);
  if (!rc) rc = check_tables(requests, width, a.c.page_shift);
  if (rc || requests == 0 || width == 0) return rc;
  if (!bounds || !tables || !lengths || !fresh) return set_error(SA_ERR_INVALID_ARG, "null pointer");
  if ((uintptr_t)bounds & 15) return set_error(SA_ERR_INVALID_ARG, "the bounds must be 16-byte aligned");
  a.bounds = static_cast<__nv_bfloat16*>(bounds);
  a.tables = tables;
  a.lengths = lengths;
  a.fresh = fresh;
  a.requests = requests;
  a.width = width;
  a.status = status_word();
  return launch_kv4_bounds(a, (cudaStream_t)stream);
}

int sa_kv4_select_pages(const void* bounds, int64_t pages, int kv_heads, int page_size, int d, const void* q,
                        const int64_t* strides, const int32_t* tables, const int32_t* lengths, int requests, int n, int heads,
                        int width, int count, int first, int last, int dtype, int32_t* selected, void* stream) {
  Kv4SelectArgs a{};
  int rc = check_dtype(dtype);
  if (!rc) rc = check_heads(heads, kv_heads);
  if (rc) return rc;
  const int shift = page_shift_of(page_size);
  if (shift < 0) return set_error(SA_ERR_INVALID_ARG, "page_size must be 16, 32, 64, 128 or 256");
  if (pages <= 0) return set_error(SA_ERR_INVALID_ARG, "the cache needs at least one page and one head");
  if (d <= 0 || d > SA_MAX_DIM) return set_error(SA_ERR_INVALID_ARG, "the cache's head width must lie in [1, %d]", SA_MAX_DIM);
  if (n < 0 || count < 0) return set_error(SA_ERR_INVALID_ARG, "sizes must be non-negative");
  if (first < 0 || last < 0 || (int64_t)first + last > count)
    return set_error(SA_ERR_INVALID_ARG, "first and last must be non-negative, and no more than count together");
  if (count > kMostCounted) return set_error(SA_ERR_UNSUPPORTED, "count must not pass 2^30");
  rc = check_tables(requests, width, shift);
  if (rc) return rc;
  if (width > kSelectMaxPages)
    return set_error(SA_ERR_UNSUPPORTED, "a row of the page table has more than %d pages to select from", kSelectMaxPages);
  if (requests == 0 || n == 0 || count == 0) return SA_OK;
  if (!bounds || !q || !strides || !lengths || !selected || (width > 0 && !tables)) return set_error(SA_ERR_INVALID_ARG, "null pointer");
  if ((uintptr_t)bounds & 15) return set_error(SA_ERR_INVALID_ARG, "the bounds must be 16-byte aligned");
  a.c.pages = pages;
  a.c.heads = kv_heads;
  a.c.d = d;
  a.c.dp = padded_dim(d);
  a.c.page_shift = shift;
  a.bounds = static_cast<const __nv_bfloat16*>(bounds);
  a.q = q;
  a.q_r = strides[0];
  a.q_n = strides[1];
  a.q_h = strides[2];
  a.tables = tables;
  a.lengths = lengths;
  a.out = selected;
  a.requests = requests;
  a.n = n;
  a.heads = heads;
  a.width = width;
  a.count = count;
  a.first = first;
  a.last = last;
  a.status = status_word();
  return launch_kv4_select(a, dtype, (cudaStream_t)stream);
}

int sa_kv4_evict(void* k_codes, void* k_params, void* v_codes, void* v_params, int64_t pages, int kv_heads, int page_size,
                 int d, float* weights, int32_t* lengths, int32_t* tables, int32_t* free_pages, int32_t* free_count,
                 int requests, int width, int free_size, int keep, int limit, int first, int last, int32_t* kept,
                 int32_t* dropped, void* stream) {
  Kv4EvictArgs a{};
  int rc = check_cache(&a.c, k_codes, k_params, v_codes, v_params, pages, kv_heads, page_size, d);
  if (!rc) rc = check_tables(requests, width, a.c.page_shift);
  if (rc) return rc;
  if (free_size < 0) return set_error(SA_ERR_INVALID_ARG, "sizes must be non-negative");
  if (keep < 1 || limit < keep) return set_error(SA_ERR_INVALID_ARG, "keep must be positive, and limit no less");
  if (keep > kMostCounted) return set_error(SA_ERR_UNSUPPORTED, "keep must not pass 2^30");
  if (((int64_t)width << a.c.page_shift) > kMostCounted)
    return set_error(SA_ERR_UNSUPPORTED, "eviction: a row of the page table covers more than 2^30 tokens");
  if (first < 0 || last < 0 || (int64_t)first + last > keep)
    return set_error(SA_ERR_INVALID_ARG, "first and last must be non-negative, and no more than keep together");
  if (requests == 0) return SA_OK;
  if (!weights || !lengths || !free_count || !kept || !dropped || (width > 0 && !tables) || (free_size > 0 && !free_pages))
    return set_error(SA_ERR_INVALID_ARG, "null pointer");
  a.weights = weights;
  a.lengths = lengths;
  a.tables = tables;
  a.kept = kept;
  a.requests = requests;
  a.width = width;
  a.keep = keep;
  a.limit = limit;
  a.first = first;
  a.last = last;
  a.status = status_word();
  rc = prepare_shrink_requests(requests);   // what it refuses leaves the cache as it is
  if (!rc) rc = launch_kv4_evict(a, (cudaStream_t)stream);
  if (rc) return rc;
  return launch_shrink_requests(lengths, tables, free_pages, free_count, dropped, requests, width, free_size,
                                a.c.page_shift, keep, limit, a.status, (cudaStream_t)stream);
}

}  // extern "C"
