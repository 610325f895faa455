// The paged 4-bit key/value cache (layout in kv4.cu) and what its kernels take.
#pragma once

#include "serving.cuh"

namespace sa {

// A kernel that the next one in the stream need not wait for to start, and the place
// where that one needs what it wrote.  Only for two kernels of one call, the first of them launched
// in the ordinary way: of other neighbours in the stream nothing is known.
__device__ __forceinline__ void next_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void previous_has_ended() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

struct Kv4Cache {
  uint8_t* k_codes;
  __nv_bfloat16* k_params;
  uint8_t* v_codes;
  __nv_bfloat16* v_params;
  int64_t pages;
  int heads, d, dp, page_shift;
};

struct Kv4AppendArgs {
  Kv4Cache c;
  const void* k;
  const void* v;
  int64_t k_t, k_h, v_t, v_h;   // strides in elements
  const int32_t* slots;
  int64_t tokens;
  int* status;
};

struct Kv4ReadArgs {
  Kv4Cache c;
  void* k;   // [tokens, heads, d]
  void* v;
  const int32_t* slots;
  int64_t tokens;
  int* status;
};

struct Kv4AttendArgs {
  Kv4Cache c;
  const void* q;   // [requests, n, heads, d]
  void* out;
  int64_t q_r, q_n, q_h;   // strides of q in elements (out is contiguous)
  int vec_q;               // rows of q start on 16-byte borders
  const int32_t* tables;
  const int32_t* lengths;
  int requests, n, heads, width;
  int64_t window, sinks;
  float scale;
  int dtype;
  int* status;
  // selected pages: [requests, n, key heads, count]
  const int32_t* pages;
  int count;
  // weights: scores [requests, key heads, score_blocks, 16, score_rows] in base 2, and of
  // each row what is added to a score before 2^x and the factor behind
  float* scores;
  float2* score_ml;
  int64_t score_blocks;
  int score_rows;
  float* weights;   // [pages, heads, page]
  // a shared prefix, and the unfinished sums of `parts` parts of it: [parts, key heads,
  // dp / 4, rows, 4], maximum and total [parts, key heads, rows], rows = requests * n * group
  const int32_t* prefix_table;
  const int32_t* prefix_length;
  int prefix_width;
  float* part_o;
  float2* part_ml;
  int parts;
};

struct Kv4BoundsArgs {
  Kv4Cache c;
  __nv_bfloat16* bounds;   // [pages, heads, 2, dp]
  const int32_t* tables;
  const int32_t* lengths;
  const int32_t* fresh;    // the newest tokens whose pages are looked at
  int requests, width;
  int* status;
};

constexpr int kSelectMaxPages = 24576;   // pages of a request: their scores stand in shared memory

struct Kv4SelectArgs {
  Kv4Cache c;
  const __nv_bfloat16* bounds;
  const void* q;   // [requests, n, heads, d]
  int64_t q_r, q_n, q_h;
  const int32_t* tables;
  const int32_t* lengths;
  int32_t* out;    // [requests, n, key heads, count]
  int requests, n, heads, width, count, first, last;
  int* status;
};

struct Kv4EvictArgs {
  Kv4Cache c;
  float* weights;   // [pages, heads, page]
  const int32_t* lengths;
  const int32_t* tables;
  int32_t* kept;    // [requests, heads, keep]
  int requests, width, keep, limit, first, last;
  int fits;         // tokens whose weights stand in shared memory
  int* status;
};

int launch_kv4_append(const Kv4AppendArgs& a, int dtype, cudaStream_t s);
int launch_kv4_read(const Kv4ReadArgs& a, int dtype, cudaStream_t s);
int launch_kv4_attend(const Kv4AttendArgs& a, cudaStream_t s);
int launch_kv4_attend_pages(const Kv4AttendArgs& a, cudaStream_t s);
size_t kv4_weigh_bytes(const Kv4AttendArgs& a);
int launch_kv4_attend_weigh(Kv4AttendArgs a, void* workspace, cudaStream_t s);
int launch_kv4_reset_weights(float* weights, const int32_t* slots, int64_t tokens, int64_t pages, int heads, int page_shift,
                             int* status, cudaStream_t s);
bool kv4_prefix_tc_takes(const Kv4AttendArgs& a, int64_t rows);
int kv4_prefix_tc_parts(const Kv4AttendArgs& a, int64_t rows);
int launch_kv4_prefix_tc(const Kv4AttendArgs& a, int64_t rows, cudaStream_t s);
size_t kv4_shared_bytes(const Kv4AttendArgs& a);
int launch_kv4_attend_shared(Kv4AttendArgs a, void* workspace, cudaStream_t s);
int launch_kv4_bounds(const Kv4BoundsArgs& a, cudaStream_t s);
int launch_kv4_select(const Kv4SelectArgs& a, int dtype, cudaStream_t s);
int launch_kv4_evict(const Kv4EvictArgs& a, cudaStream_t s);

}  // namespace sa
