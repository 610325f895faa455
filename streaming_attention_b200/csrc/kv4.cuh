// The paged 4-bit key/value cache (layout in kv4.cu) and what its kernels take.
#pragma once

#include "serving.cuh"

namespace sa {

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
  const int32_t* tables;
  const int32_t* lengths;
  int requests, n, heads, width;
  int64_t window, sinks;
  float scale;
  int dtype;
  int* status;
};

int launch_kv4_append(const Kv4AppendArgs& a, int dtype, cudaStream_t s);
int launch_kv4_read(const Kv4ReadArgs& a, int dtype, cudaStream_t s);
int launch_kv4_attend(const Kv4AttendArgs& a, cudaStream_t s);

}  // namespace sa
