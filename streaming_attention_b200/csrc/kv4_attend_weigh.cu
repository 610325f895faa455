// Attention over the 4-bit cache that also adds up what each token's softmax weight
// was (kernel in kv4_attend.cuh):
//   weights[slot of j] += sum over the queries and heads that read key head h of p_j.
// p_j needs a row's whole sum, which stands when the last block is through: the
// attention leaves its scores (4 bytes for each query row beside the 136 of a token of
// width 128, most of them still in L2) and a second launch turns them into weights.
// Each slot is added to by one thread, its rows in order: the same bits every time as
// long as no page stands in two requests' tables; where one does, both are added.
//
// 32 requests of 5000..10000 tokens, 32 heads over 8 of 128: 117 us and 14 (275 MB, 42 us):
// the attention's instructions; a token a thread took the second 19.  A thread takes a token's rows one after the
// other, so a prompt's many rows are slow: 512 tokens at once over 8000, 4 heads a key head, 3245 us, of which
// attention without weights is 340.
#include "kv4_attend.cuh"

namespace sa {

namespace {

constexpr int kWeightThreads = 256;
constexpr int kEach = 4;   // tokens of a thread

__global__ void __launch_bounds__(kWeightThreads) weights_kernel(const Kv4AttendArgs a) {
  const int hk = blockIdx.y, r = blockIdx.z;
  const int rows = a.n * (a.heads / a.c.heads);
  const int cap = a.width << a.c.page_shift;
  const int length = max(a.lengths[r], 0);
  // the blocks of the attention's kernel
  const KeyRanges kr = key_ranges(length - a.n, length - 1, min(length, cap), a.window, a.sinks);
  const int sink_blocks = (int)((kr.first + 15) >> 4);
  const int win_begin = max((int)(kr.begin >> 4), sink_blocks), win_end = (int)((kr.end + 15) >> 4);
  const int64_t seen = (int64_t)(sink_blocks + max(win_end - win_begin, 0)) * 16;
  const int64_t of = (int64_t)r * a.c.heads + hk;
  const float* scores = a.scores + of * a.score_blocks * 16 * a.score_rows;
  const float2* ml = a.score_ml + of * a.score_rows;
  const int64_t t0 = (int64_t)blockIdx.x * kWeightThreads * kEach + threadIdx.x;
  float* to[kEach];
  float sum[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int64_t t = t0 + i * kWeightThreads;
    const int v = (int)(t >> 4), j = (v < sink_blocks ? v : win_begin + v - sink_blocks) * 16 + (int)(t & 15);
    const int page = t < seen && j < length ? __ldg(a.tables + (int64_t)r * a.width + (j >> a.c.page_shift)) : -1;
    // (a bad page is reported by the attention)
    to[i] = page < 0 || page >= a.c.pages ? nullptr
                                          : a.weights + ((page * (int64_t)a.c.heads + hk) << a.c.page_shift) +
                                                (j & ((1 << a.c.page_shift) - 1));
    sum[i] = 0.0f;
  }
  previous_has_ended();
  for (int row = 0; row < rows; row += 2) {
    const float2 y = ml[row], z = row + 1 < rows ? ml[row + 1] : make_float2(0.0f, 0.0f);
    float2 x[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      x[i] = to[i] ? *reinterpret_cast<const float2*>(scores + (t0 + i * kWeightThreads) * a.score_rows + row)
                   : make_float2(-INFINITY, -INFINITY);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (x[i].x != -INFINITY) sum[i] += ex2(x[i].x + y.x) * y.y;
      if (row + 1 < rows && x[i].y != -INFINITY) sum[i] += ex2(x[i].y + z.x) * z.y;
    }
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (to[i]) atomicAdd(to[i], sum[i]);
}

// Zero for the weights of slots.
__global__ void __launch_bounds__(kWeightThreads)
reset_weights_kernel(float* weights, const int32_t* slots, int64_t tokens, int64_t pages, int heads, int page_shift,
                     int* status) {
  const int64_t x = (int64_t)blockIdx.x * kWeightThreads + threadIdx.x;
  if (x >= tokens * heads) return;
  const int64_t t = x / heads;
  const int h = (int)(x - t * heads);
  const int64_t slot = slots[t];
  if (slot < 0) return;
  const int64_t page = slot >> page_shift;
  if (page >= pages) {
    if (h == 0) report(status, kBadSlot, t);
    return;
  }
  weights[((page * heads + h) << page_shift) + (slot & ((1 << page_shift) - 1))] = 0.0f;
}

// Blocks of 16 tokens that one request's queries can see at most.
int64_t score_blocks_of(int64_t cap, int64_t n, int64_t window, int64_t sinks) {
  return std::min(ceil_div(cap, 16), ceil_div(std::min(sinks, cap), 16) + ceil_div(std::min(window + n, cap), 16) + 1);
}

size_t aligned(size_t x) { return (x + 255) & ~(size_t)255; }

}  // namespace

size_t kv4_weigh_bytes(const Kv4AttendArgs& a) {
  const int64_t rows = a.n * (int64_t)(a.heads / a.c.heads);
  const size_t each = (size_t)a.requests * a.c.heads * ((rows + 1) & ~1);
  return aligned(each * sizeof(float2)) +
         each * 16 * score_blocks_of((int64_t)a.width << a.c.page_shift, a.n, a.window, a.sinks) * sizeof(float);
}

int launch_kv4_attend_weigh(Kv4AttendArgs a, void* workspace, cudaStream_t s) {
  a.score_rows = (int)((a.n * (int64_t)(a.heads / a.c.heads) + 1) & ~1);
  a.score_blocks = score_blocks_of((int64_t)a.width << a.c.page_shift, a.n, a.window, a.sinks);
  a.score_ml = static_cast<float2*>(workspace);
  a.scores = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) +
                                      aligned((size_t)a.requests * a.c.heads * a.score_rows * sizeof(float2)));
  if (a.c.heads > 65535) return set_error(SA_ERR_UNSUPPORTED, "kv4 weights: grid too large");
  const int rc = launch_mode<kWeigh>(a, s);
  if (rc || a.score_blocks == 0) return rc;
  cudaLaunchConfig_t cfg{};   // what needs no scores of it, and its launch, run beside the attention's last CTAs
  cfg.gridDim = dim3((unsigned)ceil_div(a.score_blocks * 16, kWeightThreads * kEach), a.c.heads, a.requests);
  cfg.blockDim = dim3(kWeightThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, weights_kernel, a);
  if (e != cudaSuccess) return set_error(SA_ERR_CUDA, "kv4 weights_kernel: %s", cudaGetErrorString(e));
  return check_launch("kv4 weights_kernel");
}

int launch_kv4_reset_weights(float* weights, const int32_t* slots, int64_t tokens, int64_t pages, int heads, int page_shift,
                             int* status, cudaStream_t s) {
  const int64_t ctas = ceil_div(tokens * heads, kWeightThreads);
  if (ctas > 2147483647LL) return set_error(SA_ERR_UNSUPPORTED, "kv4 reset: too many tokens in one call");
  reset_weights_kernel<<<(unsigned)ctas, kWeightThreads, 0, s>>>(weights, slots, tokens, pages, heads, page_shift, status);
  return check_launch("kv4 reset_weights_kernel");
}

}  // namespace sa
