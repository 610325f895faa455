// Attention of a batch whose requests share a prefix: all queries over the prefix at
// once, then each request's over its own tokens with the prefix's sums joined
// (kernels in kv4_attend.cuh).
#include "kv4_attend.cuh"

namespace sa {

namespace {

size_t aligned(size_t x) { return (x + 255) & ~(size_t)255; }

int64_t all_rows(const Kv4AttendArgs& a) { return (int64_t)a.requests * a.n * (a.heads / a.c.heads); }

// Parts of the prefix.  kPrefix: each a launch dimension of clusters of eight CTAs, until
// there is a CTA for every place on the GPU, while a warp keeps four blocks.
int parts_of(const Kv4AttendArgs& a) {
  if (kv4_prefix_tc_takes(a, all_rows(a))) return kv4_prefix_tc_parts(a, all_rows(a));
  const int64_t tiles = a.c.heads * ceil_div(all_rows(a), 8);
  const int64_t longest = std::min<int64_t>((int64_t)a.prefix_width << a.c.page_shift, a.window + a.sinks + a.n);
  int parts = 1;
  while (parts < 16 && longest >= (int64_t)parts * 2 * 8 * 8 * 16 * 4 && tiles * parts * 8 < 148 * 2) parts *= 2;
  return parts;
}

}  // namespace

size_t kv4_shared_bytes(const Kv4AttendArgs& a) {
  const size_t each = (size_t)parts_of(a) * a.c.heads * all_rows(a);
  return aligned(each * sizeof(float2)) + each * a.c.dp * sizeof(float);
}

int launch_kv4_attend_shared(Kv4AttendArgs a, void* workspace, cudaStream_t s) {
  a.parts = parts_of(a);
  a.part_ml = static_cast<float2*>(workspace);
  a.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) +
                                      aligned((size_t)a.parts * a.c.heads * all_rows(a) * sizeof(float2)));
  Kv4AttendArgs prefix = a;
  prefix.width = a.prefix_width;
  const int rc = kv4_prefix_tc_takes(a, all_rows(a)) ? launch_kv4_prefix_tc(prefix, all_rows(a), s) : launch_mode<kPrefix>(prefix, s);
  return rc ? rc : launch_mode<kTail>(a, s);
}

}  // namespace sa
