// Attention over selected pages of the 4-bit cache (kernel in kv4_attend.cuh).
#include "kv4_attend.cuh"

namespace sa {

int launch_kv4_attend_pages(const Kv4AttendArgs& a, cudaStream_t s) { return launch_mode<kSelected>(a, s); }

}  // namespace sa
