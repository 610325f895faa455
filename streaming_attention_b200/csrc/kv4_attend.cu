// Attention over all visible tokens of the 4-bit cache (kernel in kv4_attend.cuh).
#include "kv4_attend.cuh"

namespace sa {

int launch_kv4_attend(const Kv4AttendArgs& a, cudaStream_t s) { return launch_mode<kPlain>(a, s); }

}  // namespace sa
