// The attention kernels over a Q4_0 cache.
#include "attn_launch.h"

namespace jamhip {

hipError_t launch_attn_q4(const AttnArgs& a, hipStream_t st) { return launch_attn_part<Q4_0, false>(a, st); }

}  // namespace jamhip
