// The attention kernels over a Q8_0 cache.
#include "attn_launch.h"

namespace jamhip {

hipError_t launch_attn_q8(const AttnArgs& a, hipStream_t st) { return launch_attn_part<Q8_0, false>(a, st); }

}  // namespace jamhip
