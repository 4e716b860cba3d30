// The attention kernels over a F16 cache.
#include "attn_launch.h"

namespace jamhip {

hipError_t launch_attn_f16(const AttnArgs& a, hipStream_t st) { return launch_attn_part<F16, false>(a, st); }

}  // namespace jamhip
