// The attention kernels over an F16 cache, of drafted trees.
#include "attn_launch.h"

namespace jamhip {

hipError_t launch_attn_tree_f16(const AttnArgs& a, hipStream_t st) { return launch_attn_part<F16, true>(a, st); }

}  // namespace jamhip
