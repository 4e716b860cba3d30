// The attention kernels over a Q8_0 cache, of drafted trees.
#include "attn_launch.h"

namespace jamhip {

hipError_t launch_attn_tree_q8(const AttnArgs& a, hipStream_t st) { return launch_attn_part<Q8_0, true>(a, st); }

}  // namespace jamhip
