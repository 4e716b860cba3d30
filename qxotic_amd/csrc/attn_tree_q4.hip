// The attention kernels over a Q4_0 cache, of drafted trees.
#include "attn_launch.h"

namespace jamhip {

hipError_t launch_attn_tree_q4(const AttnArgs& a, hipStream_t st) { return launch_attn_part<Q4_0, true>(a, st); }

}  // namespace jamhip
