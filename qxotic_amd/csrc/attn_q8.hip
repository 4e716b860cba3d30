// The attention kernel over a Q8_0 cache.
#include "attn_tile.h"

namespace jamhip {

hipError_t launch_attn_q8(const AttnArgs& a, hipStream_t st) { return launch_attn_tile<Q8_0>(a, st); }

}  // namespace jamhip
