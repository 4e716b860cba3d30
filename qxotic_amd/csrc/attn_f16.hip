// The attention kernel over a F16 cache.
#include "attn_tile.h"

namespace jamhip {

hipError_t launch_attn_f16(const AttnArgs& a, hipStream_t st) { return launch_attn_tile<F16>(a, st); }

}  // namespace jamhip
