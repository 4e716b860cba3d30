// Launches of the attention kernels over one cache type.
#pragma once

#include "attn_tile.h"
#include "attn_wave.h"

namespace jamhip {

template <int TYPE, int D> hipError_t launch_attn_part(const AttnArgs& a, hipStream_t st) {
    return attn_runs(a, (int64_t) a.g.cache.kv * a.part.tiles * a.part.splits, [&](const AttnArgs& a, uint32_t blocks) {
        switch (a.part.cfg) {
            case 0: attn_wave_kernel<TYPE, D, 16><<<blocks, 256, 0, st>>>(a); break;
            case 1:
                if constexpr (D <= ATTN_WIDE_DIM) attn_wave_kernel<TYPE, D, 32><<<blocks, 256, 0, st>>>(a);
                else return hipErrorNotSupported;   // attn_cfg does not choose it
                break;
            default: attn_tile_kernel<TYPE, D><<<blocks, 256, 0, st>>>(a); break;
        }
        return hipGetLastError();
    });
}

template <int TYPE> hipError_t launch_attn_part(const AttnArgs& a, hipStream_t st) {
    switch (a.g.cache.dim) {
        case 64: return launch_attn_part<TYPE, 64>(a, st);
        case 96: return launch_attn_part<TYPE, 96>(a, st);
        case 128: return launch_attn_part<TYPE, 128>(a, st);
        case 192: return launch_attn_part<TYPE, 192>(a, st);
        case 256: return launch_attn_part<TYPE, 256>(a, st);
    }
    return hipErrorNotSupported;
}

}  // namespace jamhip
