// Attention of a ragged batch over the paged cache, prefixes shared by groups of sequences.
//   out = Σ_k exp(s_k - m) · v_k / (Σ_k exp(s_k - m) [+ exp(sink - m)]),  s_k = scale · q · k
// over the keys at positions p' <= p of the query, with a window p' > p - window.
#include "attn.h"

namespace jamhip {

namespace {

template <int TYPE> __global__ void __launch_bounds__(256) attn_rows_kernel(Attn g) {
    __shared__ float lds[4][ATTN_ROW_FLOATS];
    const int64_t i = (int64_t) blockIdx.x * 4 + threadIdx.x / 64;
    if (i >= (int64_t) g.n_tokens * g.heads) return;
    attn_row<TYPE>(g, (int) (i / g.heads), (int) (i % g.heads), lds[threadIdx.x / 64]);
}

}  // namespace

hipError_t launch_attn(int type, const Attn& g, hipStream_t st) {
    if (g.n_tokens <= 0 || g.n_seqs <= 0) return hipSuccess;
    const int64_t blocks = ((int64_t) g.n_tokens * g.heads + 3) / 4;
    if (blocks > INT32_MAX) return hipErrorNotSupported;
    switch (type) {
        case F16: attn_rows_kernel<F16><<<(uint32_t) blocks, 256, 0, st>>>(g); break;
        case Q8_0: attn_rows_kernel<Q8_0><<<(uint32_t) blocks, 256, 0, st>>>(g); break;
        case Q4_0: attn_rows_kernel<Q4_0><<<(uint32_t) blocks, 256, 0, st>>>(g); break;
        default: return hipErrorNotSupported;
    }
    return hipGetLastError();
}

}  // namespace jamhip
