// Attention of a ragged batch over the paged cache, prefixes shared by groups of sequences.
//   out = Σ_k exp(s_k - m) · v_k / (Σ_k exp(s_k - m) [+ exp(sink - m)]),  s_k = scale · q · k
// over the keys at positions p' <= p of the query, with a window p' > p - window. attn_plan.h cuts a call into workgroups,
// attn_tile.h and attn_wave.h compute them; here the parts of a row whose keys were split are joined.
#include "attn_mma.h"

namespace jamhip {

hipError_t launch_attn_f16(const AttnArgs& a, hipStream_t st);
hipError_t launch_attn_q8(const AttnArgs& a, hipStream_t st);
hipError_t launch_attn_q4(const AttnArgs& a, hipStream_t st);

namespace {

// 2048 rows of 128 in 33 parts, 35 MB: 9.9 us; with each part's load behind the one before 16.6.
// One output row a wave: its parts (m_i, l_i, o_i) joined as Σ 2^(m_i - M) o_i / Σ 2^(m_i - M) l_i over the parts whose keys it
// sees any of (no other part was written).
template <int TYPE, int D> __global__ void __launch_bounds__(256) attn_join_kernel(AttnArgs a, AttnPlan p) {
    __shared__ float redo[4][ATTN_ROW_FLOATS];
    const Attn& g = a.g;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t n = (int64_t) g.n_tokens * g.heads, i = (a.block0 + (int64_t) blockIdx.x) * 4 + wave;
    if (i >= n) return;
    const int t = (int) (i / g.heads), head = (int) (i - (int64_t) t * g.heads);
    const bool small = fits_lanes(g);
    BatchLanes lanes;
    if (small) lanes = batch_lanes(g);
    const int sq = small ? seq_of(lanes, t) : seq_of(g, t);
    if (sq < 0) return;
    const SeqInfo s = small ? seq_info(g, lanes, sq) : seq_info(g, sq);
    if (t - s.t0 >= s.nq) return;
    const int pos = s.base + s.first + (t - s.t0), lo = g.window > 0 ? max(0, pos - g.window + 1) : 0, hi = min(s.base + s.len, pos + 1);
    constexpr int E = D > 128 ? 4 : D > 64 ? 2 : 1;   // elements a lane
    float m = -__builtin_inff(), l = 0.0f, o[E];
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = 0.0f;
    int first[2] = {0, 0}, count[2] = {0, 0};   // workspace slots
    for (int k = 0; k < p.n; k++) {
        const AttnPart& q = p.part[k];
        const int a0 = q.mode == 2 ? max(0, lo - s.base) : lo, a1 = q.mode == 2 ? hi - s.base : q.mode == 1 ? min(hi, s.base) : hi;
        if (a0 >= a1) continue;
        first[k] = q.slot0 + a0 / q.chunk;
        count[k] = min((a1 - 1) / q.chunk, q.splits - 1) - a0 / q.chunk + 1;
    }
    const int all = count[0] + count[1];
    for (int k0 = 0; k0 < all; k0 += 64) {   // a part a lane for the weights, then all lanes for each part's elements
        const int k = k0 + lane, slot = k < count[0] ? first[0] + k : first[1] + k - count[0];
        const float2 ml = k < all ? a.ml[slot * n + i] : make_float2(-__builtin_inff(), 0.0f);
        float now = ml.x;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) now = fmaxf(now, __shfl_xor(now, x));
        now = fmaxf(now, m);
        const float keep = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - now);
        const float w = ml.x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(ml.x - now);
        m = now;
        l = l * keep + wave_sum(ml.y * w);
#pragma unroll
        for (int e = 0; e < E; e++) o[e] *= keep;
        const int here = min(64, all - k0);
        for (int j0 = 0; j0 < here; j0 += 8) {   // eight loads in flight
            float v[8][E];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int q = k0 + min(j0 + j, here - 1);
                const float* src = a.acc + ((q < count[0] ? first[0] + q : first[1] + q - count[0]) * n + i) * D;
#pragma unroll
                for (int e = 0; e < E; e++) v[j][e] = D % (64 * E) == 0 || lane * E + e < D ? src[lane * E + e] : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float x = j0 + j < here ? lane_f(w, min(j0 + j, here - 1)) : 0.0f;
                if (x != 0.0f)   // what a part without a visible key holds is not looked at
#pragma unroll
                    for (int e = 0; e < E; e++) o[e] += v[j][e] * x;
            }
        }
    }
    if (g.sinks != nullptr) {
        const float x = g.sinks[head] * LOG2E, now = fmaxf(m, x), keep = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - now);
        l = l * keep + (now == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(x - now + WEIGHT_EXP));
#pragma unroll
        for (int e = 0; e < E; e++) o[e] *= keep;
    }
    bool bad = false;
#pragma unroll
    for (int e = 0; e < E; e++) {
        o[e] = l == 0.0f ? 0.0f : o[e] / l;
        bad |= !(fabsf(o[e]) < __builtin_inff());
        const int d = lane * E + e;
        if (d < D) g.out[(int64_t) t * g.ldo + (int64_t) head * D + d] = o[e];
    }
    if (__any(bad)) attn_row<TYPE>(g, t, head, redo[wave]);
}

template <int TYPE> hipError_t launch_join(const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
    return attn_runs(a, ((int64_t) a.g.n_tokens * a.g.heads + 3) / 4, [&](const AttnArgs& a, uint32_t blocks) {
        switch (a.g.cache.dim) {
            case 64: attn_join_kernel<TYPE, 64><<<blocks, 256, 0, st>>>(a, p); break;
            case 96: attn_join_kernel<TYPE, 96><<<blocks, 256, 0, st>>>(a, p); break;
            case 128: attn_join_kernel<TYPE, 128><<<blocks, 256, 0, st>>>(a, p); break;
            case 192: attn_join_kernel<TYPE, 192><<<blocks, 256, 0, st>>>(a, p); break;
            case 256: attn_join_kernel<TYPE, 256><<<blocks, 256, 0, st>>>(a, p); break;
            default: return hipErrorNotSupported;
        }
        return hipGetLastError();
    });
}

AttnPlan plan_of(const Attn& g) {
    return attn_plan(g.cache.dim, g.cache.kv, g.grp.d, g.n_tokens, g.n_seqs, g.n_prefixes, g.max_q, g.seq_cap, g.prefix_cap);
}

}  // namespace

size_t attn_workspace(const Attn& g) {
    const size_t rows = (size_t) plan_of(g).slots * g.n_tokens * g.heads;
    return rows * (g.cache.dim + 2) * sizeof(float);
}

hipError_t launch_attn(int type, const Attn& g, void* work, hipStream_t st) {
    if (g.n_tokens <= 0 || g.n_seqs <= 0) return hipSuccess;
    const AttnPlan p = plan_of(g);
    if (p.n == 0) return hipErrorNotSupported;
    AttnArgs a{};
    a.g = g;
    a.acc = static_cast<float*>(work);
    a.ml = reinterpret_cast<float2*>(a.acc + (size_t) p.slots * g.n_tokens * g.heads * g.cache.dim);
    for (int i = 0; i < p.n; i++) {
        a.part = p.part[i];
        const hipError_t e = type == F16 ? launch_attn_f16(a, st) : type == Q8_0 ? launch_attn_q8(a, st)
                           : type == Q4_0 ? launch_attn_q4(a, st) : hipErrorNotSupported;
        if (e != hipSuccess) return e;
    }
    if (p.slots == 0) return hipSuccess;
    return type == F16 ? launch_join<F16>(a, p, st) : type == Q8_0 ? launch_join<Q8_0>(a, p, st) : launch_join<Q4_0>(a, p, st);
}

}  // namespace jamhip
