// Attention of a ragged batch over the paged cache, prefixes shared by groups of sequences.
//   out = Σ_k exp(s_k - m) · v_k / (Σ_k exp(s_k - m) [+ exp(sink - m)]),  s_k = scale · q · k
// over the keys at positions p' <= p of the query, with a window p' > p - window. attn_plan.h cuts a call into workgroups,
// attn_tile.h and attn_wave.h compute them; here the parts of a row whose keys were split are joined.
#include "attn_mma.h"

namespace jamhip {

hipError_t launch_attn_f16(const AttnArgs& a, hipStream_t st);
hipError_t launch_attn_q8(const AttnArgs& a, hipStream_t st);
hipError_t launch_attn_q4(const AttnArgs& a, hipStream_t st);
hipError_t launch_attn_tree_f16(const AttnArgs& a, hipStream_t st);
hipError_t launch_attn_tree_q8(const AttnArgs& a, hipStream_t st);
hipError_t launch_attn_tree_q4(const AttnArgs& a, hipStream_t st);

namespace {

// The workspace slots of the parts that keys [lo, hi) of a row lie in, first[k] and count[k] of part k; returns their number.
JAMHIP_DEV int parts_of(const AttnPlan& p, int base, int lo, int hi, int (&first)[2], int (&count)[2]) {
#pragma unroll
    for (int k = 0; k < 2; k++) {
        first[k] = count[k] = 0;
        if (k >= p.n) continue;
        const AttnPart& q = p.part[k];
        const int a0 = q.mode == 2 ? max(0, lo - base) : lo, a1 = q.mode == 2 ? hi - base : q.mode == 1 ? min(hi, base) : hi;
        if (a0 >= a1) continue;
        first[k] = q.slot0 + a0 / q.chunk;
        count[k] = min((a1 - 1) / q.chunk, q.splits - 1) - a0 / q.chunk + 1;
    }
    return count[0] + count[1];
}

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
    const int pos = s.base + s.first + (t - s.t0);
    const int lo = g.window > 0 ? max(0, pos - g.window + 1) : 0, hi = min(s.base + s.len, pos + 1);
    constexpr int E = D > 128 ? 4 : D > 64 ? 2 : 1;   // elements a lane
    float m = -__builtin_inff(), l = 0.0f, o[E];
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = 0.0f;
    int first[2], count[2];
    const int all = parts_of(p, s.base, lo, hi, first, count);
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

// The same for drafted trees. A workgroup joins the heads of one token, whose parts are the same: what is looked up for them once takes longer
// than the join of a row. 16, 32 or 64 lanes a row, 4 elements each, so that a wave's loads are of 1024 bytes. 464 tokens of 64 heads of 64 in
// two parts, 15 MB: 9.9 us, 24 with a row a wave, as above.
template <int D> constexpr int join_lanes() { return D <= 64 ? 16 : D <= 128 ? 32 : 64; }
template <int D> constexpr int join_heads() { return 4 * (64 / join_lanes<D>()); }   // of a workgroup

template <int TYPE, int D> __global__ void __launch_bounds__(256) tree_join_kernel(AttnArgs a, AttnPlan p) {
    constexpr int G = join_lanes<D>(), R = 64 / G, PER = join_heads<D>();
    __shared__ float redo[4][ATTN_ROW_FLOATS];
    const Attn& g = a.g;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), sub = lane % G;
    const int chunks = (g.heads + PER - 1) / PER;
    const int wg = a.block0 + blockIdx.x, t = wg / chunks, head0 = (wg - t * chunks) * PER;
    const bool small = fits_lanes(g);
    BatchLanes lanes;
    if (small) lanes = batch_lanes(g);
    const int sq = small ? seq_of(lanes, t) : seq_of(g, t);
    if (sq < 0) return;
    const SeqInfo s = small ? seq_info(g, lanes, sq) : seq_info(g, sq);
    if (t - s.t0 >= s.nq) return;
    const TreeSpan span = tree_span(g, t, s);
    int first[2], count[2];   // a part between the first and the last key that it sees, none of whose keys it sees, holds a sum of zero
    const int all = parts_of(p, s.base, span_lo(span), span_hi(span), first, count);
    const int64_t n = (int64_t) g.n_tokens * g.heads;
    const bool has = D % (4 * G) == 0 || sub * 4 < D;
    const int h0 = head0 + wave * R, head = h0 + lane / G;
    if (h0 >= g.heads) return;
    const bool live = head < g.heads;
    const int64_t i = (int64_t) t * g.heads + (live ? head : h0);
    float m = -__builtin_inff(), l = 0.0f;
    float4_t o = {0, 0, 0, 0};
    for (int k0 = 0; k0 < all; k0 += G) {   // a part a lane for the weights, then all lanes of the row for each part's elements
        const int k = k0 + sub, slot = k < count[0] ? first[0] + k : first[1] + k - count[0], here = min(G, all - k0);
        const float2 ml = k < all ? a.ml[slot * n + i] : make_float2(-__builtin_inff(), 0.0f);
        float now = ml.x;
#pragma unroll
        for (int x = 1; x < G; x <<= 1) now = fmaxf(now, __shfl_xor(now, x));
        now = fmaxf(now, m);
        const float keep = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - now);
        const float w = ml.x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(ml.x - now);
        float sum = ml.y * w;
#pragma unroll
        for (int x = 1; x < G; x <<= 1) sum += __shfl_xor(sum, x);
        m = now;
        l = l * keep + sum;
        o *= keep;
        for (int j0 = 0; j0 < here; j0 += 8) {   // eight loads in flight
            float4_t v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int q = k0 + min(j0 + j, here - 1);
                const int64_t at = ((q < count[0] ? first[0] + q : first[1] + q - count[0]) * n + i) * D;
                v[j] = has ? *reinterpret_cast<const float4_t*>(a.acc + at + sub * 4) : float4_t{0, 0, 0, 0};
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float x = __shfl(w, lane - sub + min(j0 + j, here - 1));
                if (j0 + j < here && x != 0.0f) o += v[j] * x;   // what a part without a visible key holds is not looked at
            }
        }
    }
    if (g.sinks != nullptr) {
        const float x = g.sinks[live ? head : h0] * LOG2E, now = fmaxf(m, x), keep = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - now);
        l = l * keep + (now == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(x - now + WEIGHT_EXP));
        o *= keep;
    }
    bool bad = false;
    float* const dst = g.out + (int64_t) t * g.ldo + (int64_t) head * D + sub * 4;
    if (live && has) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            o[e] = l == 0.0f ? 0.0f : o[e] / l;
            bad |= !(fabsf(o[e]) < __builtin_inff());
        }
        if ((reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
            *reinterpret_cast<float4_t*>(dst) = o;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) dst[e] = o[e];
        }
    }
    const unsigned long long again = __ballot(bad);
    if (again)
        for (int r = 0; r < R; r++)
            if (again >> (r * G) & (G == 64 ? ~0ull : (1ull << G % 64) - 1)) attn_row<TYPE, true>(g, t, h0 + r, redo[wave]);
}

template <int TYPE, int D> void launch_join_part(const AttnArgs& a, const AttnPlan& p, uint32_t blocks, hipStream_t st) {
    if (a.g.masks != nullptr) tree_join_kernel<TYPE, D><<<blocks, 256, 0, st>>>(a, p);
    else attn_join_kernel<TYPE, D><<<blocks, 256, 0, st>>>(a, p);
}

template <int TYPE> hipError_t launch_join(const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
    const int dim = a.g.cache.dim, per = dim <= 64 ? join_heads<64>() : dim <= 128 ? join_heads<128>() : join_heads<256>();
    const int64_t blocks = a.g.masks != nullptr ? (int64_t) a.g.n_tokens * ((a.g.heads + per - 1) / per)
                                                : ((int64_t) a.g.n_tokens * a.g.heads + 3) / 4;
    return attn_runs(a, blocks, [&](const AttnArgs& a, uint32_t blocks) {
        switch (dim) {
            case 64: launch_join_part<TYPE, 64>(a, p, blocks, st); break;
            case 96: launch_join_part<TYPE, 96>(a, p, blocks, st); break;
            case 128: launch_join_part<TYPE, 128>(a, p, blocks, st); break;
            case 192: launch_join_part<TYPE, 192>(a, p, blocks, st); break;
            case 256: launch_join_part<TYPE, 256>(a, p, blocks, st); break;
            default: return hipErrorNotSupported;
        }
        return hipGetLastError();
    });
}

AttnPlan plan_of(const Attn& g) {
    return attn_plan(g.cache.dim, g.cache.kv, g.grp.d, g.n_tokens, g.n_seqs, g.n_prefixes, g.max_q, g.seq_cap, g.prefix_cap, g.masks != nullptr);
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
    const bool tree = g.masks != nullptr;
    for (int i = 0; i < p.n; i++) {
        a.part = p.part[i];
        const hipError_t e = type == F16    ? (tree ? launch_attn_tree_f16(a, st) : launch_attn_f16(a, st))
                             : type == Q8_0 ? (tree ? launch_attn_tree_q8(a, st) : launch_attn_q8(a, st))
                             : type == Q4_0 ? (tree ? launch_attn_tree_q4(a, st) : launch_attn_q4(a, st))
                                            : hipErrorNotSupported;
        if (e != hipSuccess) return e;
    }
    if (p.slots == 0) return hipSuccess;
    return type == F16 ? launch_join<F16>(a, p, st) : type == Q8_0 ? launch_join<Q8_0>(a, p, st) : launch_join<Q4_0>(a, p, st);
}

}  // namespace jamhip
