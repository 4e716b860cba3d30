// Attention over the paged cache: what the kernels share. Lengths, offsets and pages are device data; whatever they hold, no
// address leaves the cache, the page tables or the token rows (lengths are cut to the call's maxima, offsets to the tokens,
// a page outside the cache is read as page 0).
#pragma once

#include "kvcache.h"
#include "launch.h"

namespace jamhip {

struct SeqInfo {
    int t0, nq;           // its query tokens that are computed
    int first;            // the first one's place among its own tokens
    int base, len;        // tokens of its prefix, and its own
    const int* prefix;    // page rows
    const int* own;
};

JAMHIP_DEV int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }

// the last i in [0, n] with a[i] <= v, or -1 (a has n + 1 entries in rising order)
JAMHIP_DEV int last_not_above(const int* a, int n, int v) {
    int lo = -1, hi = n + 1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= v) lo = mid;
        else hi = mid;
    }
    return lo;
}

JAMHIP_DEV int prefix_of(const Attn& g, int s) {   // the sequence's prefix group or -1
    if (g.n_prefixes <= 0) return -1;
    const int j = last_not_above(g.prefix_seqs, g.n_prefixes, s);
    return j >= g.n_prefixes ? -1 : j;
}

JAMHIP_DEV SeqInfo seq_info(const Attn& g, int s) {
    SeqInfo r;
    r.t0 = clampi(g.q_offsets[s], 0, g.n_tokens);
    const int nq = clampi(g.q_offsets[s + 1], r.t0, g.n_tokens) - r.t0;
    r.nq = min(nq, g.max_q);
    r.len = clampi(g.seq_lens[s], 0, g.seq_cap);
    r.first = r.len - nq;
    r.own = g.seq_pages + (int64_t) s * g.ld_seq_pages;
    const int j = prefix_of(g, s);
    r.base = j < 0 ? 0 : clampi(g.prefix_lens[j], 0, g.prefix_cap);
    r.prefix = j < 0 ? nullptr : g.prefix_pages + (int64_t) j * g.ld_prefix_pages;
    return r;
}

// The sequence of token t, or -1 for one that no sequence takes.
JAMHIP_DEV int seq_of(const Attn& g, int t) {
    const int s = last_not_above(g.q_offsets, g.n_seqs, t);
    return s >= g.n_seqs ? -1 : s;
}

// A batch of up to 64 sequences and 64 groups in a wave's lanes: one round of loads, where a search through the arrays is a chain
// of them (a load that misses takes 1 us, a small call's attention 4). 64 and 65 sequences of 500 tokens in Q8_0, 8 key heads of 128:
// 18.7 and 27.0 us a call, behind a shared prefix of 2000 43 and 56.
struct BatchLanes {
    int off, next, len;      // of sequence `lane`; next: the end of its query tokens
    int cut, cut_next, plen; // of group `lane`
};
JAMHIP_DEV bool fits_lanes(const Attn& g) { return g.n_seqs <= 64 && g.n_prefixes <= 64; }
JAMHIP_DEV BatchLanes batch_lanes(const Attn& g) {   // whole waves
    const int lane = threadIdx.x & 63, s = min(lane, g.n_seqs - 1);
    BatchLanes r;
    const int off = g.q_offsets[s], next = g.q_offsets[s + 1], len = g.seq_lens[s];
    r.cut = r.cut_next = r.plen = 0;
    if (g.n_prefixes > 0) {
        const int j = min(lane, g.n_prefixes - 1);
        const int cut = g.prefix_seqs[j], cut_next = g.prefix_seqs[j + 1], plen = g.prefix_lens[j];
        r.cut = clampi(cut, 0, g.n_seqs);
        r.cut_next = lane < g.n_prefixes ? clampi(cut_next, r.cut, g.n_seqs) : r.cut;
        r.plen = clampi(plen, 0, g.prefix_cap);
    }
    r.off = clampi(off, 0, g.n_tokens);
    r.next = lane < g.n_seqs ? clampi(next, r.off, g.n_tokens) : r.off;
    r.len = clampi(len, 0, g.seq_cap);
    return r;
}
JAMHIP_DEV int lane_int(int v, int l) { return __builtin_amdgcn_readlane(v, l); }
JAMHIP_DEV SeqInfo seq_info(const Attn& g, const BatchLanes& b, int s) {   // s the same in every lane
    SeqInfo r;
    r.t0 = lane_int(b.off, s);
    const int nq = lane_int(b.next, s) - r.t0;
    r.nq = min(nq, g.max_q);
    r.len = lane_int(b.len, s);
    r.first = r.len - nq;
    r.own = g.seq_pages + (int64_t) s * g.ld_seq_pages;
    const unsigned long long in = __ballot(b.cut <= s && s < b.cut_next);
    const int j = in ? __ffsll(in) - 1 : 0;
    r.base = in ? lane_int(b.plen, j) : 0;
    r.prefix = in ? g.prefix_pages + (int64_t) j * g.ld_prefix_pages : nullptr;
    return r;
}
JAMHIP_DEV int seq_of(const BatchLanes& b, int t) {   // t the same in every lane
    const unsigned long long in = __ballot(b.off <= t && t < b.next);
    return in ? __ffsll(in) - 1 : -1;
}

// Row (KvView::row) of key `at` of head `head` of a sequence's prefix and own tokens together.
JAMHIP_DEV int64_t entry_row(const KvView& c, const SeqInfo& r, int at, int head) {
    const bool shared = at < r.base;
    const int i = shared ? at : at - r.base, pg = c.page.div(i), in = i - pg * c.page.d;
    const int p = (shared ? r.prefix : r.own)[pg];
    return ((int64_t) ((uint32_t) p < (uint32_t) c.n_pages ? p : 0) * c.kv + head) * c.page.d + in;
}

constexpr int ATTN_ROW_FLOATS = 256 + 64;   // attn_row's shared memory: the query row, then a block's weights

// One output row by one wave, every masked key left out entirely: 64 keys at a time, a key a lane for the scores, 4 elements
// a lane for the values.
template <int TYPE> JAMHIP_DEV void attn_row(const Attn& g, int t, int head, float* lds) {
    const int lane = threadIdx.x & 63, dim = g.cache.dim, kvh = g.grp.div(head);
    const int s = seq_of(g, t);
    if (s < 0) return;
    const SeqInfo r = seq_info(g, s);
    if (t - r.t0 >= r.nq) return;
    const int pos = r.base + r.first + (t - r.t0);
    const int lo = g.window > 0 ? max(0, pos - g.window + 1) : 0, hi = min(r.base + r.len, pos + 1);
    float* qs = lds;
    float* ps = lds + 256;
    const float* q = g.q + t * g.ldq + (int64_t) head * dim;
    for (int d = lane; d < dim; d += 64) qs[d] = q[d] * g.scale;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    float m = -__builtin_inff(), l = 0.0f;
    float4_t acc = {0, 0, 0, 0};
    for (int k0 = lo; k0 < hi; k0 += 64) {
        const int at = k0 + lane;
        float x = -__builtin_inff();
        if (at < hi) {
            const int64_t row = entry_row(g.cache, r, at, kvh);
            x = 0.0f;
            for (int d = 0; d < dim; d += 4) {
                const float4_t k = kv_load4<TYPE>(g.cache.k, g.cache.scale_off, dim, row, d);
#pragma unroll
                for (int i = 0; i < 4; i++) x += qs[d + i] * k[i];
            }
        }
        float top = x;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
        const float now = fmaxf(m, top), ref = now == -__builtin_inff() ? 0.0f : now;
        const float keep = expf(m - ref), p = at < hi ? expf(x - ref) : 0.0f;
        l = l * keep + wave_sum(p);
        m = now;
        ps[lane] = p;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        acc *= keep;
        if (4 * lane < dim)
            for (int j = 0; j < min(64, hi - k0); j++) {
                const int64_t row = entry_row(g.cache, r, k0 + j, kvh);
                acc += kv_load4<TYPE>(g.cache.v, g.cache.scale_off, dim, row, 4 * lane) * ps[j];
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    if (g.sinks != nullptr) {
        const float x = g.sinks[head], now = fmaxf(m, x), ref = now == -__builtin_inff() ? 0.0f : now, keep = expf(m - ref);
        l = l * keep + expf(x - ref);
        acc *= keep;
    }
    if (4 * lane < dim) {
        float* o = g.out + t * g.ldo + (int64_t) head * dim + 4 * lane;
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = l == 0.0f ? 0.0f : acc[i] / l;   // a row that sees nothing is zeros
    }
}

}  // namespace jamhip
