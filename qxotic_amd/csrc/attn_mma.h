// What the attention kernels on the matrix cores share.
//
// Both compute, for columns of 16 or 32 query rows a wave,
//   Sᵀ = K · Qᵀ            a column of scores per lane: the softmax's maximum and sum need one exchange at their end
//   Oᵀ = Vᵀ · Pᵀ           the scores' registers are the second operand's as they stand: its slots take the keys in the order in
//                          which the first product leaves them, and Vᵀ comes out of row-major shared memory in that order
//                          through the transposing read
// What a code stands for is an f16, so keys and values lose nothing. Queries and weights are f32 values carried as two f16, hi + lo,
// both cut toward zero (22 bits, 2^-21 of the value at most), a product each. An f16 ends at 2^-24, so both are scaled to near its other
// end: the query row by a power of two to a largest element in [2^14, 2^15), of which elements down to 2^-17 keep their 22 bits and
// smaller ones are off by at most 2^-38; weights are 2^(s - m + 13), which keep them down to 2^-16 of the running maximum m's and
// are off by at most 2^-37 of it below. m moves only when a score passes it by 2.75 (in powers of two; weights then stay below 2^15.75),
// so most tiles rescale nothing: against 2^(s - m + 7) and a lag of 8, 64 sequences behind 8192 tokens in Q8_0 take 71.6 us for
// 70.5, prompts the same. Sums are f32; the matrix cores round each product at about 2^-27 of the sum that it joins.
#pragma once

#include "attn.h"
#include "attn_plan.h"

namespace jamhip {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short short4_t __attribute__((ext_vector_type(4)));

struct AttnArgs {
    Attn g;
    AttnPart part;
    float* acc;    // [slot][token · heads + head][dim], unscaled
    float2* ml;    // [slot][token · heads + head]: maximum (powers of two), sum (times 2^WEIGHT_EXP)
    int block0;    // workgroups of the launches before
};

// All `blocks` workgroups in runs of ATTN_RUN.
template <typename F> hipError_t attn_runs(AttnArgs a, int64_t blocks, F&& launch) {
    hipError_t e = hipSuccess;
    for (int64_t b = 0; b < blocks && e == hipSuccess; b += ATTN_RUN) {
        a.block0 = (int) b;
        e = launch(a, (uint32_t) (blocks - b < ATTN_RUN ? blocks - b : ATTN_RUN));
    }
    return e;
}

constexpr float WEIGHT_EXP = 13.0f, LAZY = 2.75f, LOG2E = 1.44269504088896340736f;

template <int TYPE> constexpr int unit_elems() { return TYPE == F16 ? 8 : TYPE == Q8_0 ? 16 : 32; }   // of 16 bytes of codes

JAMHIP_DEV half8_t join_half(half4_t a, half4_t b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// Two f32 as a pair of f16 rounded toward zero (one instruction), and what that leaves of them.
JAMHIP_DEV half2_t pack_rtz(float a, float b) { return __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_pkrtz(a, b)); }

template <int NC> struct Mma;
template <> struct Mma<32> {
    typedef floatx16 acc_t;
    static constexpr int N = 16, DEPTH = 16;   // accumulators a lane, product depth
    JAMHIP_DEV static acc_t mma(half8_t a, half8_t b, acc_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    JAMHIP_DEV static int row(int i, int part) { return 8 * (i / 4) + 4 * part + i % 4; }   // of accumulator i in lane part
};
template <> struct Mma<16> {
    typedef floatx4 acc_t;
    static constexpr int N = 4, DEPTH = 32;
    JAMHIP_DEV static acc_t mma(half8_t a, half8_t b, acc_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    JAMHIP_DEV static int row(int i, int part) { return 4 * part + i; }
};

// Maximum and sum over the lanes that hold one column (64 / NC of them, NC apart).
template <int NC> JAMHIP_DEV float column_max(float v) {
    if constexpr (NC == 16) v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
template <int NC> JAMHIP_DEV float column_sum(float v) {
    if constexpr (NC == 16) v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}
template <int CTRL> JAMHIP_DEV int dpp_int(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, true); }
JAMHIP_DEV int wave_min(int v) {   // a butterfly within rows of 16, then the rows (as wave_sum)
    v = min(v, dpp_int<0xB1>(v));
    v = min(v, dpp_int<0x4E>(v));
    v = min(v, dpp_int<0x141>(v));
    v = min(v, dpp_int<0x140>(v));
    return min(min(lane_int(v, 0), lane_int(v, 16)), min(lane_int(v, 32), lane_int(v, 48)));
}
JAMHIP_DEV int wave_max(int v) { return -wave_min(-v); }

// Byte offset of 16-byte chunk c of a key's row. The key's low bits are spread over the chunk's: eight neighbouring keys' equal
// chunks (the first product's read) fall into eight different 16-byte columns, and so do four neighbouring keys' pairs of
// chunks (the transposing read).
template <int STRIDE> JAMHIP_DEV int lds_at(int key, int c) {
    return key * STRIDE + ((c ^ ((key & 3) * 2 + ((key >> 2) & 1))) << 4);
}

// A lane's 8 elements of the query row for each of STEPS products, element `at(step)` and 4 on, then `at4(step)` and 4 on: hi and
// lo halves of the row scaled by a power of two. Returns f: a score in powers of two is f times the product.
template <int NC, int STEPS, typename AT> JAMHIP_DEV float load_query(const float* q, float scale, half8_t (&qh)[STEPS], half8_t (&ql)[STEPS], AT&& at) {
    float top = 0.0f;
    float x[STEPS][8];
    const bool al = (reinterpret_cast<uintptr_t>(q) & 15) == 0;
#pragma unroll
    for (int st = 0; st < STEPS; st++) {
        const float *p = q + at(st, 0), *r = q + at(st, 4);
        if (al) {
            const float4_t u = *reinterpret_cast<const float4_t*>(p), v = *reinterpret_cast<const float4_t*>(r);
#pragma unroll
            for (int i = 0; i < 4; i++) x[st][i] = u[i], x[st][4 + i] = v[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) x[st][i] = p[i], x[st][4 + i] = r[i];
        }
#pragma unroll
        for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(x[st][i]));
    }
    top = column_max<NC>(top);
    const int e = max((top > 0.0f && top < __builtin_inff() ? ilogbf(top) : 0) - 14, -126);
    const float unit = ldexpf(1.0f, -e);
#pragma unroll
    for (int st = 0; st < STEPS; st++)
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float y = x[st][i] * unit, z = x[st][i + 1] * unit;
            const half2_t h = pack_rtz(y, z), r = pack_rtz(y - (float) h[0], z - (float) h[1]);
            qh[st][i] = h[0], qh[st][i + 1] = h[1], ql[st][i] = r[0], ql[st][i + 1] = r[1];
        }
    return ldexpf(scale * LOG2E, e);
}

// ---- the workgroup's rows
struct RowSet {
    SeqInfo s;         // the keys' tables (mode 1: the group's prefix alone)
    int r0, n_rows;    // its first row, rows of the set
    int t_first;       // the set's first token
    BatchLanes lanes;  // where the batch fits
};

// The rows of tile `tile` of ROWS each, false for none. Every lane takes part.
template <int ROWS> JAMHIP_DEV bool attn_row_set(const AttnArgs& a, int tile, RowSet* w) {
    const Attn& g = a.g;
    const int lane = threadIdx.x & 63;
    w->s = SeqInfo{};
    const bool small = fits_lanes(g);
    if (small) w->lanes = batch_lanes(g);
    if (a.part.mode == 1 && small) {
        const BatchLanes& b = w->lanes;
        // tokens of the group's sequences: from the first one's on
        const int t0 = __shfl(b.off, min(b.cut, g.n_seqs - 1)), t1 = __shfl(b.next, max(b.cut_next, 1) - 1);
        const int rows = b.cut < b.cut_next ? max(t1 - t0, 0) * g.grp.d : 0, tiles = (rows + ROWS - 1) / ROWS;
        const int before = wave_exclusive_scan(tiles);
        const unsigned long long hit = __ballot(tile >= before && tile < before + tiles);
        if (!hit) return false;
        const int j = __ffsll(hit) - 1;
        w->r0 = (tile - lane_int(before, j)) * ROWS;
        w->t_first = lane_int(t0, j);
        w->n_rows = lane_int(rows, j);
        w->s.base = lane_int(b.plen, j);
        w->s.prefix = g.prefix_pages + (int64_t) j * g.ld_prefix_pages;
    } else if (a.part.mode == 1) {
        int j = -1, rt = 0, from = 0;   // from: tiles of the groups before
        for (int j0 = 0; j0 < g.n_prefixes && j < 0; j0 += 64) {
            const int jj = min(j0 + lane, g.n_prefixes - 1);
            const int s0 = clampi(g.prefix_seqs[jj], 0, g.n_seqs), s1 = clampi(g.prefix_seqs[jj + 1], s0, g.n_seqs);
            const int t0 = clampi(g.q_offsets[s0], 0, g.n_tokens), t1 = clampi(g.q_offsets[s1], t0, g.n_tokens);
            const int tiles = j0 + lane < g.n_prefixes ? ((t1 - t0) * g.grp.d + ROWS - 1) / ROWS : 0;
            const int before = from + wave_exclusive_scan(tiles);
            const unsigned long long hit = __ballot(tile >= before && tile < before + tiles);
            if (hit) {
                const int l = __ffsll(hit) - 1;
                j = j0 + l;
                rt = tile - __builtin_amdgcn_readlane(before, l);
                w->t_first = __builtin_amdgcn_readlane(t0, l);
                w->n_rows = (__builtin_amdgcn_readlane(t1, l) - w->t_first) * g.grp.d;
            }
            from = __builtin_amdgcn_readlane(before + tiles, 63);
        }
        if (j < 0) return false;
        w->r0 = rt * ROWS;
        w->s.base = clampi(g.prefix_lens[j], 0, g.prefix_cap);
        w->s.prefix = g.prefix_pages + (int64_t) j * g.ld_prefix_pages;
    } else {
        const int per = (g.max_q * g.grp.d + ROWS - 1) / ROWS, q = tile / per;
        w->s = small ? seq_info(g, w->lanes, q) : seq_info(g, q);
        w->t_first = w->s.t0;
        w->n_rows = w->s.nq * g.grp.d;
        w->r0 = (tile - q * per) * ROWS;
        if (a.part.mode == 2) w->s.base = 0;   // positions among its own keys
    }
    return w->r0 < w->n_rows;
}

// ---- a lane's column: a row and the keys that it sees, those of the workgroup's run of chunk keys
struct Column {
    int tok, head;
    bool live;
    int see_lo, see_n;     // key sees: (unsigned) (key - see_lo) <= see_n
    int lo, hi;            // the wave's first and last key that a row sees
    int all_lo, all_hi;    // between these every live row sees all
};

JAMHIP_DEV Column attn_column(const AttnArgs& a, const RowSet& w, int r, int kvh, int split) {
    const Attn& g = a.g;
    Column c;
    const int rr = min(r, w.n_rows - 1), total = w.s.base + w.s.len;
    c.tok = w.t_first + g.grp.div(rr);
    c.head = kvh * g.grp.d + (rr - (c.tok - w.t_first) * g.grp.d);
    c.live = r < w.n_rows;
    int pos = w.s.base + w.s.first + (c.tok - w.s.t0);
    if (a.part.mode == 1) {
        if (fits_lanes(g)) {   // the sequences of the wave's tokens, one after another
            const BatchLanes& b = w.lanes;
            int at = 0, t0 = 0, nq = -1;   // at: SeqInfo::first
            const int t0_wave = wave_min(c.tok), t1_wave = wave_max(c.tok);
            unsigned long long on = __ballot(b.off < b.next && b.next > t0_wave && b.off <= t1_wave);
            for (; on; on &= on - 1) {
                const int q = __ffsll(on) - 1, first = lane_int(b.off, q), end = lane_int(b.next, q);
                if (c.tok >= first && c.tok < end) t0 = first, nq = min(end - first, g.max_q), at = lane_int(b.len, q) - (end - first);
            }
            c.live = c.live && c.tok - t0 < nq;
            pos = w.s.base + at + (c.tok - t0);
        } else {
            const int q = seq_of(g, c.tok);
            const SeqInfo mine = seq_info(g, max(q, 0));
            c.live = c.live && q >= 0 && c.tok - mine.t0 < mine.nq;
            pos = mine.base + mine.first + (c.tok - mine.t0);
        }
    }
    const int c0 = split * a.part.chunk;
    const int k_lo = max(c0, g.window > 0 ? pos - g.window + 1 : 0), k_hi = min(min(total, c0 + a.part.chunk) - 1, pos);   // first and last
    const bool some = c.live && k_lo <= k_hi;
    c.see_lo = some ? k_lo : INT32_MAX, c.see_n = some ? k_hi - k_lo : 0;
    c.lo = wave_min(some ? k_lo : INT32_MAX), c.hi = wave_max(some ? k_hi : -1);
    c.all_lo = wave_max(c.live ? (some ? k_lo : INT32_MAX) : -1), c.all_hi = wave_min(c.live ? (some ? k_hi : -1) : INT32_MAX);
    return c;
}

// ---- the softmax's step: a tile's scores sc (of ST products' accumulators) become weights; o and l follow the maximum
template <typename M, int ST, int DT, int NC, typename ACC>
JAMHIP_DEV void attn_weights(ACC (&sc)[ST], ACC (&o)[DT], float& m, float& l, float f, const Column& c, int kw, int part) {
    if (kw < c.all_lo || kw + ST * NC - 1 > c.all_hi) {
#pragma unroll
        for (int i = 0; i < ST; i++)
#pragma unroll
            for (int k = 0; k < M::N; k++)
                if ((unsigned) (kw + i * NC + M::row(k, part) - c.see_lo) > (unsigned) c.see_n) sc[i][k] = -__builtin_inff();
    }
    float top = sc[0][0];
#pragma unroll
    for (int i = 0; i < ST; i++)
#pragma unroll
        for (int k = 0; k < M::N; k++) top = fmaxf(top, sc[i][k]);
    top = column_max<NC>(top) * f;
    if (__any(top > m + LAZY)) {
        const float now = fmaxf(m, top), keep = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - now);
        m = now;
        l *= keep;
#pragma unroll
        for (int i = 0; i < DT; i++)
#pragma unroll
            for (int k = 0; k < M::N; k++) o[i][k] *= keep;
    }
    const float shift = WEIGHT_EXP - (m == -__builtin_inff() ? 0.0f : m);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < ST; i++)
#pragma unroll
        for (int k = 0; k < M::N; k++) {
            sc[i][k] = __builtin_amdgcn_exp2f(fmaf(sc[i][k], f, shift));
            sum += sc[i][k];
        }
    l += sum;
}

// The weights of product u (16 or 32 keys) as its second operand, hi and lo halves: 8 a lane, in the order in which the scores'
// accumulators hold them (two of a 32-row tile's four groups, or two 16-row tiles).
template <int NC, int ST, typename ACC> JAMHIP_DEV void weight_halves(const ACC (&sc)[ST], int u, half8_t& ph, half8_t& pl) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const float x = NC == 32 ? sc[u / 2][8 * (u % 2) + e] : sc[2 * u + e / 4][e % 4];
        const float y = NC == 32 ? sc[u / 2][8 * (u % 2) + e + 1] : sc[2 * u + e / 4][e % 4 + 1];
        const half2_t h = pack_rtz(x, y), r = pack_rtz(fmaf((float) h[0], -1.0f, x), fmaf((float) h[1], -1.0f, y));   // exact; one instruction each
        ph[e] = h[0], ph[e + 1] = h[1], pl[e] = r[0], pl[e + 1] = r[1];
    }
}

// O += Vᵀ · P for product u, the values at `lv` in rows of STRIDE bytes from key kb on: 16 lanes read 4 keys of 16 elements and get
// 4 keys of their element, twice, which is the keys' order in the weights.
template <int NC, int DT, int STRIDE, typename M, typename ACC>
JAMHIP_DEV void add_values(ACC (&o)[DT], const uint8_t* lv, int kb, int u, half8_t ph, half8_t pl) {
    const int lane = threadIdx.x & 63, part = lane / NC, in = lane % 16, sub = NC == 32 ? (lane / 16) % 2 : 0;
    const int key = kb + u * M::DEPTH + 4 * part + in / 4;
    constexpr int PAIR = NC == 32 ? 2 : 1;   // two products between hi and lo of one sum, where there are registers for them
#pragma unroll
    for (int d0 = 0; d0 < DT; d0 += PAIR) {
        half8_t v[PAIR];
#pragma unroll
        for (int i = 0; i < PAIR && d0 + i < DT; i++) {
            const int e0 = (d0 + i) * NC + sub * 16 + 4 * (in % 4);
            auto at = [&](int k) {
                const uint8_t* p = lv + lds_at<STRIDE>(k, e0 / 8) + e0 % 8 * 2;
                const short4_t w = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) short4_t*) (uintptr_t) (__attribute__((address_space(3))) const uint8_t*) p);
                return __builtin_bit_cast(half4_t, w);
            };
            v[i] = join_half(at(key), at(key + M::DEPTH / 2));
        }
#pragma unroll
        for (int i = 0; i < PAIR && d0 + i < DT; i++) o[d0 + i] = M::mma(v[i], ph, o[d0 + i]);
#pragma unroll
        for (int i = 0; i < PAIR && d0 + i < DT; i++) o[d0 + i] = M::mma(v[i], pl, o[d0 + i]);
    }
}

// ---- where a key's codes and scales are: byte offsets into the cache's buffers, made once for a key and read by every lane that
// loads a piece of it
struct KeyAt {
    int64_t code, scale;
};
template <int TYPE, int D> JAMHIP_DEV KeyAt key_at(const KvView& c, const SeqInfo& s, int at, int head) {
    const int64_t row = entry_row(c, s, at, head);
    return {row * kv_row_bytes(TYPE, D), c.scale_off + row * (D / 32) * 2};
}

// ---- 16 bytes of codes of a row into shared memory as f16
template <int TYPE, int STRIDE> JAMHIP_DEV void put_unit(uint8_t* plane, const uint4_t& w, _Float16 sc, int key, int c) {
    if constexpr (TYPE == F16) {
        *reinterpret_cast<uint4_t*>(plane + lds_at<STRIDE>(key, c)) = w;
    } else {
        const half2_t scale = {sc, sc};
        half2_t h[16];
        if constexpr (TYPE == Q8_0) {
#pragma unroll
            for (int i = 0; i < 4; i++) q8_word(w[i], scale, h + 2 * i);
        } else {   // byte j: element j low, element 16 + j high
#pragma unroll
            for (int i = 0; i < 4; i++) q4_word(w[i], scale, h + 2 * i), q4_word(w[i] >> 4, scale, h + 8 + 2 * i);
        }
        constexpr int N = unit_elems<TYPE>() / 8;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint4_t v = {as_u32(h[4 * i]), as_u32(h[4 * i + 1]), as_u32(h[4 * i + 2]), as_u32(h[4 * i + 3])};
            *reinterpret_cast<uint4_t*>(plane + lds_at<STRIDE>(key, c * N + i)) = v;
        }
    }
}

// ---- the wave's columns to the output (direct) or to the workspace, by the lanes that hold them, the element tiles `turn`,
// turn + TURNS, ...; returns the columns (a bit each) whose rows have to be computed again. A row that is not finite may owe it
// to an entry that it does not see (0 times what a masked value holds).
template <int D, int NC, int DT, int TURNS, typename M, typename ACC>
JAMHIP_DEV unsigned long long attn_emit(const AttnArgs& a, const Column& c, const ACC (&o)[DT], float m, float l, int split, int turn) {
    const Attn& g = a.g;
    const int part = (threadIdx.x & 63) / NC;
    float scale = 1.0f;
    float* dst;
    if (a.part.direct) {
        if (g.sinks != nullptr) {
            const float x = g.sinks[c.head] * LOG2E, now = fmaxf(m, x);
            const float keep = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - now);
            l = l * keep + (now == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(x - now + WEIGHT_EXP));
            scale = keep;
        }
        scale = l == 0.0f ? 0.0f : scale / l;
        dst = g.out + (int64_t) c.tok * g.ldo + (int64_t) c.head * D;
    } else {
        const int64_t n = (int64_t) g.n_tokens * g.heads, at = (int64_t) (a.part.slot0 + split) * n + (int64_t) c.tok * g.heads + c.head;
        dst = a.acc + at * D;
        if (c.live && part == 0 && turn == 0) a.ml[at] = make_float2(m, l);
    }
    const bool al = (reinterpret_cast<uintptr_t>(dst) & 15) == 0;
    bool bad = false;
#pragma unroll
    for (int dt = 0; dt < DT; dt++) {
        if (dt % TURNS != turn) continue;
#pragma unroll
        for (int k = 0; k < M::N; k += 4) {
            float4_t v;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v[e] = o[dt][k + e] * scale;
                bad |= !(fabsf(v[e]) < __builtin_inff());
            }
            float* p = dst + dt * NC + M::row(k, part);
            if (c.live) {
                if (al) {
                    *reinterpret_cast<float4_t*>(p) = v;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) p[e] = v[e];
                }
            }
        }
    }
    unsigned long long again = a.part.direct ? __ballot(bad && c.live) : 0;
#pragma unroll
    for (int k = NC; k < 64; k <<= 1) again |= again >> k;
    return again & ((1ull << NC) - 1);
}

}  // namespace jamhip
