// The attention kernel for few rows of a key head (16 or 32): decoding.
//
// The four waves of a workgroup hold the same rows and share out a run of keys, 32 at a time each, with nothing between them until
// their results are joined at the end: no barrier makes one wave's loads wait for another's. Keys go from the cache straight into
// the first product's operand: its depth may take the elements in any order that the query takes too, so a lane reads 16 bytes
// of a row and uses them over several products. Values go through the wave's own piece of shared memory for the transposing
// read. The next tile's codes are on their way while one is computed.
//
// Bound by memory while all workgroups run, then by the longest sequence: 64 sequences of 33 to 1024 keys in Q8_0, 8 key heads of
// 128, 26 us (2.9 TB/s over all, 6 at the start). With 32 rows behind 4 x 24001 tokens in Q4_0, 46 us (2.3 TB/s): the bytes take about 23
// of them, the two products 22, turning codes into f16 (7 instructions for 4) 9, and two waves a SIMD do not overlap the three. One
// sequence of 745 keys 7.2 us: launch and three rounds of dependent loads (lengths, pages, codes); a tree of 25 tokens of it 12.0. A workgroup of
// one tile with a barrier between loads and products took 28.8 and 76.9 for the first two. 32 rows of 128 in F16 keep 20 registers in scratch (trees 14).
#pragma once

#include "attn_mma.h"

namespace jamhip {

// A lane's share of a key's row, D / PARTS elements for D / (8 · PARTS) products: pieces of 32, 16 and 8 elements, each over
// all parts: [begin, begin + PARTS · piece) of the row.
template <int TYPE, int D, int NC> struct KeyLane {
    static constexpr int PARTS = 64 / NC, E = D / PARTS, STEPS = E / 8;
    static constexpr int BIG = TYPE == Q4_0 ? 32 : TYPE == Q8_0 ? 16 : 8;                 // elements of 16 bytes
    static constexpr int NB = E / BIG, R1 = E % BIG, MID = BIG / 2, NM = R1 >= MID && MID >= 8 ? 1 : 0, R2 = R1 - NM * MID;
    static constexpr int NS = R2 / 8;
    static_assert(NB * BIG + NM * MID + NS * 8 == E && NS <= (TYPE == Q4_0 && NC == 16) && (TYPE != F16 || NM == 0));
    uint4_t big[NB > 0 ? NB : 1];
    uint2_t mid;
    uint32_t sml;
    _Float16 sb[NB > 0 ? NB : 1], sm, ss;

    // the row's element of the lane's element j (0 .. 7) of product st: first of four in a row for j = 0 and j = 4
    JAMHIP_DEV static constexpr int element(int st, int part, int j) {
        const int e = 8 * st;   // of the lane's share
        if (e < NB * BIG) {
            const int p = e / BIG, in = e % BIG;
            return PARTS * BIG * p + BIG * part + in + j;
        }
        const int at = PARTS * BIG * NB;
        if (e < NB * BIG + NM * MID) {
            const int in = e - NB * BIG;
            if (TYPE == Q4_0) return at + 32 * (part / 2) + 8 * (part % 2) + 2 * in + j;   // in 0: low nibbles, 8: high, 16 on
            return at + MID * part + in + j;
        }
        const int s = at + PARTS * MID * NM;
        return s + 4 * part + (j >= 4 ? 16 + j - 4 : j);   // Q4_0 alone
    }
    JAMHIP_DEV void load(const uint8_t* buf, const KeyAt& row, int part) {
        // bytes per element times 2: F16 4, Q8_0 2, Q4_0 1
        constexpr int B2 = TYPE == F16 ? 4 : TYPE == Q8_0 ? 2 : 1;
        constexpr int at = PARTS * BIG * NB, at2 = at + PARTS * MID * NM;
        const uint8_t* r = buf + row.code;
        const uint8_t* s = buf + row.scale;
#pragma unroll
        for (int i = 0; i < NB; i++) {
            big[i] = *reinterpret_cast<const uint4_t*>(r + 16 * part + PARTS * 16 * i);
            if constexpr (TYPE != F16) sb[i] = *reinterpret_cast<const _Float16*>(s + BIG * part / 32 * 2 + PARTS * BIG * i / 32 * 2);
        }
        if constexpr (NM > 0) {
            mid = *reinterpret_cast<const uint2_t*>(r + 8 * part + at * B2 / 2);
            sm = *reinterpret_cast<const _Float16*>(s + MID * part / 32 * 2 + at / 32 * 2);
        }
        if constexpr (NS > 0) {
            sml = *reinterpret_cast<const uint32_t*>(r + 4 * part + at2 / 2);
            ss = *reinterpret_cast<const _Float16*>(s + at2 / 32 * 2);
        }
    }
    template <int ST> JAMHIP_DEV half8_t step() const {
        constexpr int e = 8 * ST;
        if constexpr (TYPE == F16) {
            return __builtin_bit_cast(half8_t, big[ST]);
        } else {
            half2_t h[4];
            if constexpr (e < NB * BIG) {
                constexpr int p = e / BIG, in = e % BIG;
                const half2_t scale = {sb[p], sb[p]};
                if constexpr (TYPE == Q8_0) {
                    q8_word(big[p][in / 4], scale, h), q8_word(big[p][in / 4 + 1], scale, h + 2);
                } else {   // elements 0 .. 15 low nibbles of bytes 0 .. 15, 16 .. 31 high
                    constexpr int w = in % 16 / 4;
                    q4_word(in < 16 ? big[p][w] : big[p][w] >> 4, scale, h), q4_word(in < 16 ? big[p][w + 1] : big[p][w + 1] >> 4, scale, h + 2);
                }
            } else if constexpr (e < NB * BIG + NM * MID) {
                constexpr int in = e - NB * BIG;
                const half2_t scale = {sm, sm};
                if constexpr (TYPE == Q8_0) {
                    q8_word(mid[0], scale, h), q8_word(mid[1], scale, h + 2);
                } else {
                    q4_word(in ? mid[0] >> 4 : mid[0], scale, h), q4_word(in ? mid[1] >> 4 : mid[1], scale, h + 2);
                }
            } else {
                const half2_t scale = {ss, ss};
                q4_word(sml, scale, h), q4_word(sml >> 4, scale, h + 2);
            }
            half8_t v;
#pragma unroll
            for (int i = 0; i < 4; i++) v[2 * i] = h[i][0], v[2 * i + 1] = h[i][1];
            return v;
        }
    }
};

template <int TYPE, int D, int NC> struct Wave {
    static constexpr int KEYS = 32, ROWS = NC;
    static constexpr int CHUNKS = (D / 8 + 7) / 8 * 8, STRIDE = CHUNKS * 16;
    static constexpr int EPU = unit_elems<TYPE>(), UPK = D / EPU, UNITS = KEYS * UPK, PER = (UNITS + 63) / 64;
    using M = Mma<NC>;
    using K = KeyLane<TYPE, D, NC>;
    static constexpr int ST = KEYS / NC, DT = D / NC, STEPS = K::STEPS;
    static constexpr int JD = NC == 16 ? DT : (DT + 1) / 2;              // element tiles that are joined at once
    static constexpr int JOIN = 4 * (JD * NC * NC + 2 * NC) * 4;         // bytes of the waves' results
    static constexpr int PLANE = KEYS * STRIDE, LDS = 4 * PLANE > JOIN ? 4 * PLANE : JOIN;
};

// waves a SIMD that the registers are to leave room for
constexpr int wave_occupancy(int dim, int nc) { return dim >= 192 ? 1 : nc == 16 && dim == 64 ? 3 : 2; }

template <int TYPE, int D, int NC, bool TREE> __global__ void __launch_bounds__(256, (wave_occupancy(D, NC))) attn_wave_kernel(AttnArgs a) {
    using T = Wave<TYPE, D, NC>;
    using M = typename T::M;
    using acc_t = typename M::acc_t;
    __shared__ __align__(16) uint8_t lds[T::LDS];
    __shared__ __align__(16) KeyAt rows[4][2][T::KEYS];
    __shared__ float redo[4][ATTN_ROW_FLOATS];
    const Attn& g = a.g;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane % NC, part = lane / NC;
    int b = a.block0 + blockIdx.x;
    const int kvh = b % g.cache.kv;
    b /= g.cache.kv;
    // a prefix's tiles past the last are the last workgroups; a sequence's run of keys past its end is
    const bool rows_last = a.part.mode == 1;
    const int tile = rows_last ? b / a.part.splits : b % a.part.tiles, split = rows_last ? b % a.part.splits : b / a.part.tiles;
    RowSet w;
    if (!attn_row_set<T::ROWS>(a, tile, &w)) return;
    const Column c = attn_column<TREE>(a, w, w.r0 + col, kvh, split);
    const int lo = c.lo, hi = c.hi + 1;   // the same in every wave

    half8_t qh[T::STEPS], ql[T::STEPS];
    const float f = load_query<NC>(g.q + (int64_t) c.seen.tok * g.ldq + (int64_t) c.seen.head * D, g.scale, qh, ql,
                                   [&](int st, int j) { return T::K::element(st, part, j); });

    acc_t o[T::DT];
#pragma unroll
    for (int i = 0; i < T::DT; i++)
#pragma unroll
        for (int k = 0; k < M::N; k++) o[i][k] = 0.0f;
    float m = -__builtin_inff(), l = 0.0f;

    KeyAt (*const rw)[T::KEYS] = rows[wave];
    uint8_t* const lv = lds + wave * T::PLANE;
    typename T::K kf[T::ST];
    uint4_t vr[T::PER];
    _Float16 vs[T::PER] = {};
    // past the last key it stands for that one: no load is behind a branch, and nothing that no row sees comes in
    auto entry_of = [&](int at) { return entry_at(g.cache, w.s, min(at, hi - 1)); };
    auto row_of = [&](int at) { return key_at<TYPE, D>(g.cache, entry_of(at), kvh); };
    auto sync = [] { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); __builtin_amdgcn_wave_barrier(); };
    auto fetch_k = [&](const KeyAt* r) {
#pragma unroll
        for (int i = 0; i < T::ST; i++) kf[i].load(g.cache.k, r[i * NC + col], part);
    };
    auto fetch_v = [&](const KeyAt* r) {
#pragma unroll
        for (int i = 0; i < T::PER; i++) {
            const int u = lane + 64 * i, key = u / T::UPK, ch = u % T::UPK;
            const KeyAt row = r[T::UNITS % 64 == 0 ? key : min(key, T::KEYS - 1)];
            vr[i] = *reinterpret_cast<const uint4_t*>(g.cache.v + row.code + ch * 16);
            if constexpr (TYPE != F16) vs[i] = *reinterpret_cast<const _Float16*>(g.cache.v + row.scale + ch * T::EPU / 32 * 2);
        }
    };
    const int first = lo < hi ? lo + T::KEYS * wave : hi, step = 4 * T::KEYS;
    if (first < hi) {
        if (lane < T::KEYS) rw[0][lane] = row_of(first + lane), rw[1][lane] = row_of(first + step + lane);
        sync();
        fetch_k(rw[0]);
        fetch_v(rw[0]);
    }
    int buf = 1;
    for (int k0 = first; k0 < hi; k0 += step, buf ^= 1) {
#pragma unroll
        for (int i = 0; i < T::PER; i++) {
            const int u = lane + 64 * i;
            if (T::UNITS % 64 == 0 || u < T::UNITS) put_unit<TYPE>(lv, vr[i], vs[i], unit_at<TYPE, T::STRIDE>(u / T::UPK, u % T::UPK));
        }
        const bool more = k0 + step < hi;
        // the page of the next but one's keys is asked for first and looked at last: loads come back in their order
        EntryAt after = {};
        if (lane < T::KEYS && k0 + 2 * step < hi) after = entry_of(k0 + 2 * step + lane);
        if (more) fetch_v(rw[buf]);
        acc_t sc[T::ST];
#pragma unroll
        for (int i = 0; i < T::ST; i++)
#pragma unroll
            for (int k = 0; k < M::N; k++) sc[i][k] = 0.0f;
        unroll<0, T::STEPS>([&](auto st) {
            half8_t x[T::ST];
#pragma unroll
            for (int i = 0; i < T::ST; i++) x[i] = kf[i].template step<decltype(st)::value>();
#pragma unroll
            for (int i = 0; i < T::ST; i++) sc[i] = M::mma(x[i], qh[decltype(st)::value], sc[i]);
#pragma unroll
            for (int i = 0; i < T::ST; i++) sc[i] = M::mma(x[i], ql[decltype(st)::value], sc[i]);
        });
        if (more) fetch_k(rw[buf]);
        attn_weights<M, T::ST, T::DT, NC, TREE>(sc, o, m, l, f, c, c.seen, a.g, k0, part);
        sync();   // the values are in shared memory
#pragma unroll
        for (int u = 0; u < T::KEYS / M::DEPTH; u++) {
            half8_t ph, pl;
            weight_halves<NC>(sc, u, ph, pl);
            add_values<NC, T::DT, T::STRIDE, M>(o, lv, u, ph, pl);
        }
        // only where the walk gets there: 512 sequences of up to 500 keys, heads of 64 in Q4_0, 33.8 us, with it for every tile 34.3
        if (lane < T::KEYS && k0 + 2 * step < hi) rw[buf ^ 1][lane] = key_at<TYPE, D>(g.cache, after, kvh);
        sync();   // and read, before the next tile's take their place
    }

    // ---- the waves' results, through shared memory: each sums every fourth element tile
    l = column_sum<NC>(l);
    float* const po = reinterpret_cast<float*>(lds);                      // [wave][element][column]
    float* const pm = po + 4 * T::JD * NC * NC;                           // [wave][column], then the sums
    float wt[4];
#pragma unroll
    for (int d0 = 0; d0 < T::DT; d0 += T::JD) {
        __syncthreads();
#pragma unroll
        for (int dt = d0; dt < T::DT && dt < d0 + T::JD; dt++)
#pragma unroll
            for (int k = 0; k < M::N; k++) po[((wave * T::JD + dt - d0) * NC + M::row(k, part)) * NC + col] = o[dt][k];
        if (d0 == 0 && part == 0) pm[wave * NC + col] = m, pm[(4 + wave) * NC + col] = l;
        __syncthreads();
        if (d0 == 0) {
            m = fmaxf(fmaxf(pm[col], pm[NC + col]), fmaxf(pm[2 * NC + col], pm[3 * NC + col]));
            l = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                wt[i] = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(pm[i * NC + col] - m);
                l += pm[(4 + i) * NC + col] * wt[i];
            }
        }
#pragma unroll
        for (int dt = d0; dt < T::DT && dt < d0 + T::JD; dt++)
            if (dt % 4 == wave)
#pragma unroll
                for (int k = 0; k < M::N; k++) {
                    float v = 0.0f;
#pragma unroll
                    for (int i = 0; i < 4; i++) v += wt[i] * po[((i * T::JD + dt - d0) * NC + M::row(k, part)) * NC + col];
                    o[dt][k] = v;
                }
    }
    unsigned long long again = attn_emit<D, NC, T::DT, 4, M>(a, c, o, m, l, split, wave);
    if (!a.part.direct) return;
    __syncthreads();   // a row that one wave finds not finite is whole before it is written again
    for (; again; again &= again - 1) {
        const int k = __ffsll(again) - 1;
        attn_row<TYPE, TREE>(g, __builtin_amdgcn_readlane(c.seen.tok, k), __builtin_amdgcn_readlane(c.seen.head, k), redo[wave]);
    }
}

}  // namespace jamhip
