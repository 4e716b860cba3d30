// The attention kernel for many rows of a key head.
//
// A workgroup of four waves holds 128 query rows (rows of one key head: its tokens times the query heads that share it), 32 a
// wave, and walks a run of keys, a tile of keys and values at a time: codes come from the cache into registers while the tile
// before is computed, are turned into f16 and laid out in shared memory once for all rows.
//
// Bound by the matrix cores, the VALU and the power that both take. Products of 32 x 32 x 16 alone, of ordinary values, run at 1.62 PFLOP/s on this
// card: the clock falls to 1.6 GHz (of zeros 2.45 PFLOP/s). At head_dim 128 a tile costs a wave 2048 cycles of products (two for each, for the
// halves), and VALU beside them (turning codes into f16, an exponential, a fused multiply-add, a sum, a maximum, two conversions and a
// difference for each of 32 scores a lane). Two workgroups of a CU get through a tile every 3350 cycles between them (Q4_0, at 2.1 GHz; 61 % products where
// all 128 rows are there), one alone takes 5100. Over whole launches of trees the products take 30 to 40 % of the cycles, 41 to 48 % of those in which a
// CU has work: 5 to 8 us pass before the first tile, waves whose rows a tree does not fill rest, CUs have unequal numbers of tiles, and of two
// workgroups on a CU one ends first and leaves the other alone. 64 sequences of 4
// heads behind 8192 tokens in Q8_0, 8 key heads of 128: 30 us; 8 prompts of up to 256 tokens behind 4096 in F16, heads of 64: 285 us (446
// TFLOP/s, counted once) after some fifty calls in a row, more before, while the clock rises; trees of up to 32 tokens of 64 sequences
// of 200 to 4096 tokens in Q8_0 188 to 195, of 63 of four of 20011 to 32771 in Q4_0 229 to 237 (458 to 443).
//
// What made it faster (calls of the trees' 64 sequences and long ones): loads that wait for themselves alone, limits and bounds out of the
// vector registers, operands a product ahead and a wave's priority in its products, together 236 -> 205 and 276 -> 257. No register goes to
// scratch. What did not: conversion beside the products, with two halves of shared memory and one barrier a tile, 202 -> 212 and 246 -> 251;
// equal shares of all keys, cut by the device's lengths and joined, 202 -> 207 (179 and a join of 26) and 257 -> 257; two, three and four
// times the runs of keys 196 -> 229, 218, 224 and 246 -> 260, 271, 269.
#pragma once

#include "attn_mma.h"

namespace jamhip {

template <int TYPE, int D> struct Tile {
    static constexpr int NC = 32, ROWS = attn_rows(2), KEYS = attn_keys(2, D);
    static constexpr int CHUNKS = (D / 8 + 7) / 8 * 8, STRIDE = CHUNKS * 16;   // of a key's row in shared memory
    static constexpr int PLANE = KEYS * STRIDE;
    static constexpr int EPU = unit_elems<TYPE>(), UPK = D / EPU, UNITS = KEYS * UPK, PER = (UNITS + 255) / 256;
    using M = Mma<NC>;
    static constexpr int STEPS = D / M::DEPTH, ST = KEYS / NC, DT = D / NC;
};

template <int TYPE, int D, bool TREE> __global__ void __launch_bounds__(256, D <= 128 ? 2 : 1) attn_tile_kernel(AttnArgs a) {
    using T = Tile<TYPE, D>;
    using M = typename T::M;
    using acc_t = typename M::acc_t;
    constexpr int NC = T::NC, KEYS = T::KEYS;
    __shared__ __align__(16) uint8_t lds[2 * T::PLANE];
    __shared__ __align__(16) KeyAt rows[2][KEYS];
    __shared__ int range[2][4];
    __shared__ Seen seen[4][NC];   // looked at for tiles that some row does not see whole: not kept in registers
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
    Column c = attn_column<TREE>(a, w, w.r0 + wave * NC + col, kvh, split);
    seen[wave][col] = c.seen;   // both parts of a column the same
    if (lane == 0) range[0][wave] = c.lo, range[1][wave] = c.hi;
    half8_t qh[T::STEPS], ql[T::STEPS];
    const float f = load_query<NC>(g.q + (int64_t) c.seen.tok * g.ldq + (int64_t) c.seen.head * D, g.scale, qh, ql,
                                   [&](int st, int j) { return st * M::DEPTH + part * 8 + j; });
    __syncthreads();
    const int lo = uniform(min(min(range[0][0], range[0][1]), min(range[0][2], range[0][3])));
    const int hi = uniform(max(max(range[1][0], range[1][1]), max(range[1][2], range[1][3]))) + 1;   // one past the last

    acc_t o[T::DT];
#pragma unroll
    for (int i = 0; i < T::DT; i++)
#pragma unroll
        for (int k = 0; k < M::N; k++) o[i][k] = 0.0f;
    float m = -__builtin_inff(), l = 0.0f;

    uint4_t kr[T::PER], vr[T::PER];
    _Float16 ks[T::PER] = {}, vs[T::PER] = {};
    // past the last key it stands for that one: no load is behind a branch, and nothing that no row sees comes in
    auto entry_of = [&](int at) { return entry_at(g.cache, w.s, min(at, hi - 1)); };
    auto row_of = [&](int at) { return key_at<TYPE, D>(g.cache, entry_of(at), kvh); };
    // unit i of a thread: where the units of 256 threads are whole rows, 8 or a multiple apart, its place follows from the first one's
    constexpr bool EVEN = 256 % T::UPK == 0 && 256 / T::UPK % 8 == 0;
    auto key_of = [&](int i) { return EVEN ? tid / T::UPK + i * (256 / T::UPK) : (tid + 256 * i) / T::UPK; };
    auto place_of = [&](int i) {
        return EVEN ? unit_at<TYPE, T::STRIDE>(tid / T::UPK, tid % T::UPK) + i * (256 / T::UPK) * T::STRIDE
                    : unit_at<TYPE, T::STRIDE>(key_of(i), (tid + 256 * i) % T::UPK);
    };
    auto fetch = [&](const KeyAt* rw) {
#pragma unroll
        for (int i = 0; i < T::PER; i++) {
            const KeyAt row = rw[T::UNITS % 256 == 0 ? key_of(i) : min(key_of(i), KEYS - 1)];
            int ch = EVEN ? tid % T::UPK : (tid + 256 * i) % T::UPK;
            asm volatile("" : "+v"(ch));   // added here: four addresses kept for it over the loop are eight registers
            kr[i] = *reinterpret_cast<const uint4_t*>(g.cache.k + (row.code + ch * 16));
            vr[i] = *reinterpret_cast<const uint4_t*>(g.cache.v + (row.code + ch * 16));
            if constexpr (TYPE != F16) {
                ks[i] = *reinterpret_cast<const _Float16*>(g.cache.k + (row.scale + ch * T::EPU / 32 * 2));
                vs[i] = *reinterpret_cast<const _Float16*>(g.cache.v + (row.scale + ch * T::EPU / 32 * 2));
            }
        }
    };
    uint8_t* const lk = lds;
    uint8_t* const lv = lds + T::PLANE;
    const int own = lds_at<T::STRIDE>(col, part);   // the lane's first chunk of a tile's keys
    if (lo < hi) {
        if (tid < KEYS) rows[0][tid] = row_of(lo + tid), rows[1][tid] = row_of(lo + KEYS + tid);
        __syncthreads();
        fetch(rows[0]);
    }
    int buf = 1;
    for (int k0 = lo; k0 < hi; k0 += KEYS, buf ^= 1) {
        __syncthreads();   // the tile before is read; rows[buf] is the next one's
#pragma unroll
        for (int i = 0; i < T::PER; i++) {
            if (T::UNITS % 256 == 0 || tid + 256 * i < T::UNITS) {
                put_unit<TYPE>(lk, kr[i], ks[i], place_of(i));
                put_unit<TYPE>(lv, vr[i], vs[i], place_of(i));
            }
        }
        // the page of the next but one's keys is asked for first and looked at last: loads come back in their order
        EntryAt after = {};
        if (k0 + KEYS < hi) {
            if (tid < KEYS) after = entry_of(k0 + 2 * KEYS + tid);
            fetch(rows[buf]);
        }
        __syncthreads();
        if (k0 <= c.hi && k0 + KEYS > c.lo) {
            acc_t sc[T::ST];
#pragma unroll
            for (int i = 0; i < T::ST; i++)
#pragma unroll
                for (int k = 0; k < M::N; k++) sc[i][k] = 0.0f;
            half8_t x[2][T::ST];   // a step's keys are on their way while the step before is multiplied
            auto keys_of = [&](int st) {
#pragma unroll
                for (int i = 0; i < T::ST; i++)
                    x[st % 2][i] = *reinterpret_cast<const half8_t*>(lk + lds_step(own, st * 2) + i * NC * T::STRIDE);
            };
            __builtin_amdgcn_s_setprio(1);
            keys_of(0);
            __builtin_amdgcn_sched_group_barrier(0x100, T::ST, 0);
            unroll<0, T::STEPS>([&](auto step) {
                constexpr int st = decltype(step)::value;
                if constexpr (st + 1 < T::STEPS) keys_of(st + 1);
#pragma unroll
                for (int i = 0; i < T::ST; i++) sc[i] = M::mma(x[st % 2][i], qh[st], sc[i]);
#pragma unroll
                for (int i = 0; i < T::ST; i++) sc[i] = M::mma(x[st % 2][i], ql[st], sc[i]);
                if constexpr (st + 1 < T::STEPS) __builtin_amdgcn_sched_group_barrier(0x100, T::ST, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, 2 * T::ST, 0);
            });
            __builtin_amdgcn_s_setprio(0);
            attn_weights<M, T::ST, T::DT, NC, TREE>(sc, o, m, l, f, c, seen[wave][col], a.g, k0, part);
            constexpr int PAIRS = (T::DT + 1) / 2, ALL = KEYS / M::DEPTH * PAIRS;   // pairs of element tiles, over all products
            half8_t v[2][2], ph[2], pl[2];
            auto values_of = [&](int n) {
#pragma unroll
                for (int i = 0; i < 2; i++)
                    if (2 * (n % PAIRS) + i < T::DT) v[n % 2][i] = value_tile<NC, T::STRIDE, M>(lv, 2 * (n % PAIRS) + i, n / PAIRS);
            };
            weight_halves<NC>(sc, 0, ph[0], pl[0]);
            __builtin_amdgcn_s_setprio(1);
            values_of(0);
            unroll<0, ALL>([&](auto step) {
                constexpr int n = decltype(step)::value, u = n / PAIRS, d = 2 * (n % PAIRS), width = d + 1 < T::DT ? 2 : 1;
                constexpr bool more = n + 1 < ALL;
                if constexpr (more) values_of(n + 1);
                if constexpr (more && (n + 1) % PAIRS == 0) weight_halves<NC>(sc, u + 1, ph[(u + 1) % 2], pl[(u + 1) % 2]);
#pragma unroll
                for (int i = 0; i < width; i++) o[d + i] = M::mma(v[n % 2][i], ph[u % 2], o[d + i]);
#pragma unroll
                for (int i = 0; i < width; i++) o[d + i] = M::mma(v[n % 2][i], pl[u % 2], o[d + i]);
                if constexpr (more) __builtin_amdgcn_sched_group_barrier(0x100, (n + 1) % PAIRS * 2 + 1 < T::DT ? 4 : 2, 1);
                __builtin_amdgcn_sched_group_barrier(0x008, 2 * width, 1);
            });
            __builtin_amdgcn_s_setprio(0);
        }
        if (tid < KEYS) rows[buf ^ 1][tid] = key_at<TYPE, D>(g.cache, after, kvh);   // read for the tile before this one; now the next but one's
    }
    l = column_sum<NC>(l);
    c.seen = seen[wave][col];
    for (unsigned long long again = attn_emit<D, NC, T::DT, 1, M>(a, c, o, m, l, split, 0); again; again &= again - 1) {
        const int k = __ffsll(again) - 1;
        attn_row<TYPE, TREE>(g, __builtin_amdgcn_readlane(c.seen.tok, k), __builtin_amdgcn_readlane(c.seen.head, k), redo[wave]);
    }
}

}  // namespace jamhip
