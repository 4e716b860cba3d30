// The attention kernel for many rows of a key head.
//
// A workgroup of four waves holds 128 query rows (rows of one key head: its tokens times the query heads that share it), 32 a
// wave, and walks a run of keys, a tile of keys and values at a time: codes come from the cache into registers while the tile
// before is computed, are turned into f16 and laid out in shared memory once for all rows.
//
// Bound by the matrix cores and the VALU alike, each busy about half of the time: at head_dim 64 a tile costs a wave 1024 cycles of
// products (two for each, for the halves) and about 1100 of VALU (an exponential of 16 cycles, a fused multiply-add, a sum, a
// maximum, two conversions and a difference for each of 32 scores a lane), and two waves a SIMD take 3900 for it. 64 sequences of 4 heads
// behind 8192 tokens in Q8_0, 8 key heads of 128: 31 to 33 us; 8 prompts of up to 256 tokens behind 4096 in F16, heads of 64: 293 to 301 us
// from card to card (434 to 422 TFLOP/s, counted once) after some fifty calls in a row, 340 to 390 before, while the clock rises. Two halves of
// shared memory with one barrier a tile took 37.8 for the first, 16 runs of keys for 32 took 38. At head_dim 128 the two halves of
// the query and the next tile's codes are more than 256 registers: 25 (F16), 14 (Q8_0) and 4 (Q4_0) of them go to scratch, at 256 24 to 33.
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

template <int TYPE, int D> __global__ void __launch_bounds__(256, D <= 128 ? 2 : 1) attn_tile_kernel(AttnArgs a) {
    using T = Tile<TYPE, D>;
    using M = typename T::M;
    using acc_t = typename M::acc_t;
    constexpr int NC = T::NC, KEYS = T::KEYS;
    __shared__ __align__(16) uint8_t lds[2 * T::PLANE];
    __shared__ __align__(16) KeyAt rows[2][KEYS];
    __shared__ int range[2][4];
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
    const Column c = attn_column(a, w, w.r0 + wave * NC + col, kvh, split);
    if (lane == 0) range[0][wave] = c.lo, range[1][wave] = c.hi;
    half8_t qh[T::STEPS], ql[T::STEPS];
    const float f = load_query<NC>(g.q + (int64_t) c.tok * g.ldq + (int64_t) c.head * D, g.scale, qh, ql,
                                   [&](int st, int j) { return st * M::DEPTH + part * 8 + j; });
    __syncthreads();
    const int lo = min(min(range[0][0], range[0][1]), min(range[0][2], range[0][3]));
    const int hi = max(max(range[1][0], range[1][1]), max(range[1][2], range[1][3])) + 1;   // one past the last

    acc_t o[T::DT];
#pragma unroll
    for (int i = 0; i < T::DT; i++)
#pragma unroll
        for (int k = 0; k < M::N; k++) o[i][k] = 0.0f;
    float m = -__builtin_inff(), l = 0.0f;

    uint4_t kr[T::PER], vr[T::PER];
    _Float16 ks[T::PER] = {}, vs[T::PER] = {};
    // past the last key it stands for that one: no load is behind a branch, and nothing that no row sees comes in
    auto row_of = [&](int at) { return key_at<TYPE, D>(g.cache, w.s, min(at, hi - 1), kvh); };
    auto fetch = [&](const KeyAt* rw) {
#pragma unroll
        for (int i = 0; i < T::PER; i++) {
            const int u = tid + 256 * i, key = u / T::UPK, ch = u % T::UPK;
            const KeyAt row = rw[T::UNITS % 256 == 0 ? key : min(key, KEYS - 1)];
            kr[i] = *reinterpret_cast<const uint4_t*>(g.cache.k + row.code + ch * 16);
            vr[i] = *reinterpret_cast<const uint4_t*>(g.cache.v + row.code + ch * 16);
            if constexpr (TYPE != F16) {
                ks[i] = *reinterpret_cast<const _Float16*>(g.cache.k + row.scale + ch * T::EPU / 32 * 2);
                vs[i] = *reinterpret_cast<const _Float16*>(g.cache.v + row.scale + ch * T::EPU / 32 * 2);
            }
        }
    };
    uint8_t* const lk = lds;
    uint8_t* const lv = lds + T::PLANE;
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
            const int u = tid + 256 * i, key = u / T::UPK, ch = u % T::UPK;
            if (T::UNITS % 256 == 0 || u < T::UNITS) {
                put_unit<TYPE, T::STRIDE>(lk, kr[i], ks[i], key, ch);
                put_unit<TYPE, T::STRIDE>(lv, vr[i], vs[i], key, ch);
            }
        }
        KeyAt after = {};
        if (k0 + KEYS < hi) {
            fetch(rows[buf]);
            if (tid < KEYS) after = row_of(k0 + 2 * KEYS + tid);
        }
        __syncthreads();
        if (k0 <= c.hi && k0 + KEYS > c.lo) {
            acc_t sc[T::ST];
#pragma unroll
            for (int i = 0; i < T::ST; i++)
#pragma unroll
                for (int k = 0; k < M::N; k++) sc[i][k] = 0.0f;
#pragma unroll
            for (int st = 0; st < T::STEPS; st++) {
                half8_t x[T::ST];
#pragma unroll
                for (int i = 0; i < T::ST; i++) x[i] = *reinterpret_cast<const half8_t*>(lk + lds_at<T::STRIDE>(i * NC + col, st * 2 + part));
#pragma unroll
                for (int i = 0; i < T::ST; i++) sc[i] = M::mma(x[i], qh[st], sc[i]);
#pragma unroll
                for (int i = 0; i < T::ST; i++) sc[i] = M::mma(x[i], ql[st], sc[i]);
            }
            attn_weights<M, T::ST, T::DT, NC>(sc, o, m, l, f, c, k0, part);
#pragma unroll
            for (int u = 0; u < KEYS / M::DEPTH; u++) {
                half8_t ph, pl;
                weight_halves<NC>(sc, u, ph, pl);
                add_values<NC, T::DT, T::STRIDE, M>(o, lv, 0, u, ph, pl);
            }
        }
        if (tid < KEYS) rows[buf ^ 1][tid] = after;   // read for the tile before this one; now the next but one's
    }
    l = column_sum<NC>(l);
    for (unsigned long long again = attn_emit<D, NC, T::DT, 1, M>(a, c, o, m, l, split, 0); again; again &= again - 1) {
        const int k = __ffsll(again) - 1;
        attn_row<TYPE>(g, __builtin_amdgcn_readlane(c.tok, k), __builtin_amdgcn_readlane(c.head, k), redo[wave]);
    }
}

}  // namespace jamhip
