// The attention kernel on the matrix cores.
//
// A workgroup of four waves holds a tile of query rows (rows of one key head: its tokens times the query heads that share it)
// and walks a run of keys, a tile of keys and values at a time: codes come from the cache into registers while the tile before
// is computed, are turned into f16 (what a code stands for is an f16, so nothing is lost) and laid out in shared memory once for
// all rows. Each wave computes, for its columns of NC rows,
//   Sᵀ = K · Qᵀ            a column of scores per lane: the softmax's maximum and sum need one exchange at their end
//   Oᵀ = Vᵀ · Pᵀ           the scores' registers are the second operand's as they stand: its slots take the keys in the order in
//                          which the first product leaves them, and Vᵀ comes out of row-major shared memory in that order
//                          through the transposing read
// Queries and weights are f32 values carried as two f16, hi + lo (22 bits), a product each; the query row is scaled by a power
// of two to a largest element in [1, 2), and weights are 2^(s - m + 7), so neither half runs out of range or into f16's last
// bits. The running maximum m moves only when a score passes it by 8 (in powers of two; weights then stay below 2^15), so
// most tiles rescale nothing. Sums are f32.
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
};

constexpr float WEIGHT_EXP = 7.0f, LAZY = 8.0f, LOG2E = 1.44269504088896340736f;

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
JAMHIP_DEV int wave_min(int v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v = min(v, __shfl_xor(v, o));
    return __builtin_amdgcn_readfirstlane(v);
}
JAMHIP_DEV int wave_max(int v) { return -wave_min(-v); }

template <int TYPE, int D, int CFG> struct Tile {
    static constexpr int NC = CFG == 0 ? 16 : 32;             // rows of a wave
    static constexpr int WK = CFG == 2 ? 1 : 4;               // waves that share a tile's keys
    static constexpr int ROWS = attn_rows(CFG), KEYS = attn_keys(CFG, D), KW = KEYS / WK;
    static_assert(ROWS == NC * (4 / WK) && KW % 32 == 0);
    static constexpr int CHUNKS = (D / 8 + 7) / 8 * 8, STRIDE = CHUNKS * 16;   // of a key's row in shared memory
    static constexpr int PLANE = KEYS * STRIDE;
    static constexpr int EPU = unit_elems<TYPE>(), UPK = D / EPU, UNITS = KEYS * UPK, PER = (UNITS + 255) / 256;
    using M = Mma<NC>;
    static constexpr int PARTS = 64 / NC, STEPS = D / M::DEPTH, ST = KW / NC, DT = D / NC;
    static constexpr int MERGE = WK > 1 ? WK * (D * NC + 2 * NC) * 4 : 0;
    static constexpr int LDS = 2 * PLANE > MERGE ? 2 * PLANE : MERGE;
};

// Byte offset of 16-byte chunk c of a key's row. The key's low bits are spread over the chunk's: eight neighbouring keys' equal
// chunks (the first product's read) fall into eight different 16-byte columns, and so do four neighbouring keys' pairs of
// chunks (the transposing read).
template <int STRIDE> JAMHIP_DEV int lds_at(int key, int c) {
    return key * STRIDE + ((c ^ ((key & 3) * 2 + ((key >> 2) & 1))) << 4);
}

template <int TYPE, int D, int CFG>
__global__ void __launch_bounds__(256, (CFG == 2 && D <= 128) || D <= 64 ? 2 : 1) attn_tile_kernel(AttnArgs a) {
    using T = Tile<TYPE, D, CFG>;
    using M = typename T::M;
    using acc_t = typename M::acc_t;
    constexpr int NC = T::NC, KW = T::KW, KEYS = T::KEYS;
    __shared__ __align__(16) uint8_t lds[T::LDS];
    __shared__ int64_t rows[2][KEYS];
    __shared__ int range[2][4];
    __shared__ float redo[4][ATTN_ROW_FLOATS];
    const Attn& g = a.g;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane % NC, part = lane / NC;
    const int wk = wave % T::WK, wr = wave / T::WK;
    int b = blockIdx.x;
    const int kvh = b % g.cache.kv;
    b /= g.cache.kv;
    const int tile = b % a.part.tiles, split = b / a.part.tiles, mode = a.part.mode;

    // ---- the workgroup's rows and keys
    SeqInfo s = {};
    int r0, n_rows, t_first;   // its first row, rows of the set, the set's first token
    if (mode == 1) {
        int j = -1, rt = 0, from = 0;   // from: tiles of the groups before
        for (int j0 = 0; j0 < g.n_prefixes && j < 0; j0 += 64) {
            const int jj = min(j0 + lane, g.n_prefixes - 1);
            const int s0 = clampi(g.prefix_seqs[jj], 0, g.n_seqs), s1 = clampi(g.prefix_seqs[jj + 1], s0, g.n_seqs);
            const int t0 = clampi(g.q_offsets[s0], 0, g.n_tokens), t1 = clampi(g.q_offsets[s1], t0, g.n_tokens);
            const int tiles = j0 + lane < g.n_prefixes ? ((t1 - t0) * g.grp.d + T::ROWS - 1) / T::ROWS : 0;
            const int before = from + wave_exclusive_scan(tiles);
            const unsigned long long hit = __ballot(tile >= before && tile < before + tiles);
            if (hit) {
                const int l = __ffsll(hit) - 1;
                j = j0 + l;
                rt = tile - __builtin_amdgcn_readlane(before, l);
                t_first = __builtin_amdgcn_readlane(t0, l);
                n_rows = (__builtin_amdgcn_readlane(t1, l) - t_first) * g.grp.d;
            }
            from = __builtin_amdgcn_readlane(before + tiles, 63);
        }
        if (j < 0) return;
        r0 = rt * T::ROWS;
        s.base = clampi(g.prefix_lens[j], 0, g.prefix_cap);
        s.prefix = g.prefix_pages + (int64_t) j * g.ld_prefix_pages;
        s.own = nullptr;
        s.len = 0;
    } else {
        const int per = (g.max_q * g.grp.d + T::ROWS - 1) / T::ROWS, q = tile / per;
        s = seq_info(g, q);
        t_first = s.t0;
        n_rows = s.nq * g.grp.d;
        r0 = (tile - q * per) * T::ROWS;
        if (mode == 2) s.base = 0;   // positions among its own keys
    }
    if (r0 >= n_rows) return;
    const int total = s.base + s.len;

    // ---- the lane's column: a row, the keys that it sees, and its query as the second operand of Sᵀ = K · Qᵀ
    const int r = r0 + wr * NC + col;
    const bool valid = r < n_rows;
    const int tok = t_first + g.grp.div(min(r, n_rows - 1)), head = kvh * g.grp.d + (min(r, n_rows - 1) - (tok - t_first) * g.grp.d);
    int pos = s.base + s.len - s.nq + (tok - s.t0);
    bool live = valid;
    if (mode == 1) {
        const int q = seq_of(g, tok);
        const SeqInfo mine = seq_info(g, max(q, 0));
        live = valid && q >= 0 && tok - mine.t0 < mine.nq;
        pos = mine.base + mine.len - mine.nq + (tok - mine.t0);
    }
    const int c0 = split * a.part.chunk;
    const int k_lo = max(c0, g.window > 0 ? pos - g.window + 1 : 0), k_hi = min(min(total, c0 + a.part.chunk) - 1, pos);   // first and last
    const bool some = live && k_lo <= k_hi;
    const int see_lo = some ? k_lo : INT32_MAX, see_n = some ? k_hi - k_lo : 0;   // key sees: (unsigned) (key - see_lo) <= see_n
    const int w_lo = wave_min(some ? k_lo : INT32_MAX), w_hi = wave_max(some ? k_hi : -1);
    const int all_lo = wave_max(live ? (some ? k_lo : INT32_MAX) : -1), all_hi = wave_min(live ? (some ? k_hi : -1) : INT32_MAX);
    if (lane == 0) range[0][wave] = w_lo, range[1][wave] = w_hi;

    half8_t qh[T::STEPS], ql[T::STEPS];
    float f;   // a score in powers of two is f times the product
    {
        const float* q = g.q + (int64_t) tok * g.ldq + (int64_t) head * D;
        float top = 0.0f;
        float x[T::STEPS][8];
        const bool al = (reinterpret_cast<uintptr_t>(q) & 15) == 0;
#pragma unroll
        for (int st = 0; st < T::STEPS; st++) {
            const float* p = q + st * M::DEPTH + part * 8;
            if (al) {
                const float4_t u = *reinterpret_cast<const float4_t*>(p), v = *reinterpret_cast<const float4_t*>(p + 4);
#pragma unroll
                for (int i = 0; i < 4; i++) x[st][i] = u[i], x[st][4 + i] = v[i];
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) x[st][i] = p[i];
            }
#pragma unroll
            for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(x[st][i]));
        }
        top = column_max<NC>(top);
        const int e = top > 0.0f && top < __builtin_inff() ? ilogbf(top) : 0;
        f = ldexpf(g.scale * LOG2E, e);
#pragma unroll
        for (int st = 0; st < T::STEPS; st++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float y = ldexpf(x[st][i], -e);
                qh[st][i] = (_Float16) y;
                ql[st][i] = (_Float16) (y - (float) qh[st][i]);
            }
    }
    __syncthreads();
    const int lo = min(min(range[0][0], range[0][1]), min(range[0][2], range[0][3]));
    const int hi = max(max(range[1][0], range[1][1]), max(range[1][2], range[1][3])) + 1;   // one past the last

    acc_t o[T::DT];
#pragma unroll
    for (int i = 0; i < T::DT; i++)
#pragma unroll
        for (int k = 0; k < M::N; k++) o[i][k] = 0.0f;
    float m = -__builtin_inff(), l = 0.0f;

    // ---- the keys
    uint4_t kr[T::PER], vr[T::PER];
    _Float16 ks[T::PER], vs[T::PER];
    auto row_of = [&](int at) -> int64_t { return at < hi ? entry_row(g.cache, s, at, kvh) : -1; };
    auto fetch = [&](const int64_t* rw) {
#pragma unroll
        for (int i = 0; i < T::PER; i++) {
            const int u = tid + 256 * i, key = u / T::UPK, c = u % T::UPK;
            const int64_t row = T::UNITS % 256 == 0 || u < T::UNITS ? rw[key] : -1;
            kr[i] = vr[i] = uint4_t{0, 0, 0, 0};
            ks[i] = vs[i] = (_Float16) 0.0f;
            if (row >= 0) {
                const int64_t at = (row * T::UPK + c) * 16;
                kr[i] = *reinterpret_cast<const uint4_t*>(g.cache.k + at);
                vr[i] = *reinterpret_cast<const uint4_t*>(g.cache.v + at);
                if constexpr (TYPE != F16) {
                    const int64_t sc = g.cache.scale_off + (row * (D / 32) + c * T::EPU / 32) * 2;
                    ks[i] = *reinterpret_cast<const _Float16*>(g.cache.k + sc);
                    vs[i] = *reinterpret_cast<const _Float16*>(g.cache.v + sc);
                }
            }
        }
    };
    auto put = [&](uint8_t* plane, const uint4_t& w, _Float16 sc, int key, int c) {
        if constexpr (TYPE == F16) {
            *reinterpret_cast<uint4_t*>(plane + lds_at<T::STRIDE>(key, c)) = w;
        } else {
            const half2_t scale = {sc, sc};
            half2_t h[16];
            if constexpr (TYPE == Q8_0) {
#pragma unroll
                for (int i = 0; i < 4; i++) q8_word(w[i], scale, h + 2 * i);
            } else {
                // bytes j: element j low, element 16 + j high. Zeros of an absent key: its scale is 0
#pragma unroll
                for (int i = 0; i < 4; i++) q4_word(w[i], scale, h + 2 * i), q4_word(w[i] >> 4, scale, h + 8 + 2 * i);
            }
#pragma unroll
            for (int i = 0; i < T::EPU / 8; i++) {
                const uint4_t v = {as_u32(h[4 * i]), as_u32(h[4 * i + 1]), as_u32(h[4 * i + 2]), as_u32(h[4 * i + 3])};
                *reinterpret_cast<uint4_t*>(plane + lds_at<T::STRIDE>(key, c * (T::EPU / 8) + i)) = v;
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
            const int u = tid + 256 * i, key = u / T::UPK, c = u % T::UPK;
            if (T::UNITS % 256 == 0 || u < T::UNITS) {
                put(lk, kr[i], ks[i], key, c);
                put(lv, vr[i], vs[i], key, c);
            }
        }
        if (k0 + KEYS < hi) fetch(rows[buf]);
        int64_t after = -1;
        if (tid < KEYS && k0 + 2 * KEYS < hi) after = row_of(k0 + 2 * KEYS + tid);
        __syncthreads();
        const int kb = wk * KW, kw = k0 + kb;   // the wave's keys
        if (kw <= w_hi && kw + KW > w_lo) {
            acc_t sc[T::ST];
#pragma unroll
            for (int i = 0; i < T::ST; i++) {
#pragma unroll
                for (int k = 0; k < M::N; k++) sc[i][k] = 0.0f;
#pragma unroll
                for (int st = 0; st < T::STEPS; st++) {
                    const half8_t x = *reinterpret_cast<const half8_t*>(lk + lds_at<T::STRIDE>(kb + i * NC + col, st * T::PARTS + part));
                    sc[i] = M::mma(x, qh[st], sc[i]);
                    sc[i] = M::mma(x, ql[st], sc[i]);
                }
            }
            if (kw < all_lo || kw + KW - 1 > all_hi) {
#pragma unroll
                for (int i = 0; i < T::ST; i++)
#pragma unroll
                    for (int k = 0; k < M::N; k++)
                        if ((unsigned) (kw + i * NC + M::row(k, part) - see_lo) > (unsigned) see_n) sc[i][k] = -__builtin_inff();
            }
            float top = sc[0][0];
#pragma unroll
            for (int i = 0; i < T::ST; i++)
#pragma unroll
                for (int k = 0; k < M::N; k++) top = fmaxf(top, sc[i][k]);
            top = column_max<NC>(top) * f;
            if (__any(top > m + LAZY)) {
                const float now = fmaxf(m, top), keep = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - now);
                m = now;
                l *= keep;
#pragma unroll
                for (int i = 0; i < T::DT; i++)
#pragma unroll
                    for (int k = 0; k < M::N; k++) o[i][k] *= keep;
            }
            const float shift = WEIGHT_EXP - (m == -__builtin_inff() ? 0.0f : m);
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < T::ST; i++)
#pragma unroll
                for (int k = 0; k < M::N; k++) {
                    sc[i][k] = __builtin_amdgcn_exp2f(fmaf(sc[i][k], f, shift));
                    sum += sc[i][k];
                }
            l += sum;
            // 8 weights a lane are one product's second operand: 16 keys (two of a 32-row tile's four groups) or 32 (two tiles)
#pragma unroll
            for (int u = 0; u < KW / M::DEPTH; u++) {
                half8_t ph, pl;
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float x = NC == 32 ? sc[u / 2][8 * (u % 2) + e] : sc[2 * u + e / 4][e % 4];
                    const float y = NC == 32 ? sc[u / 2][8 * (u % 2) + e + 1] : sc[2 * u + e / 4][e % 4 + 1];
                    const half2_t h = pack_rtz(x, y), r2 = pack_rtz(x - (float) h[0], y - (float) h[1]);
                    ph[e] = h[0], ph[e + 1] = h[1], pl[e] = r2[0], pl[e + 1] = r2[1];
                }
#pragma unroll
                for (int dt = 0; dt < T::DT; dt++) {
                    // 16 lanes read 4 keys of 16 elements and get 4 keys of their element
                    const int in = lane % 16, sub = NC == 32 ? (lane / 16) % 2 : 0;
                    const int key = kb + u * M::DEPTH + 4 * part + in / 4, e0 = dt * NC + sub * 16 + 4 * (in % 4);
                    auto at = [&](int k) {
                        const uint8_t* p = lv + lds_at<T::STRIDE>(k, e0 / 8) + e0 % 8 * 2;
                        const short4_t v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) short4_t*) (uintptr_t) (__attribute__((address_space(3))) const uint8_t*) p);
                        return __builtin_bit_cast(half4_t, v);
                    };
                    const half8_t v = join_half(at(key), at(key + M::DEPTH / 2));
                    o[dt] = M::mma(v, ph, o[dt]);
                    o[dt] = M::mma(v, pl, o[dt]);
                }
            }
        }
        if (tid < KEYS) rows[buf ^ 1][tid] = after;   // read for the tile before this one; now the next but one's
    }

    // ---- the result
    l = column_sum<NC>(l);
    if constexpr (T::WK > 1) {   // the waves' parts, through shared memory: [wave][element][column], then [wave][column] m and l
        __syncthreads();
        float* const po = reinterpret_cast<float*>(lds);
        float* const pm = po + T::WK * D * NC;
        float* const pl = pm + T::WK * NC;
#pragma unroll
        for (int dt = 0; dt < T::DT; dt++)
#pragma unroll
            for (int k = 0; k < M::N; k++) po[(wave * D + dt * NC + M::row(k, part)) * NC + col] = o[dt][k];
        if (part == 0) pm[wave * NC + col] = m, pl[wave * NC + col] = l;
        __syncthreads();
        float w[T::WK], top = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < T::WK; i++) top = fmaxf(top, pm[i * NC + col]);
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < T::WK; i++) {
            w[i] = top == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(pm[i * NC + col] - top);
            l += pl[i * NC + col] * w[i];
        }
        m = top;
        // wave w sums the element tiles w, w + 4, ...
#pragma unroll
        for (int dt = 0; dt < T::DT; dt++)
            if (dt % T::WK == wave)
#pragma unroll
                for (int k = 0; k < M::N; k++) {
                    float v = 0.0f;
#pragma unroll
                    for (int i = 0; i < T::WK; i++) v += w[i] * po[(i * D + dt * NC + M::row(k, part)) * NC + col];
                    o[dt][k] = v;
                }
    }
    const int64_t out_row = (int64_t) tok * g.heads + head;
    float scale = 1.0f;
    float* dst;
    if (a.part.direct) {
        if (g.sinks != nullptr) {
            const float x = g.sinks[head] * LOG2E, now = fmaxf(m, x);
            const float keep = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - now);
            l = l * keep + (now == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(x - now + WEIGHT_EXP));
            scale = keep;
        }
        scale = l == 0.0f ? 0.0f : scale / l;
        dst = g.out + (int64_t) tok * g.ldo + (int64_t) head * D;
    } else {
        const int64_t n = (int64_t) g.n_tokens * g.heads, at = (int64_t) (a.part.slot0 + split) * n + out_row;
        dst = a.acc + at * D;
        if (live && part == 0 && (T::WK == 1 || wave == 0)) a.ml[at] = make_float2(m, l);
    }
    const bool al = (reinterpret_cast<uintptr_t>(dst) & 15) == 0;
    bool bad = false;
#pragma unroll
    for (int dt = 0; dt < T::DT; dt++) {
        if (T::WK > 1 && dt % T::WK != wave) continue;
#pragma unroll
        for (int k = 0; k < M::N; k += 4) {
            float4_t v;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v[e] = o[dt][k + e] * scale;
                bad |= !(fabsf(v[e]) < __builtin_inff());
            }
            float* p = dst + dt * NC + M::row(k, part);
            if (live) {
                if (al) {
                    *reinterpret_cast<float4_t*>(p) = v;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) p[e] = v[e];
                }
            }
        }
    }
    // A row that is not finite may owe it to an entry that it does not see (0 times what a masked value holds): computed again,
    // masked entries left out entirely
    if (a.part.direct) {
        unsigned long long again = __ballot(bad && live);
        if constexpr (T::WK > 1) {
            __syncthreads();
            if (lane == 0) range[0][wave] = (int) (uint32_t) again, range[1][wave] = (int) (uint32_t) (again >> 32);
            __syncthreads();
            again = 0;
            for (int i = 0; i < 4; i++) again |= (uint32_t) range[0][i] | (unsigned long long) (uint32_t) range[1][i] << 32;
        }
#pragma unroll
        for (int o2 = NC; o2 < 64; o2 <<= 1) again |= again >> o2;
        again &= (1ull << NC) - 1;
        for (; again; again &= again - 1) {
            const int c = __ffsll(again) - 1;
            if (T::WK == 1 || c % 4 == wave)
                attn_row<TYPE>(g, __builtin_amdgcn_readlane(tok, c), __builtin_amdgcn_readlane(head, c), redo[wave]);
        }
    }
}

template <int TYPE, int D, int CFG> hipError_t launch_attn_tile(const AttnArgs& a, hipStream_t st) {
    const int64_t blocks = (int64_t) a.g.cache.kv * a.part.tiles * a.part.splits;
    if (blocks > INT32_MAX) return hipErrorNotSupported;
    attn_tile_kernel<TYPE, D, CFG><<<(uint32_t) blocks, 256, 0, st>>>(a);
    return hipGetLastError();
}

template <int TYPE, int D> hipError_t launch_attn_tile(const AttnArgs& a, hipStream_t st) {
    switch (a.part.cfg) {
        case 0: return launch_attn_tile<TYPE, D, 0>(a, st);
        case 1: return launch_attn_tile<TYPE, D, 1>(a, st);
        default: return launch_attn_tile<TYPE, D, 2>(a, st);
    }
}

template <int TYPE> hipError_t launch_attn_tile(const AttnArgs& a, hipStream_t st) {
    switch (a.g.cache.dim) {
        case 64: return launch_attn_tile<TYPE, 64>(a, st);
        case 96: return launch_attn_tile<TYPE, 96>(a, st);
        case 128: return launch_attn_tile<TYPE, 128>(a, st);
        case 192: return launch_attn_tile<TYPE, 192>(a, st);
        case 256: return launch_attn_tile<TYPE, 256>(a, st);
    }
    return hipErrorNotSupported;
}

hipError_t launch_attn_f16(const AttnArgs& a, hipStream_t st);
hipError_t launch_attn_q8(const AttnArgs& a, hipStream_t st);
hipError_t launch_attn_q4(const AttnArgs& a, hipStream_t st);

}  // namespace jamhip
