// The next token of each row of logits from a given random number: temperature, top-k, top-p, min-p.
//
// With x sorted by value, largest first and equal ones by index, and w = exp((x - max) / t) in 64 bits:
//   top-k keeps the first k; top-p, of those, the ones before which less than p · (their sum) has been summed, the first in
//   any case; min-p those with w >= min_p. The token is the first in the vocabulary's order whose running sum of kept weights
//   exceeds u · (their sum). Temperature 0: the first of the largest. logprob = x - max - log(sum of exp(x - max)), over all.
//
// Two launches. The first reads the logits once, a slice of 4096 a workgroup: the largest and its first index, the sums at
// temperature 1 and t relative to the slice's largest, the largest of every 16 elements, and, for a row that top-p or min-p
// cuts without top-k, a histogram of the weights over 1024 bins of the value. The second, a workgroup per row, finds the
// cut: with top-k the k-th largest of the 16-element maxima bounds the k-th largest element from below, which leaves few
// candidates to read again and sort; from the histogram the cut falls into one bin, whose elements alone are sorted. The kept
// set is then {(x, index) >= T}, a slice's kept sum follows from its histogram, and only the slice in which the token lies
// is read once more. Where candidates or a bin are too many to sort (large k, thousands of equal values), and past 262144
// logits, the cut is found digit by digit of the values' order-preserving 32-bit keys from histograms over the whole row, by one
// workgroup: with all filters one row of 262144 takes 15 us and of 262145 2.3 ms, 64 rows 31 us and 4.8 ms.
// Weights are summed in histograms as 64-bit integers, so that the order of the atomics does not matter.
//
// 128256 logits, first + second launch: one row with all filters 4 + 10 us, without any 6.5 + 7; 64 rows 11 + 13 and 19 + 7 (33 MB: the
// first is 3.1 TB/s without 64-bit weights, which are the rest). With top-p alone 64 rows take 26 + 43, min-p alone 23 + 32: where the
// cut lies in the bulk of the row, its workgroup reads the row again, at what one CU gets from beyond its L2.
#include "launch.h"
#include "sample_sort.h"

namespace jamhip {

namespace {

// A larger value has the larger key; NaN counts as -Inf. Both zeros have one key, as they are equal.
JAMHIP_DEV uint32_t key_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x == 0.0f ? 0.0f : x != x ? -__builtin_inff() : x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
JAMHIP_DEV float of_key(uint32_t k) { return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

JAMHIP_DEV int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }

template <int CTRL, int ROWS = 0xF> JAMHIP_DEV int dpp_int(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, true); }
template <int CTRL, int ROWS = 0xF> JAMHIP_DEV double dpp_f64(double v) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
    const uint32_t lo = dpp_int<CTRL, ROWS>((int) b), hi = dpp_int<CTRL, ROWS>((int) (b >> 32));
    return __builtin_bit_cast(double, (unsigned long long) hi << 32 | lo);
}
JAMHIP_DEV double lane_f64(double v, int l) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int) b, l), hi = __builtin_amdgcn_readlane((int) (b >> 32), l);
    return __builtin_bit_cast(double, (unsigned long long) hi << 32 | lo);
}

// Over the 64 lanes, the same in each: a butterfly within rows of 16, then the rows (as wave_sum).
JAMHIP_DEV double wave_sum_f64(double v) {
    v += dpp_f64<0xB1>(v);
    v += dpp_f64<0x4E>(v);
    v += dpp_f64<0x141>(v);
    v += dpp_f64<0x140>(v);
    return (lane_f64(v, 0) + lane_f64(v, 16)) + (lane_f64(v, 32) + lane_f64(v, 48));
}
JAMHIP_DEV int wave_sum_int(int v) {
    v += dpp_int<0xB1>(v);
    v += dpp_int<0x4E>(v);
    v += dpp_int<0x141>(v);
    v += dpp_int<0x140>(v);
    return __builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16) + __builtin_amdgcn_readlane(v, 32) +
           __builtin_amdgcn_readlane(v, 48);
}
JAMHIP_DEV uint32_t wave_max_u32(uint32_t v) {
    v = max(v, (uint32_t) dpp_int<0xB1>((int) v));
    v = max(v, (uint32_t) dpp_int<0x4E>((int) v));
    v = max(v, (uint32_t) dpp_int<0x141>((int) v));
    v = max(v, (uint32_t) dpp_int<0x140>((int) v));
    return max(max((uint32_t) __builtin_amdgcn_readlane((int) v, 0), (uint32_t) __builtin_amdgcn_readlane((int) v, 16)),
               max((uint32_t) __builtin_amdgcn_readlane((int) v, 32), (uint32_t) __builtin_amdgcn_readlane((int) v, 48)));
}
// The largest key and, of the lanes that have it, the lowest index.
JAMHIP_DEV void wave_largest(uint32_t* key, int* idx) {
    const uint32_t k = wave_max_u32(*key);
    *idx = (int) ~wave_max_u32(*key == k ? ~(uint32_t) *idx : 0);
    *key = k;
}

// 2^(-j / 64). A kernel that needs weights copies it to shared memory: its code is read for the first time on every launch, so
// one short series over a table beats a long one (and every site of it counts).
__device__ const double POW[64] = {
    0x1.0000000000000p+0, 0x1.fa7c1819e90d8p-1, 0x1.f50765b6e4540p-1, 0x1.efa1bee615a27p-1,
    0x1.ea4afa2a490dap-1, 0x1.e502ee78b3ff6p-1, 0x1.dfc97337b9b5fp-1, 0x1.da9e603db3285p-1,
    0x1.d5818dcfba487p-1, 0x1.d072d4a07897cp-1, 0x1.cb720dcef9069p-1, 0x1.c67f12e57d14bp-1,
    0x1.c199bdd85529cp-1, 0x1.bcc1e904bc1d2p-1, 0x1.b7f76f2fb5e47p-1, 0x1.b33a2b84f15fbp-1,
    0x1.ae89f995ad3adp-1, 0x1.a9e6b5579fdbfp-1, 0x1.a5503b23e255dp-1, 0x1.a0c667b5de565p-1,
    0x1.9c49182a3f090p-1, 0x1.97d829fde4e50p-1, 0x1.93737b0cdc5e5p-1, 0x1.8f1ae99157736p-1,
    0x1.8ace5422aa0dbp-1, 0x1.868d99b4492edp-1, 0x1.82589994cce13p-1, 0x1.7e2f336cf4e62p-1,
    0x1.7a11473eb0187p-1, 0x1.75feb564267c9p-1, 0x1.71f75e8ec5f74p-1, 0x1.6dfb23c651a2fp-1,
    0x1.6a09e667f3bcdp-1, 0x1.6623882552225p-1, 0x1.6247eb03a5585p-1, 0x1.5e76f15ad2148p-1,
    0x1.5ab07dd485429p-1, 0x1.56f4736b527dap-1, 0x1.5342b569d4f82p-1, 0x1.4f9b2769d2ca7p-1,
    0x1.4bfdad5362a27p-1, 0x1.486a2b5c13cd0p-1, 0x1.44e086061892dp-1, 0x1.4160a21f72e2ap-1,
    0x1.3dea64c123422p-1, 0x1.3a7db34e59ff7p-1, 0x1.371a7373aa9cbp-1, 0x1.33c08b26416ffp-1,
    0x1.306fe0a31b715p-1, 0x1.2d285a6e4030bp-1, 0x1.29e9df51fdee1p-1, 0x1.26b4565e27cddp-1,
    0x1.2387a6e756238p-1, 0x1.2063b88628cd6p-1, 0x1.1d4873168b9aap-1, 0x1.1a35beb6fcb75p-1,
    0x1.172b83c7d517bp-1, 0x1.1429aaea92de0p-1, 0x1.11301d0125b51p-1, 0x1.0e3ec32d3d1a2p-1,
    0x1.0b5586cf9890fp-1, 0x1.0874518759bc8p-1, 0x1.059b0d3158574p-1, 0x1.02c9a3e778061p-1,
};

// e^-y, y >= 0, in 64 bits: y = n · ln 2 / 64 - r with ln 2 / 64 in two parts, 2^(-n / 64) from the table, and the series of e^r to
// r^5, whose first omitted term is 0.0055^6 / 6!, below 4e-17.
JAMHIP_DEV double exp_neg(double y, const double* pow) {
    const double magic = 6755399441055744.0;   // 1.5 · 2^52: adding it rounds to a whole number, in the low bits
    const double live = y < 700.0 ? 1.0 : 0.0;   // past e^-700 nothing is left; a factor, since a branch would keep weights apart
    y = fmin(y, 700.0);
    const double t = fma(y, 92.332482616893656877, magic), n = t - magic;
    double r = fma(n, 0.010830424696249145, -y);
    r = fma(n, 3.623510646634843e-19, r);
    double p = fma(1.0 / 120.0, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    const unsigned long long i = __builtin_bit_cast(unsigned long long, t);
    const unsigned long long v = __builtin_bit_cast(unsigned long long, p * pow[i & 63]);
    // times 2^-(n / 64), in the exponent's bits
    return __builtin_bit_cast(double, v - ((unsigned long long) ((uint32_t) i >> 6) << 52)) * live;
}

// exp(-(top - x) / t); equal to 1 at the top whatever its value, 0 for -Inf below it
JAMHIP_DEV double weight(double top, float x, double inv_t, const double* pow) {
    const double w = exp_neg((top - (double) x) * inv_t, pow);
    return (double) x >= top ? 1.0 : w;
}

struct RowParams {
    float t;
    int k;
    double p, min_p, u;
};
JAMHIP_DEV RowParams params_of(const Sample& g, int row) {
    // every array is read, one that is absent through another's address, so that no load waits for a branch
    const float t = (g.temperature ? g.temperature : g.u)[row], p = (g.top_p ? g.top_p : g.u)[row], m = (g.min_p ? g.min_p : g.u)[row];
    const int k = (g.top_k ? g.top_k : reinterpret_cast<const int*>(g.u))[row];
    RowParams r;
    r.t = g.temperature ? t : 1.0f;
    r.k = g.top_k ? k : 0;
    r.p = g.top_p ? (double) p : 1.0;
    r.p = r.p < 0.0 ? 0.0 : r.p;
    r.min_p = g.min_p ? fmin((double) m, 1.0) : 0.0;
    r.u = (double) g.u[row];
    return r;
}

struct Kept {          // the kept set: keys above `key`, and the first `ties` with that key
    uint32_t key;
    int64_t ties;
};

// The general way: the token of a row whose largest key is bk, T found digit by digit.
struct GeneralLds {
    unsigned long long hist[256];
    double wsum[SM_WAVES];
    int wtie[SM_WAVES];
    uint32_t digit;
    unsigned long long rest;
    int token;
};
JAMHIP_DEV int sample_general(const Sample& g, int row, uint32_t bk, const RowParams& rp, GeneralLds& sh, const double* pow) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = g.vocab;
    const float* x = g.logits + (int64_t) row * g.ld;
    const double top = (double) of_key(bk), inv_t = 1.0 / (double) rp.t;
    Kept kept = {0, (int64_t) n};
    int bits = 0;   // 2^bits >= n: the fixed-point weights' sum stays below 2^63
    while ((int64_t(1) << bits) < n) bits++;
    const double unit = __builtin_ldexp(1.0, 62 - bits);
    // T from a histogram of the next 8 bits below `prefix`, four times: the digit in whose bin the running sum, from the
    // top, first reaches `want`
    auto select = [&](auto&& add, unsigned long long want) -> Kept {
        uint32_t prefix = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int b = tid; b < 256; b += SM_THREADS) sh.hist[b] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += SM_THREADS) {
                const uint32_t k = key_of(x[i]);
                if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) {
                    const unsigned long long a = add(i, k);
                    if (a) atomicAdd(&sh.hist[(k >> shift) & 255], a);
                }
            }
            __syncthreads();
            if (tid == 0) {
                unsigned long long run = 0;
                int b = 255;
                for (; b > 0 && run + sh.hist[b] < want; b--) run += sh.hist[b];
                sh.digit = b;
                sh.rest = want - run;
            }
            __syncthreads();
            prefix |= sh.digit << shift;
            want = sh.rest;
            __syncthreads();
        }
        return Kept{prefix, (int64_t) want};   // want: what is still wanted of the bin of this one key
    };
    const int64_t k = rp.k;
    if (k > 0 && k < n) kept = select([&](int, uint32_t) { return 1ull; }, (unsigned long long) k);
    const double p = rp.p;
    auto fixed = [&](uint32_t key) { return (unsigned long long) (weight(top, of_key(key), inv_t, pow) * unit); };
    if (p < 1.0) {
        // the sum of what top-k left, its ties by their number
        if (tid == 0) sh.rest = 0;
        __syncthreads();
        unsigned long long mine = 0;
        for (int i = tid; i < n; i += SM_THREADS) {
            const uint32_t key = key_of(x[i]);
            if (key > kept.key) mine += fixed(key);
        }
        atomicAdd(&sh.rest, mine);
        __syncthreads();
        const unsigned long long at = fixed(kept.key);
        const unsigned long long total = sh.rest + (kept.key ? at * (unsigned long long) kept.ties : 0ull);
        __syncthreads();
        const double goal = p * (double) total;
        unsigned long long want = (unsigned long long) ceil(goal);
        if (want < 1) want = 1;
        const Kept was = kept;
        // a kept value's weight; T's own ties count in its bin as often as they are kept
        Kept now = select([&](int, uint32_t key) { return key > was.key ? fixed(key) : 0ull; }, want);
        const unsigned long long w = fixed(now.key);
        if (now.key > was.key) {   // first j with j · w >= the rest of the bin
            kept.key = now.key;
            kept.ties = w ? ((unsigned long long) now.ties + w - 1) / w : (int64_t) n;
        } else if (was.key) {      // among top-k's own ties
            const unsigned long long over = total - at * (unsigned long long) was.ties;   // summed above them
            const unsigned long long rest = want > over ? want - over : 1;
            const int64_t j = at ? (int64_t) ((rest + at - 1) / at) : was.ties;
            kept.ties = j < was.ties ? j : was.ties;
        }
        if (kept.ties < 1) kept.ties = 1;
    }
    const double minp = rp.min_p;
    // wave w takes the run [w · span, (w + 1) · span) of the vocabulary
    const int span = (n + SM_WAVES - 1) / SM_WAVES, lo = min(n, wave * span), hi = min(n, lo + span);
    int ties = 0;
    for (int i0 = lo; i0 < hi; i0 += 64) {
        const int i = i0 + lane;
        ties += __popcll(__ballot(i < hi && key_of(x[min(i, n - 1)]) == kept.key));
    }
    if (lane == 0) sh.wtie[wave] = ties;
    __syncthreads();
    int64_t before = 0;
    for (int w = 0; w < wave; w++) before += sh.wtie[w];
    // one 64-element step of the wave's run: the element's kept weight
    auto step = [&](int i, int64_t* seen) -> double {
        const float v = i < hi ? x[i] : 0.0f;
        const uint32_t key = key_of(v);
        const bool tie = i < hi && key == kept.key;
        const unsigned long long b = __ballot(tie);
        const int64_t rank = *seen + __popcll(b & ((1ull << lane) - 1));
        *seen += __popcll(b);
        if (i >= hi || key < kept.key || (tie && rank >= kept.ties)) return 0.0;
        const double w = weight(top, of_key(key), inv_t, pow);
        return w >= minp || key == bk ? w : 0.0;
    };
    double mine = 0.0;
    int64_t seen = before;
    for (int i0 = lo; i0 < hi; i0 += 64) mine += step(i0 + lane, &seen);
    mine = wave_sum_f64(mine);
    if (lane == 0) sh.wsum[wave] = mine;
    if (tid == 0) sh.token = -1;
    __syncthreads();
    double total = 0.0;
    for (int w = 0; w < SM_WAVES; w++) total += sh.wsum[w];
    const double goal = rp.u * total;
    double run = 0.0;
    int at = -1, last = 0;
    for (int w = 0; w < SM_WAVES; w++) {
        if (sh.wsum[w] > 0.0) last = w;
        if (at < 0) {
            if (run + sh.wsum[w] > goal) at = w;
            else run += sh.wsum[w];
        }
    }
    const bool over = at < 0;   // rounding: the last kept one
    if (over) at = last;
    if (wave == at) {
        seen = before;
        int found = -1, final_one = -1;
        if (over) run = 0.0;
        for (int i0 = lo; i0 < hi && found < 0; i0 += 64) {
            double w = step(i0 + lane, &seen), s = w;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const double y = __shfl_up(s, o);
                if (lane >= o) s += y;
            }
            const unsigned long long kb = __ballot(w > 0.0), hit = __ballot(w > 0.0 && run + s > goal);
            if (kb) final_one = i0 + 63 - __clzll(kb);
            if (hit && !over) found = i0 + __ffsll((unsigned long long) hit) - 1;
            run += __shfl(s, 63);
        }
        if (lane == 0) sh.token = found >= 0 ? found : final_one;
    }
    __syncthreads();
    return sh.token;
}

constexpr int SLICE = 4096, SLICE_THREADS = 256, MAX_SLICES = 64;
constexpr int BINS = 1024, LIST = SLICE, NARROW = 3000;
constexpr int GROUPS = SLICE_THREADS;   // 16-element groups of a slice: thread t's, elements 4t + 1024j + {0 .. 3}

// Bins in the order of values: 32 to a power of two from 2^-8 to 2^8, for both signs.
constexpr int BIN_BASE = (127 - 8) << 5;
JAMHIP_DEV int bin_of(uint32_t key) {
    const uint32_t a = (key & 0x80000000u ? key : ~key) & 0x7FFFFFFFu;
    const int m = clampi((int) (a >> 18) - BIN_BASE, 0, BINS / 2 - 1);
    return key & 0x80000000u ? BINS / 2 + m : BINS / 2 - 1 - m;
}
// the smallest key of a bin
JAMHIP_DEV uint32_t bin_first(int b) {
    if (b <= 0) return 0;
    if (b >= BINS / 2) return b == BINS / 2 ? 0x80000000u : 0x80000000u | (uint32_t) (b - BINS / 2 + BIN_BASE) << 18;
    return ~(0x80000000u | (((uint32_t) (BINS / 2 - 1 - b + 1 + BIN_BASE) << 18) - 1));
}

struct SliceStat {
    double zt;       // sum of exp((x - max) / t) of what is in no bin (a row without filters: of all)
    double z1;       // sum of exp(x - max)
    uint32_t key;    // of the largest
    int idx;         // its first index
};

struct SampleWork {
    SliceStat* stat;            // [row][slice]
    uint32_t* group;            // [row][slice][GROUPS] largest keys
    unsigned long long* hist;   // [row][slice][BINS] of the bin and those above: weights relative to the slice's largest, times 2^50, of what may be kept
    int row0, slices;
};

// What the second launch needs of a row.
enum RowWay { GREEDY, TOP_K, CUT, OPEN };
JAMHIP_DEV RowWay way_of(const RowParams& r, int n) {
    if (!(r.t > 0.0f)) return GREEDY;
    if (r.k > 0 && r.k < n) return TOP_K;
    return r.p < 1.0 || r.min_p > 0.0 ? CUT : OPEN;
}

constexpr double HIST_UNIT = 1125899906842624.0;   // 2^50: 4096 weights of at most 1 stay below 2^63

// Four logits from i on. Loads are never behind a branch, so that several are in flight: out of the row they read another
// place of it. row_end() then makes NaN of what is past the end (and reads the row's last, partial four again). VEC: vocab >= 4.
template <bool VEC> JAMHIP_DEV float4_t load4(const float* x, int i, int n) {
    if constexpr (VEC) {
        return *reinterpret_cast<const float4_t*>(x + min(i, (n - 4) & ~3));
    } else {
        float4_t v;
#pragma unroll
        for (int c = 0; c < 4; c++) v[c] = x[min(i + c, n - 1)];
        return v;
    }
}
JAMHIP_DEV void row_end(float4_t& v, const float* x, int i, int n) {
    if (i + 4 > n)
#pragma unroll
        for (int c = 0; c < 4; c++) v[c] = i + c < n ? x[i + c] : __builtin_nanf("");
}

template <bool VEC> __global__ void __launch_bounds__(SLICE_THREADS) sample_slice_kernel(Sample g, SampleWork work) {
    __shared__ unsigned long long hist[BINS];
    __shared__ double pow[64];
    __shared__ uint32_t wkey[4];
    __shared__ int widx[4];
    __shared__ double w1[4], wt[4];
    const int row = work.row0 + blockIdx.y, slice = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = g.vocab, first = slice * SLICE + 4 * tid;
    const float* x = g.logits + (int64_t) row * g.ld;
    float4_t v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = load4<VEC>(x, first + 1024 * j, n);
    const RowParams rp = params_of(g, row);
    const double power = POW[lane];
    uint32_t key[16];   // 0 past the row's end
    float val[16];      // -Inf there
#pragma unroll
    for (int j = 0; j < 4; j++) {
        row_end(v[j], x, first + 1024 * j, n);
#pragma unroll
        for (int c = 0; c < 4; c++) {
            key[4 * j + c] = first + 1024 * j + c < n ? key_of(v[j][c]) : 0;
            val[4 * j + c] = v[j][c] == v[j][c] ? v[j][c] : -__builtin_inff();
        }
    }
    if (tid < 64) pow[tid] = power;
    const RowWay way = way_of(rp, g.vocab);
    if (way == CUT)
        for (int b = tid; b < BINS; b += SLICE_THREADS) hist[b] = 0;
    uint32_t bk = 0;
    int bi = 0;
#pragma unroll
    for (int i = 0; i < 16; i++)
        if (key[i] > bk) bk = key[i], bi = first + 1024 * (i / 4) + i % 4;
    const int64_t at = (int64_t) blockIdx.y * work.slices + slice;
    work.group[at * GROUPS + tid] = bk;
    wave_largest(&bk, &bi);
    if (lane == 0) wkey[wave] = bk, widx[wave] = bi;
    __syncthreads();
    bk = wkey[0], bi = widx[0];
#pragma unroll
    for (int i = 1; i < 4; i++)
        if (wkey[i] > bk || (wkey[i] == bk && widx[i] < bi)) bk = wkey[i], bi = widx[i];
    // f32 weights for the log probability: their error, 2^-23 and that of (x - max) · log2 e, is small where they are large
    const float ftop = of_key(bk);
    float s1 = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const float e = __builtin_amdgcn_exp2f((val[i] - ftop) * 1.44269504088896340736f);
        s1 += val[i] == ftop ? 1.0f : e;
    }
    double z1 = wave_sum_f64((double) s1), zt = 0.0;
    if (way == CUT || way == OPEN) {
        const double top = (double) ftop, inv_t = 1.0 / (double) rp.t;
        // What cannot be kept goes into no bin. A kept value has at least min_p of the largest's weight, which is at least the
        // slice's largest's; and top-p's cut has at least (1 - p) / vocab of the whole sum, since what lies below it is at
        // most that often as much and 1 - p of the sum. With min-p alone it need not be summed either.
        const double least = way == OPEN ? 2.0 : fmax(rp.p < 1.0 ? (1.0 - rp.p) / (double) g.vocab * (1.0 - 1e-9) : 0.0, rp.min_p * (1.0 - 1e-9));
        const bool sums = way == OPEN || rp.p < 1.0;
        const float far = sums || rp.min_p <= 0.0 ? __builtin_inff() : 1.001f * rp.t * -__logf((float) rp.min_p) + 1e-3f * rp.t;
        double wt[16];
        if (sums) {
#pragma unroll
            for (int i = 0; i < 16; i++) wt[i] = weight(top, val[i], inv_t, pow);
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) wt[i] = __any(!(ftop - val[i] > far)) ? weight(top, val[i], inv_t, pow) : 0.0;
        }
#pragma unroll
        for (int i = 0; i < 16; i++) {
            if (wt[i] >= least) atomicAdd(&hist[bin_of(key[i])], (unsigned long long) (wt[i] * HIST_UNIT));
            zt += wt[i] < least ? wt[i] : 0.0;
        }
        zt = wave_sum_f64(sums ? zt : 0.0);
    }
    if (lane == 0) w1[wave] = z1, wt[wave] = zt;
    __syncthreads();
    if (tid == 0) {
        SliceStat s;
        s.z1 = (w1[0] + w1[1]) + (w1[2] + w1[3]);
        s.zt = (wt[0] + wt[1]) + (wt[2] + wt[3]);
        s.key = bk, s.idx = bi;
        work.stat[at] = s;
    }
    if (way == CUT) {   // running sums from the largest values down
        unsigned long long part[BINS / SLICE_THREADS], mine = 0;
#pragma unroll
        for (int k = 0; k < BINS / SLICE_THREADS; k++) part[k] = mine += hist[BINS - 1 - (BINS / SLICE_THREADS * tid + k)];
        unsigned long long run = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned long long y = __shfl_up(run, o);
            if (lane >= o) run += y;
        }
        __syncthreads();
        if (lane == 63) hist[wave] = run;
        __syncthreads();
        run -= mine;
        for (int i = 0; i < wave; i++) run += hist[i];
#pragma unroll
        for (int k = 0; k < BINS / SLICE_THREADS; k++) work.hist[at * BINS + BINS - 1 - (BINS / SLICE_THREADS * tid + k)] = run + part[k];
    }
}

struct PickLds {
    unsigned long long list[LIST];
    double w[LIST];                               // weights of the list's elements, or of a slice's
    union {
        uint16_t pass[MAX_SLICES * GROUPS];       // groups that may hold some
        struct {                                  // narrow()'s
            unsigned long long sub[BINS], few[NARROW];
        };
    };
    GeneralLds general;
    double pow[64];
    double scan[SM_WAVES];
    int iscan[SM_WAVES];
    double factor[MAX_SLICES], sum[MAX_SLICES];   // exp((slice max - top) / t); kept sums
    unsigned long long bound[MAX_SLICES];
    uint32_t key[MAX_SLICES];
    int n, bin, at, token, rank;
    double above, base;
};

// Running sum over the lanes: shifts by 1, 2, 4 and 8 within rows of 16, then each row's last to the next rows.
JAMHIP_DEV double wave_scan(double v) {
    v += dpp_f64<0x111>(v);
    v += dpp_f64<0x112>(v);
    v += dpp_f64<0x114>(v);
    v += dpp_f64<0x118>(v);
    v += dpp_f64<0x142, 0xA>(v);
    v += dpp_f64<0x143, 0xC>(v);
    return v;
}
JAMHIP_DEV int wave_scan(int v) {
    v += dpp_int<0x111>(v);
    v += dpp_int<0x112>(v);
    v += dpp_int<0x114>(v);
    v += dpp_int<0x118>(v);
    v += dpp_int<0x142, 0xA>(v);
    v += dpp_int<0x143, 0xC>(v);
    return v;
}
JAMHIP_DEV int block_scan(int v, int* lds, int* total) {
    const int wave = threadIdx.x >> 6, s = wave_scan(v);
    if ((threadIdx.x & 63) == 63) lds[wave] = s;
    __syncthreads();
    int before = s - v, all = 0;
#pragma unroll
    for (int w = 0; w < SM_WAVES; w++) {
        if (w < wave) before += lds[w];
        all += lds[w];
    }
    __syncthreads();
    *total = all;
    return before;
}

// Sum of v over the threads before this one, in thread order, and over all.
JAMHIP_DEV double block_scan(double v, double* lds, double* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const double s = wave_scan(v);
    if (lane == 63) lds[wave] = s;
    __syncthreads();
    double before = 0.0, all = 0.0;
#pragma unroll
    for (int w = 0; w < SM_WAVES; w++) {
        if (w < wave) before += lds[w];
        all += lds[w];
    }
    __syncthreads();
    *total = all;
    return before + dpp_f64<0x138>(s);   // the lane before's (wave_shr:1; 0 into lane 0)
}

JAMHIP_DEV int wave_below(unsigned long long lanes) {   // how many of them are below this one
    return (int) __builtin_amdgcn_mbcnt_hi((uint32_t) (lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t) lanes, 0));
}

// The indices of those of the elements v, from index i on, that lie in [lo, hi] (NaN does not), onto the wave's list of `held` so far
// (each wave has its own, so that none waits for another's count). Whole waves.
constexpr int WAVE_LIST = 2 * LIST / SM_WAVES;
JAMHIP_DEV void collect4(const float4_t& v, int i, float lo, float hi, uint32_t* list, int* held) {
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const bool in = __builtin_amdgcn_fmed3f(v[c], lo, hi) == v[c];
        const unsigned long long hit = __ballot(in);
        if (!hit) continue;
        const int k = *held + wave_below(hit);
        if (in && k < WAVE_LIST) list[k] = (uint32_t) (i + c);
        *held += __popcll(hit);
    }
}

// Sum of the first m weights before this thread's share of them, `per` in a row.
JAMHIP_DEV double scan_weights(PickLds& sh, int m, int per, double* total) {
    const int tid = threadIdx.x;
    double mine = 0.0;
#pragma unroll 1
    for (int e = tid * per; e < min(m, (tid + 1) * per); e++) mine += sh.w[e];
    return block_scan(mine, sh.scan, total);
}

// The weights of the sorted list's first m, and how many are kept: those before which, with `above` before them all, less than
// goal has been summed, and that are at least min_p; the row's largest in any case. p > 0: goal is p times their sum.
JAMHIP_DEV int kept_of(PickLds& sh, int m, double top, double inv_t, const RowParams& rp, double above, double goal, double p,
                       unsigned long long first) {
    const int tid = threadIdx.x, per = (m + SM_THREADS - 1) / SM_THREADS;
#pragma unroll 1
    for (int e = tid; e < m; e += SM_THREADS) sh.w[e] = weight(top, of_key(pair_key(sh.list[e])), inv_t, sh.pow);
    if (tid == 0) sh.n = 0;
    __syncthreads();
    double total;
    double run = above + scan_weights(sh, m, per, &total);
    if (p > 0.0) goal = p * total;
    int kept = 0;
#pragma unroll 1
    for (int e = tid * per; e < min(m, (tid + 1) * per); e++) {
        const double w = sh.w[e];
        if ((run < goal && w >= rp.min_p) || sh.list[e] == first) kept++;
        run += w;
    }
    kept = wave_sum_int(kept);
    if (kept && (tid & 63) == 0) atomicAdd(&sh.n, kept);
    __syncthreads();
    const int n = sh.n;
    __syncthreads();
    return n;
}

// A bin of too many elements to sort by counting: a histogram of 1024 parts of it finds the one in which the running sum reaches
// the goal, which becomes the list (its length is returned, what is summed before it goes to above). Elements above that
// part are kept and go to their slices' sums; *cut is the least pair that is surely kept (0: none). -1: still too many.
JAMHIP_DEV int narrow(PickLds& sh, int found, double top, double inv_t, double min_p, int bin, unsigned long long first, double goal,
                      double* above, unsigned long long* cut) {
    const int tid = threadIdx.x, lane = tid & 63;
    const uint32_t k0 = bin_first(bin), range = (bin + 1 < BINS ? bin_first(bin + 1) : 0xFFFFFFFFu) - k0;
    const int shift = max(0, 32 - __clz((int) (range - 1)) - 10);
    auto part = [&](unsigned long long pair) { return (int) ((pair_key(pair) - k0) >> shift); };   // 0 .. 1023
#pragma unroll
    for (int i = 0; i < BINS / SM_THREADS; i++) sh.sub[tid + SM_THREADS * i] = 0;
    if (tid == 0) sh.at = -1, sh.n = 0;
    __syncthreads();
#pragma unroll 1
    for (int e = tid; e < found; e += SM_THREADS) {
        const unsigned long long v = sh.list[e];
        double w = weight(top, of_key(pair_key(v)), inv_t, sh.pow);
        if (w < min_p && v != first) w = 0.0;
        sh.w[e] = w;
        if (w > 0.0) atomicAdd(&sh.sub[part(v)], (unsigned long long) (w * HIST_UNIT));
    }
    __syncthreads();
    constexpr int BPT = BINS / SM_THREADS;
    const int last = BINS - 1 - BPT * tid;
    double s[BPT], mine = 0.0, total;
#pragma unroll
    for (int k = 0; k < BPT; k++) mine += s[k] = (double) sh.sub[last - k] * (1.0 / HIST_UNIT);
    double run = *above + block_scan(mine, sh.scan, &total);
#pragma unroll
    for (int k = 0; k < BPT; k++) {
        if (run < goal && run + s[k] >= goal) sh.at = last - k, sh.above = run;   // one part's
        run += s[k];
    }
    __syncthreads();
    const int at = sh.at;   // -1: all of them are kept
    unsigned long long least = ~0ull;
#pragma unroll 1
    for (int e = tid; e < found; e += SM_THREADS) {
        const unsigned long long v = sh.list[e];
        const double w = sh.w[e];
        if (!(w > 0.0)) continue;
        const int p = part(v);
        if (p > at) {
            least = min(least, v);
            atomicAdd(&sh.bound[pair_idx(v) / SLICE], (unsigned long long) (w * HIST_UNIT));
        } else if (p == at) {
            const int k = atomicAdd(&sh.n, 1);
            if (k < NARROW) sh.few[k] = v;
        }
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned long long y = (unsigned long long) __shfl_xor((int) (least >> 32), o) << 32 | (uint32_t) __shfl_xor((int) least, o);
        least = min(least, y);
    }
    unsigned long long* const all = reinterpret_cast<unsigned long long*>(sh.scan);   // past their last use
    if (lane == 0) all[tid >> 6] = least;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SM_WAVES; i++) least = min(least, all[i]);
    *cut = least == ~0ull ? 0 : least;
    const int left = sh.n;
    if (at >= 0) *above = sh.above;
    __syncthreads();
    if (left > NARROW) return -1;
#pragma unroll 1
    for (int e = tid; e < left; e += SM_THREADS) sh.list[e] = sh.few[e];
    __syncthreads();
    return left;
}

// The token among a thread's weights of(i), i < count, at places first + i, with `run` summed before them: the first place whose
// running sum exceeds goal, else the last with a weight; -1 if none has. UNROLL: count, where it is fixed.
template <int UNROLL, typename W> JAMHIP_DEV int pick(PickLds& sh, W&& of, int first, int count, double run, double goal) {
    const int lane = threadIdx.x & 63;
    if (threadIdx.x == 0) sh.token = INT32_MAX, sh.at = -1;
    __syncthreads();
    int hit = INT32_MAX, last = -1;
#pragma unroll UNROLL
    for (int i = 0; i < count; i++) {
        const double w = of(i);
        run += w;
        if (w > 0.0) {
            last = first + i;
            if (hit == INT32_MAX && run > goal) hit = first + i;
        }
    }
    // the first of the hits, and the last with a weight: one lane's of a wave, one atomic each
    const unsigned long long hits = __ballot(hit != INT32_MAX), any = __ballot(last >= 0);
    if (hits && lane == __ffsll(hits) - 1) atomicMin(&sh.token, hit);
    if (any && lane == 63 - __clzll(any)) atomicMax(&sh.at, last);
    __syncthreads();
    return sh.token != INT32_MAX ? sh.token : sh.at;
}

// The token and its key, or -1 where the cut is not among few enough elements to sort.
template <bool VEC> JAMHIP_DEV int pick_row(const Sample& g, const SampleWork& w, int row, const RowParams& rp, RowWay way, uint32_t bk,
                                            int bi, PickLds& sh, uint32_t* token_key) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = g.vocab, S = w.slices;
    const float* x = g.logits + (int64_t) row * g.ld;
    const double top = (double) of_key(bk), inv_t = 1.0 / (double) rp.t;
    const unsigned long long first = pair_of(bk, bi);
    // the largest of 16 elements each, four groups in a row a register
    const uint4_t* groups = reinterpret_cast<const uint4_t*>(w.group + (int64_t) blockIdx.x * S * GROUPS);
    constexpr int PER = MAX_SLICES * GROUPS / 4 / SM_THREADS;
    uint4_t mine[PER];
    uint32_t coarse[PER];
    if (way != OPEN) {
#pragma unroll
        for (int i = 0; i < PER; i++) mine[i] = tid + SM_THREADS * i < S * GROUPS / 4 ? groups[tid + SM_THREADS * i] : uint4_t{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < PER; i++) coarse[i] = max(max(mine[i][0], mine[i][1]), max(mine[i][2], mine[i][3]));
    }
    // The elements in [lo, hi] onto sh.list, and how many they are; more than LIST are not kept, and LIST + 1 is returned. Where fewer than half
    // of the groups reach `bound`, their elements alone are read, four a thread and load, else the row as it lies.
    auto gather = [&](uint32_t bound, float lo, float hi) -> int {
        unsigned long long hits = 0;
#pragma unroll
        for (int i = 0; i < PER; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) hits |= (unsigned long long) (mine[i][c] >= bound) << (4 * i + c);
        int held;
        int to = block_scan(__popcll(hits), sh.iscan, &held);
        const bool some = 8 * held < (n + 3) / 4;
        if (some)
            for (; hits; hits &= hits - 1) {
                const int b = __ffsll(hits) - 1;
                sh.pass[to++] = (uint16_t) (4 * (tid + SM_THREADS * (b / 4)) + b % 4);
            }
        __syncthreads();
        uint32_t* const list = reinterpret_cast<uint32_t*>(sh.w) + wave * WAVE_LIST;
        int got = 0;
        if (some) {
            auto place = [&](int e) {
                const int p = sh.pass[min(e / 4, held - 1)];
                return e < 4 * held ? p / GROUPS * SLICE + 4 * (p % GROUPS) + 1024 * (e % 4) : n;
            };
            int e0 = 0;
            for (; e0 + 4 * SM_THREADS <= 4 * held; e0 += 4 * SM_THREADS) {   // four loads in flight
                float4_t v[4];
                int at[4];
#pragma unroll
                for (int k = 0; k < 4; k++) at[k] = place(e0 + SM_THREADS * k + tid);
#pragma unroll
                for (int k = 0; k < 4; k++) v[k] = load4<VEC>(x, at[k], n);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    row_end(v[k], x, at[k], n);
                    collect4(v[k], at[k], lo, hi, list, &got);
                }
            }
#pragma unroll 1
            for (; e0 < 4 * held; e0 += SM_THREADS) {
                const int at = place(e0 + tid);
                float4_t v = load4<VEC>(x, at, n);
                row_end(v, x, at, n);
                collect4(v, at, lo, hi, list, &got);
            }
        } else {
            for (int i0 = 0; i0 < n; i0 += 4 * 16 * SM_THREADS) {   // 16 loads in flight
                float4_t v[16];
#pragma unroll
                for (int k = 0; k < 16; k++) v[k] = load4<VEC>(x, i0 + 4 * (SM_THREADS * k + tid), n);
#pragma unroll
                for (int k = 0; k < 16; k++) row_end(v[k], x, i0 + 4 * (SM_THREADS * k + tid), n);
                uint32_t half[2] = {0, 0};   // the thread's 64 elements, the first one's bit at the top
#pragma unroll
                for (int e = 0; e < 64; e++) {
                    const float a = v[e / 4][e % 4];
                    half[e / 32] = half[e / 32] << 1 | (__builtin_amdgcn_fmed3f(a, lo, hi) == a ? 1u : 0u);
                }
                unsigned long long bits = (unsigned long long) half[0] << 32 | half[1];
                for (unsigned long long some = __ballot(bits != 0); some; some = __ballot(bits != 0)) {   // one of each lane's a round
                    const int e = __clzll(bits | 1), k = got + wave_below(some);
                    if (bits && k < WAVE_LIST) list[k] = (uint32_t) (i0 + 4 * (SM_THREADS * (e / 4) + tid) + e % 4);
                    got += __popcll(some);
                    if (bits) bits &= ~(1ull << (63 - e));
                }
            }
        }
        if (lane == 0) sh.iscan[wave] = got;
        __syncthreads();
        int first_of = 0, all = 0, most = 0;
#pragma unroll
        for (int i = 0; i < SM_WAVES; i++) {
            const int c = sh.iscan[i];
            if (i < wave) first_of += c;
            all += c, most = max(most, c);
        }
        if (most > WAVE_LIST || all > LIST) return LIST + 1;
#pragma unroll 2
        for (int e = lane; e < got; e += 64) {
            const int i = (int) list[e];
            sh.list[first_of + e] = pair_of(key_of(x[i]), i);
        }
        __syncthreads();
        return all;
    };
    uint32_t bound = 0;
    int bin = 0, found = 0;
    double above = 0.0, goal = __builtin_inf();
    const unsigned long long* hist = w.hist + (int64_t) blockIdx.x * S * BINS;
    constexpr double unit = 1.0 / HIST_UNIT;
    if (way == TOP_K) {
        // The k-th largest of the largest of every 64 (for large k: 16) elements lies in the bin in which their number, from
        // the top, reaches k: at least k elements are not below that bin's first value
        // Of every 64 there are S · GROUPS / 4, of which k has to leave the bound well above their smallest: 128256 logits, one row, by 64 /
        // by 16 in us: k = 50 14.5 / 16.0, 256 27.3 / 28.9, 1024 74.9 / 73.5, 1025 92.9 / 90.6, 2048 741 / 137; 32000: 512 99 / 43
        const bool fine = rp.k > S * GROUPS / 8;
        int* const count = reinterpret_cast<int*>(sh.w);
#pragma unroll
        for (int i = 0; i < BINS / SM_THREADS; i++) count[tid + SM_THREADS * i] = 0;
        if (tid == 0) sh.bin = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; i++) {
            if (fine) {
#pragma unroll
                for (int c = 0; c < 4; c++)
                    if (mine[i][c]) atomicAdd(&count[bin_of(mine[i][c])], 1);
            } else if (coarse[i]) {
                atomicAdd(&count[bin_of(coarse[i])], 1);
            }
        }
        __syncthreads();
        constexpr int BPT = BINS / SM_THREADS;
        const int last = BINS - 1 - BPT * tid;
        int c[BPT], sum = 0, total;
#pragma unroll
        for (int i = 0; i < BPT; i++) sum += c[i] = count[last - i];
        int run = block_scan(sum, sh.iscan, &total);
#pragma unroll
        for (int i = 0; i < BPT; i++) {
            if (run < rp.k && run + c[i] >= rp.k) sh.bin = last - i;
            run += c[i];
        }
        __syncthreads();
        bound = bin_first(sh.bin);
        bound = max(bound, key_of(-__builtin_inff()));   // 0 stands for no element
        found = gather(bound, of_key(bound), __builtin_inff());
    } else {
        // slices' weights are relative to their own largest
        if (tid < S) sh.factor[tid] = weight(top, of_key(sh.key[tid]), inv_t, sh.pow), sh.bound[tid] = 0;
        if (tid == 0) sh.bin = 0, sh.rank = BINS, sh.n = 0;
        __syncthreads();
        if (way == CUT) {
            constexpr int BPT = BINS / SM_THREADS;   // a thread's bins, in a row, from the largest values down: last, last - 1, ..
            const int last = BINS - 1 - BPT * tid;
            double s[BPT] = {};
#pragma unroll 8
            for (int i = 0; i < S; i++) {
                const double f = sh.factor[i];
                const ulong2 u = *reinterpret_cast<const ulong2*>(hist + i * BINS + last - 3), v = *reinterpret_cast<const ulong2*>(hist + i * BINS + last - 1);
                s[0] += (double) v.y * f, s[1] += (double) v.x * f, s[2] += (double) u.y * f, s[3] += (double) u.x * f;
            }
            static_assert(BPT == 4, "two loads of two bins");
#pragma unroll
            for (int k = 0; k < BPT; k++) sh.w[last - k] = s[k] *= unit;
            __syncthreads();
            above = tid ? sh.w[last + 1] : 0.0;
            double total = sh.w[0];
            if (wave == 0) {   // what the slices left out of their bins
                const double rest = lane < S ? w.stat[(int64_t) blockIdx.x * S + lane].zt * sh.factor[lane] : 0.0;
                sh.base = lane_f64(wave_scan(rest), 63);
            }
            __syncthreads();
            total += sh.base;
            if (rp.p < 1.0) goal = fmax(rp.p * total, 1e-300);
            // the bin in which the running sum reaches the goal; min-p's cut falls into the one below the lowest whose every
            // value passes. The higher one cuts
            int enough = 0;
            double run = above;
#pragma unroll
            for (int k = 0; k < BPT; k++) {
                if (run < goal && s[k] >= goal) sh.bin = last - k;   // one bin's
                run = s[k];
                if (rp.min_p > 0.0) enough += __popcll(__ballot(weight(top, of_key(bin_first(last - k)), inv_t, sh.pow) >= rp.min_p));
            }
            if (lane == 0 && enough) atomicSub(&sh.rank, enough);
            __syncthreads();
            bin = min(max(sh.bin, rp.min_p > 0.0 ? sh.rank - 1 : 0), bin_of(bk));
#pragma unroll
            for (int k = 0; k < BPT; k++) {
                if (last - k == bin) sh.above = above;
                above = s[k];
            }
            // its largest value; below the first bin from 0 on that is the one before -0, which is a 0
            const uint32_t next = bin + 1 < BINS ? bin_first(bin + 1) : key_of(__builtin_inff()) + 1;
            found = gather(bin_first(bin), bin ? of_key(bin_first(bin)) : -__builtin_inff(), of_key(next - (bin + 1 == BINS / 2 ? 2 : 1)));
            above = sh.above;
        }
    }
    unsigned long long cut = 0;   // kept: pairs not below it
    if (way != OPEN) {
        if (found > LIST || (way == TOP_K && found < rp.k)) return -1;
        if (way == CUT && found > SM_THREADS) {
            found = narrow(sh, found, top, inv_t, rp.min_p, bin, first, goal, &above, &cut);
            if (found < 0) return -1;
        }
        sort_falling(sh.list, found);
        const int m = kept_of(sh, way == TOP_K ? rp.k : found, top, inv_t, rp, above, goal, way == TOP_K && rp.p < 1.0 ? fmax(rp.p, 1e-300) : 0.0,
                              first);
        if (way == TOP_K) {
            order_by_index(sh.list, m);
            const int per = (m + SM_THREADS - 1) / SM_THREADS, from = min(m, tid * per), count = min(m, from + per) - from;
            auto of = [&](int i) { return sh.w[(uint32_t) sh.list[from + i]]; };
            double mine_sum = 0.0, total;
#pragma unroll 1
            for (int i = 0; i < count; i++) mine_sum += of(i);
            const double run = block_scan(mine_sum, sh.scan, &total);
            const int e = pick<1>(sh, of, from, count, run, rp.u * total);
            const int token = (int) ~(uint32_t) (sh.list[e] >> 32);
            *token_key = key_of(x[token]);
            return token;
        }
        if (m > 0) cut = sh.list[m - 1];
        else if (cut == 0) cut = (unsigned long long) bin_first(bin + 1) << 32;
        // the slices' kept sums: their bins above, and what is kept of this one
#pragma unroll 1
        for (int e = tid; e < m; e += SM_THREADS)
            atomicAdd(&sh.bound[pair_idx(sh.list[e]) / SLICE], (unsigned long long) (sh.w[e] * HIST_UNIT));
        if (tid < S) sh.sum[tid] = bin + 1 < BINS ? (double) hist[tid * BINS + bin + 1] * unit * sh.factor[tid] : 0.0;
        __syncthreads();
        if (tid < S) sh.sum[tid] += (double) sh.bound[tid] * unit;
    } else if (tid < S) {
        sh.sum[tid] = w.stat[(int64_t) blockIdx.x * S + tid].zt * sh.factor[tid];
    }
    __syncthreads();
    if (wave == 0) {   // the slice in which the running sum passes u times all
        const double v = lane < S ? sh.sum[lane] : 0.0, s = wave_scan(v), all = lane_f64(s, 63);
        const unsigned long long hit = __ballot(v > 0.0 && s > rp.u * all), any = __ballot(v > 0.0);
        const int at = hit ? __ffsll(hit) - 1 : 63 - __clzll(any);
        if (lane == 0) sh.bin = at, sh.base = at ? lane_f64(s, at - 1) : 0.0, sh.above = all;
    }
    __syncthreads();
    // 16 elements in a row a thread
    const int start = sh.bin * SLICE, from = start + 16 * tid;
    double wt[16], mine_sum = 0.0, total;
    float4_t quad[4];
#pragma unroll
    for (int j = 0; j < 4; j++) quad[j] = load4<VEC>(x, from + 4 * j, n);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float4_t v = quad[j];
        row_end(v, x, from + 4 * j, n);
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const int i = from + 4 * j + c;
            const float a = v[c] == v[c] ? v[c] : -__builtin_inff();
            const double w1 = weight(top, a, inv_t, sh.pow);
            wt[4 * j + c] = w1 * (i < n && pair_of(key_of(a), i) >= cut ? 1.0 : 0.0);
            mine_sum += wt[4 * j + c];
        }
    }
    const int e = pick<16>(sh, [&](int i) { return wt[i]; }, 16 * tid, 16, sh.base + block_scan(mine_sum, sh.scan, &total), rp.u * sh.above);
    if (e < 0) return -1;
    *token_key = key_of(x[start + e]);
    return start + e;
}

// A row's largest, log normaliser and token from its slices.
template <bool VEC> __global__ void __launch_bounds__(SM_THREADS) sample_pick_kernel(Sample g, SampleWork w) {
    __shared__ PickLds sh;
    const int row = w.row0 + blockIdx.x, tid = threadIdx.x, lane = tid & 63, S = w.slices;
    const SliceStat st = w.stat[(int64_t) blockIdx.x * S + min(lane, S - 1)];
    const RowParams rp = params_of(g, row);
    const double power = POW[lane];
    uint32_t bk = st.key;
    int bi = st.idx;
    wave_largest(&bk, &bi);
    const double top = (double) of_key(bk);
    if (tid < 64) sh.pow[tid] = power;
    if (tid < S) sh.key[tid] = st.key;
    __syncthreads();
    const double z = wave_sum_f64(lane < S ? st.z1 * weight(top, of_key(st.key), 1.0, sh.pow) : 0.0);
    const bool none = bk <= key_of(-__builtin_inff());
    int token = bi;
    uint32_t token_key = bk;
    if (!none && rp.t > 0.0f) {
        token = pick_row<VEC>(g, w, row, rp, way_of(rp, g.vocab), bk, bi, sh, &token_key);
        if (token < 0) {
            token = sample_general(g, row, bk, rp, sh.general, sh.pow);
            token_key = key_of(g.logits[(int64_t) row * g.ld + token]);
        }
    }
    if (tid == 0) {
        g.token[row] = token;
        if (g.logprob != nullptr) {
            const double v = (double) of_key(token_key);
            g.logprob[row] = none ? -__builtin_inff() : (float) ((v == top ? 0.0 : v - top) - log(z));
        }
    }
}

// Rows of more slices than a wave has lanes: the largest and the sum by one workgroup, the rest the general way.
__global__ void __launch_bounds__(SM_THREADS) sample_long_kernel(Sample g) {
    __shared__ GeneralLds sh;
    __shared__ double pow[64];
    __shared__ int widx[SM_WAVES];
    __shared__ uint32_t wkey[SM_WAVES];
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = g.vocab;
    const float* x = g.logits + (int64_t) row * g.ld;
    if (tid < 64) pow[tid] = POW[tid];
    uint32_t bk = 0;
    int bi = 0;
    for (int i = tid; i < n; i += SM_THREADS) {
        const uint32_t k = key_of(x[i]);
        if (k > bk) bk = k, bi = i;
    }
    wave_largest(&bk, &bi);
    if (lane == 0) wkey[wave] = bk, widx[wave] = bi;
    __syncthreads();
    bk = wkey[0], bi = widx[0];
    for (int w = 1; w < SM_WAVES; w++)
        if (wkey[w] > bk || (wkey[w] == bk && widx[w] < bi)) bk = wkey[w], bi = widx[w];
    const double top = (double) of_key(bk);
    double z = 0.0;
    for (int i = tid; i < n; i += SM_THREADS) z += weight(top, of_key(key_of(x[i])), 1.0, pow);
    z = wave_sum_f64(z);
    if (lane == 0) sh.wsum[wave] = z;
    __syncthreads();
    z = 0.0;
    for (int w = 0; w < SM_WAVES; w++) z += sh.wsum[w];
    __syncthreads();
    const RowParams rp = params_of(g, row);
    const bool none = bk <= key_of(-__builtin_inff());
    int token = bi;
    if (!none && rp.t > 0.0f) token = sample_general(g, row, bk, rp, sh, pow);
    if (tid == 0) {
        g.token[row] = token;
        if (g.logprob != nullptr) {
            const double v = (double) of_key(key_of(x[token]));
            g.logprob[row] = none ? -__builtin_inff() : (float) ((v == top ? 0.0 : v - top) - log(z));
        }
    }
}

// Rows of one pair of launches: their workspace is 9 KB a slice, 0.6 MB for the longest row.
constexpr int ROWS_AT_ONCE = 256;

size_t slice_bytes() { return sizeof(SliceStat) + GROUPS * sizeof(uint32_t) + BINS * sizeof(unsigned long long); }

}  // namespace

size_t sample_workspace(const Sample& g) {
    const int64_t slices = ((int64_t) g.vocab + SLICE - 1) / SLICE;
    if (slices > MAX_SLICES) return 0;
    return (size_t) (g.rows < ROWS_AT_ONCE ? g.rows : ROWS_AT_ONCE) * slices * slice_bytes();
}

hipError_t launch_sample(const Sample& g, void* work, hipStream_t st) {
    if (g.rows <= 0) return hipSuccess;
    const int64_t slices = ((int64_t) g.vocab + SLICE - 1) / SLICE;
    if (slices > MAX_SLICES) {
        sample_long_kernel<<<g.rows, SM_THREADS, 0, st>>>(g);
        return hipGetLastError();
    }
    const int rows = g.rows < ROWS_AT_ONCE ? g.rows : ROWS_AT_ONCE;
    SampleWork w;
    w.slices = (int) slices;
    w.hist = static_cast<unsigned long long*>(work);
    w.stat = reinterpret_cast<SliceStat*>(w.hist + (size_t) rows * slices * BINS);
    w.group = reinterpret_cast<uint32_t*>(w.stat + (size_t) rows * slices);
    const bool vec = (reinterpret_cast<uintptr_t>(g.logits) & 15) == 0 && g.ld % 4 == 0 && g.vocab >= 4;
    for (w.row0 = 0; w.row0 < g.rows; w.row0 += rows) {
        const int n = g.rows - w.row0 < rows ? g.rows - w.row0 : rows;
        const dim3 grid((uint32_t) slices, n);
        if (vec) {
            sample_slice_kernel<true><<<grid, SLICE_THREADS, 0, st>>>(g, w);
            sample_pick_kernel<true><<<n, SM_THREADS, 0, st>>>(g, w);
        } else {
            sample_slice_kernel<false><<<grid, SLICE_THREADS, 0, st>>>(g, w);
            sample_pick_kernel<false><<<n, SM_THREADS, 0, st>>>(g, w);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace jamhip
