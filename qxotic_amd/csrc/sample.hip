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
// logits, the cut is found digit by digit of the values' order-preserving 32-bit keys from histograms over the whole row.
// Weights are summed in histograms as 64-bit integers, so that the order of the atomics does not matter.
#include "launch.h"

namespace jamhip {

namespace {

constexpr int SM_THREADS = 1024, SM_WAVES = SM_THREADS / 64;

// A larger value has the larger key; NaN counts as -Inf. Both zeros have one key, as they are equal.
JAMHIP_DEV uint32_t key_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x == 0.0f ? 0.0f : x != x ? -__builtin_inff() : x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
JAMHIP_DEV float of_key(uint32_t k) { return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

JAMHIP_DEV int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }

JAMHIP_DEV double wave_sum_f64(double v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    return v;
}

// e^-y, y >= 0, in 64 bits: y = n · ln 2 - r with ln 2 in two parts, then the Taylor series to r^12, whose first omitted term
// is 0.347^13 / 13!, below 2e-16.
JAMHIP_DEV double exp_neg(double y) {
    y = fmin(y, 800.0);   // e^-800 is 0
    const double n = rint(y * 1.44269504088896340736);
    double r = fma(n, 0.69314718055994528623, -y);
    r = fma(n, 2.3190468138462995584e-17, r);
    double p = 1.0 / 479001600.0;
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, -(int) n);
}

// exp(-(top - x) / t); equal to 1 at the top whatever its value, 0 for -Inf below it
JAMHIP_DEV double weight(double top, float x, double inv_t) {
    return (double) x == top ? 1.0 : exp_neg((top - (double) x) * inv_t);
}

struct RowParams {
    float t;
    int k;
    double p, min_p, u;
};
JAMHIP_DEV RowParams params_of(const Sample& g, int row) {
    RowParams r;
    r.t = g.temperature ? g.temperature[row] : 1.0f;
    r.k = g.top_k ? g.top_k[row] : 0;
    r.p = g.top_p ? (double) g.top_p[row] : 1.0;
    r.min_p = g.min_p ? fmin((double) g.min_p[row], 1.0) : 0.0;
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
JAMHIP_DEV int sample_general(const Sample& g, int row, uint32_t bk, const RowParams& rp, GeneralLds& sh) {
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
    auto fixed = [&](uint32_t key) { return (unsigned long long) (weight(top, of_key(key), inv_t) * unit); };
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
        const double w = weight(top, of_key(key), inv_t);
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
constexpr int BINS = 1024, LIST = 8192;
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
    double zt;       // sum of exp((x - max) / t) (a row without filters)
    double z1;       // sum of exp(x - max)
    uint32_t key;    // of the largest
    int idx;         // its first index
};

struct SampleWork {
    SliceStat* stat;            // [row][slice]
    uint32_t* group;            // [row][slice][GROUPS] largest keys
    unsigned long long* hist;   // [row][slice][BINS] weights relative to the slice's largest, times 2^50
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

// 16 logits of thread t of a slice, as keys; 0 past the row's end.
template <bool VEC> JAMHIP_DEV void slice_keys(const float* x, int first, int n, int t, uint32_t* key) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int i = first + 4 * t + 1024 * j;
        if (VEC && i + 4 <= n) {
            const float4_t v = *reinterpret_cast<const float4_t*>(x + i);
#pragma unroll
            for (int c = 0; c < 4; c++) key[4 * j + c] = key_of(v[c]);
        } else {
#pragma unroll
            for (int c = 0; c < 4; c++) key[4 * j + c] = i + c < n ? key_of(x[i + c]) : 0;
        }
    }
}

template <bool VEC> __global__ void __launch_bounds__(SLICE_THREADS) sample_slice_kernel(Sample g, SampleWork w) {
    __shared__ unsigned long long hist[BINS];
    __shared__ uint32_t wkey[4];
    __shared__ int widx[4];
    __shared__ double w1[4], wt[4];
    const int row = w.row0 + blockIdx.y, slice = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t key[16];
    slice_keys<VEC>(g.logits + (int64_t) row * g.ld, slice * SLICE, g.vocab, tid, key);
    const RowParams rp = params_of(g, row);
    const RowWay way = way_of(rp, g.vocab);
    if (way == CUT)
        for (int b = tid; b < BINS; b += SLICE_THREADS) hist[b] = 0;
    uint32_t bk = 0;
    int bi = 0;
#pragma unroll
    for (int i = 0; i < 16; i++)
        if (key[i] > bk) bk = key[i], bi = slice * SLICE + 4 * tid + 1024 * (i / 4) + i % 4;
    const int64_t at = (int64_t) blockIdx.y * w.slices + slice;
    w.group[at * GROUPS + tid] = bk;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t ok = __shfl_xor(bk, o);
        const int oi = __shfl_xor(bi, o);
        if (ok > bk || (ok == bk && oi < bi)) bk = ok, bi = oi;
    }
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
        const float v = of_key(key[i]);
        s1 += key[i] == 0 ? 0.0f : v == ftop ? 1.0f : __builtin_amdgcn_exp2f((v - ftop) * 1.44269504088896340736f);
    }
    double z1 = wave_sum_f64((double) s1), zt = 0.0;
    if (way == CUT || way == OPEN) {
        const double top = (double) ftop, inv_t = 1.0 / (double) rp.t;
        if (way == OPEN) {
#pragma unroll
            for (int i = 0; i < 16; i++) zt += key[i] == 0 ? 0.0 : weight(top, of_key(key[i]), inv_t);
            zt = wave_sum_f64(zt);
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const unsigned long long v = key[i] == 0 ? 0 : (unsigned long long) (weight(top, of_key(key[i]), inv_t) * HIST_UNIT);
                if (v) atomicAdd(&hist[bin_of(key[i])], v);
            }
        }
    }
    if (lane == 0) w1[wave] = z1, wt[wave] = zt;
    __syncthreads();
    if (tid == 0) {
        SliceStat s;
        s.z1 = (w1[0] + w1[1]) + (w1[2] + w1[3]);
        s.zt = (wt[0] + wt[1]) + (wt[2] + wt[3]);
        s.key = bk, s.idx = bi;
        w.stat[at] = s;
    }
    if (way == CUT)
        for (int b = tid; b < BINS; b += SLICE_THREADS) w.hist[at * BINS + b] = hist[b];
}

struct PickLds {
    unsigned long long list[LIST];
    GeneralLds general;
    double scan[SM_WAVES];
    double factor[MAX_SLICES], sum[MAX_SLICES];   // exp((slice max - top) / t); kept sums
    unsigned long long bound[MAX_SLICES];
    uint32_t key[MAX_SLICES];
    int count[SM_WAVES];
    int n, bin, at, token;
    double above, base;
};

// Sum of v over the threads before this one, in thread order, and over all.
JAMHIP_DEV double block_scan(double v, double* lds, double* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double y = __shfl_up(s, o);
        if (lane >= o) s += y;
    }
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
    const double up = __shfl_up(s, 1);
    return before + (lane ? up : 0.0);
}

// list[0 .. 2^k) in falling order, 2^k >= n, filled up with zeros.
JAMHIP_DEV int sort_falling(unsigned long long* list, int n) {
    int size = 1;
    while (size < n) size <<= 1;
    const int tid = threadIdx.x;
    for (int i = n + tid; i < size; i += SM_THREADS) list[i] = 0;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int p = tid; p < size / 2; p += SM_THREADS) {
                const int a = 2 * p - (p & (j - 1)), b = a + j;   // bit j of a is 0
                const unsigned long long u = list[a], v = list[b];
                if ((u < v) == ((a & k) == 0)) list[a] = v, list[b] = u;
            }
            __syncthreads();
        }
    return size;
}

JAMHIP_DEV unsigned long long pair_of(uint32_t key, int idx) { return (unsigned long long) key << 32 | (uint32_t) ~idx; }
JAMHIP_DEV uint32_t pair_key(unsigned long long p) { return (uint32_t) (p >> 32); }
JAMHIP_DEV int pair_idx(unsigned long long p) { return (int) ~(uint32_t) p; }

// The elements of the row whose largest-of-16 passes `group` and whose key passes `one`, as pairs; how many (the first LIST are held).
template <bool VEC, typename G, typename O>
JAMHIP_DEV int collect(const Sample& g, const SampleWork& w, int row, const uint32_t* groups, PickLds& sh, G&& group, O&& one) {
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < w.slices * GROUPS; i += SM_THREADS) {
        if (!group(groups[i])) continue;
        const int first = i / GROUPS * SLICE, t = i % GROUPS;
        uint32_t key[16];
        slice_keys<VEC>(g.logits + (int64_t) row * g.ld, first, g.vocab, t, key);
#pragma unroll
        for (int j = 0; j < 16; j++)
            if (key[j] && one(key[j])) {
                const int k = atomicAdd(&sh.n, 1);
                if (k < LIST) sh.list[k] = pair_of(key[j], first + 4 * t + 1024 * (j / 4) + j % 4);
            }
    }
    __syncthreads();
    return sh.n;
}

// How many of the sorted list's first m (in falling order) are kept: those before which, with `above` before them all, less
// than `goal` has been summed, and that are at least min_p; the row's largest in any case.
JAMHIP_DEV int kept_of(PickLds& sh, int m, double top, double inv_t, double min_p, double above, double goal, uint32_t bk, int bi) {
    const int tid = threadIdx.x, per = (m + SM_THREADS - 1) / SM_THREADS;
    double mine = 0.0, total;
    for (int e = tid * per; e < min(m, (tid + 1) * per); e++) mine += weight(top, of_key(pair_key(sh.list[e])), inv_t);
    double run = above + block_scan(mine, sh.scan, &total);
    if (tid == 0) sh.n = 0;
    __syncthreads();
    int kept = 0;
    for (int e = tid * per; e < min(m, (tid + 1) * per); e++) {
        const double w = weight(top, of_key(pair_key(sh.list[e])), inv_t);
        if ((run < goal && w >= min_p) || sh.list[e] == pair_of(bk, bi)) kept++;
        run += w;
    }
    if (kept) atomicAdd(&sh.n, kept);
    __syncthreads();
    const int n = sh.n;
    __syncthreads();
    return n;
}

// The token among weights in index order: thread t holds `cnt` of them from w[0] on, at indices idx[..]; `base` is summed before.
// Returns the first whose running sum exceeds goal, else the last with a weight.
template <int CNT>
JAMHIP_DEV int pick(PickLds& sh, const double* w, const int* idx, double base, double goal) {
    double mine = 0.0, total;
#pragma unroll
    for (int i = 0; i < CNT; i++) mine += w[i];
    double run = base + block_scan(mine, sh.scan, &total);
    if (threadIdx.x == 0) sh.token = INT32_MAX, sh.at = -1;
    __syncthreads();
    int hit = INT32_MAX, last = -1;
#pragma unroll
    for (int i = 0; i < CNT; i++) {
        run += w[i];
        if (w[i] > 0.0) {
            last = idx[i];
            if (hit == INT32_MAX && run > goal) hit = idx[i];
        }
    }
    if (hit != INT32_MAX) atomicMin(&sh.token, hit);
    if (last >= 0) atomicMax(&sh.at, last);
    __syncthreads();
    return sh.token != INT32_MAX ? sh.token : sh.at;
}

template <bool VEC> JAMHIP_DEV int pick_row(const Sample& g, const SampleWork& w, int row, const RowParams& rp, RowWay way, uint32_t bk,
                                            int bi, PickLds& sh) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = g.vocab, S = w.slices;
    const uint32_t* groups = w.group + (int64_t) blockIdx.x * S * GROUPS;
    const double top = (double) of_key(bk), inv_t = 1.0 / (double) rp.t;
    if (way == TOP_K) {
        // the k-th largest of the groups' largest, 20 bits of it, two at a time: at least k elements are not below it
        constexpr int PER = MAX_SLICES * GROUPS / SM_THREADS;
        uint32_t mine[PER];
#pragma unroll
        for (int i = 0; i < PER; i++) mine[i] = tid + SM_THREADS * i < S * GROUPS ? groups[tid + SM_THREADS * i] : 0;
        uint32_t bound = 0;
        for (int shift = 30; shift >= 12; shift -= 2) {
            uint32_t c = 0, c3 = 0;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                c += (mine[i] >= (bound | 1u << shift)) + ((mine[i] >= (bound | 2u << shift)) << 16);
                c3 += mine[i] >= (bound | 3u << shift);
            }
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) c += __shfl_xor(c, o), c3 += __shfl_xor(c3, o);
            // two alternating places, so that one barrier a round does
            unsigned long long* const cell = sh.list + (shift & 2 ? SM_WAVES : 0);
            if (lane == 0) cell[wave] = (unsigned long long) c3 << 32 | c;
            __syncthreads();
            int n1 = 0, n2 = 0, n3 = 0;
#pragma unroll
            for (int i = 0; i < SM_WAVES; i++) {
                const unsigned long long v = cell[i];
                n1 += (int) (v & 0xFFFF), n2 += (int) (v >> 16 & 0xFFFF), n3 += (int) (v >> 32);
            }
            bound |= (n3 >= rp.k ? 3u : n2 >= rp.k ? 2u : n1 >= rp.k ? 1u : 0u) << shift;
        }
        __syncthreads();
        const int found = collect<VEC>(g, w, row, groups, sh, [&](uint32_t k) { return k >= bound && k; }, [&](uint32_t k) { return k >= bound; });
        if (found > LIST || found < rp.k) return -1;   // too many to sort
        sort_falling(sh.list, found);
        int m = rp.k;
        {   // the sum of the k
            const int per = (m + SM_THREADS - 1) / SM_THREADS;
            double s = 0.0, total = 0.0;
            if (rp.p < 1.0) {
                for (int e = tid * per; e < min(m, (tid + 1) * per); e++) s += weight(top, of_key(pair_key(sh.list[e])), inv_t);
                (void) block_scan(s, sh.scan, &total);
            }
            if (rp.p < 1.0 || rp.min_p > 0.0)
                m = kept_of(sh, m, top, inv_t, rp.min_p, 0.0, rp.p < 1.0 ? rp.p * total : __builtin_inf(), bk, bi);
        }
        for (int e = tid; e < m; e += SM_THREADS) {   // by index
            const unsigned long long v = sh.list[e];
            sh.list[e] = (unsigned long long) (uint32_t) ~pair_idx(v) << 32 | pair_key(v);
        }
        sort_falling(sh.list, m);
        constexpr int CNT = LIST / SM_THREADS;
        double wt[CNT];
        int idx[CNT];
        const int per = (m + SM_THREADS - 1) / SM_THREADS;
        double s = 0.0, total;
#pragma unroll
        for (int i = 0; i < CNT; i++) {
            const int e = tid * per + i;
            const bool in = i < per && e < m;
            const unsigned long long v = in ? sh.list[e] : 0;
            idx[i] = in ? (int) ~(uint32_t) (v >> 32) : 0;
            wt[i] = in ? weight(top, of_key((uint32_t) v), inv_t) : 0.0;
            s += wt[i];
        }
        (void) block_scan(s, sh.scan, &total);
        return pick<CNT>(sh, wt, idx, 0.0, rp.u * total);
    }

    // CUT and OPEN: slices' weights are relative to their own largest
    if (tid < S) sh.factor[tid] = weight(top, of_key(sh.key[tid]), inv_t), sh.bound[tid] = 0;
    __syncthreads();
    unsigned long long cut = 0;   // kept: pairs not below it
    const unsigned long long* hist = w.hist + (int64_t) blockIdx.x * S * BINS;
    const double unit = 1.0 / HIST_UNIT;
    if (way == CUT) {
        static_assert(BINS == SM_THREADS, "a bin a thread");
        const int b = BINS - 1 - tid;   // from the largest values down
        double s = 0.0, total;
        for (int i = 0; i < S; i++) s += (double) hist[i * BINS + b] * unit * sh.factor[i];
        const double above = block_scan(s, sh.scan, &total), goal = rp.p < 1.0 ? fmax(rp.p * total, 1e-300) : __builtin_inf();
        if (tid == 0) {
            int mb = -1;   // the bin that min-p's cut falls into
            if (rp.min_p > 0.0) {
                auto enough = [&](int k) { return weight(top, of_key(bin_first(k)), inv_t) >= rp.min_p; };
                mb = bin_of(key_of((float) (top + (double) rp.t * log(rp.min_p))));
                while (mb + 1 < BINS && !enough(mb + 1)) mb++;
                while (mb > 0 && enough(mb)) mb--;
                mb = min(mb, bin_of(bk));
            }
            sh.bin = mb;
        }
        __syncthreads();
        // the bin in which the running sum reaches the goal (the last that holds any, should rounding leave it short)
        if (s > 0.0 && above < goal && (above + s >= goal)) atomicMax(&sh.bin, b);
        __syncthreads();
        const int bin = max(sh.bin, 0);
        if (b == bin) sh.above = above;
        __syncthreads();
        const int found = collect<VEC>(g, w, row, groups, sh, [&](uint32_t k) { return bin_of(k) >= bin && k; },
                                       [&](uint32_t k) { return bin_of(k) == bin; });
        if (found > LIST) return -1;
        sort_falling(sh.list, found);
        const int m = kept_of(sh, found, top, inv_t, rp.min_p, sh.above, goal, bk, bi);
        cut = m > 0 ? sh.list[m - 1] : (unsigned long long) bin_first(bin + 1) << 32;
        // the slices' kept sums: their bins above, and what is kept of this one
        for (int e = tid; e < m; e += SM_THREADS) {
            const unsigned long long v = (unsigned long long) (weight(top, of_key(pair_key(sh.list[e])), inv_t) * (HIST_UNIT / 2));
            atomicAdd(&sh.bound[pair_idx(sh.list[e]) / SLICE], v);
        }
        for (int i = wave; i < S; i += SM_WAVES) {
            double v = 0.0;
            for (int k = bin + 1 + lane; k < BINS; k += 64) v += (double) hist[i * BINS + k] * unit;
            v = wave_sum_f64(v);
            if (lane == 0) sh.sum[i] = v * sh.factor[i];
        }
        __syncthreads();
        if (tid < S) sh.sum[tid] += (double) sh.bound[tid] * (2.0 * unit);
    } else if (tid < S) {
        sh.sum[tid] = w.stat[(int64_t) blockIdx.x * S + tid].zt * sh.factor[tid];
    }
    __syncthreads();
    if (wave == 0) {   // the slice in which the running sum passes u times all
        double v = lane < S ? sh.sum[lane] : 0.0, s = v;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double y = __shfl_up(s, o);
            if (lane >= o) s += y;
        }
        const double all = __shfl(s, 63), goal = rp.u * all;
        const unsigned long long hit = __ballot(v > 0.0 && s > goal), any = __ballot(v > 0.0);
        const int at = hit ? __ffsll(hit) - 1 : 63 - __clzll(any);
        const double up = __shfl(s, max(at - 1, 0));
        if (lane == 0) sh.bin = at, sh.base = at ? up : 0.0, sh.above = goal;
    }
    __syncthreads();
    double wt[4];
    int idx[4];
    const int first = sh.bin * SLICE + 4 * tid;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        idx[i] = first + i;
        const uint32_t k = idx[i] < n ? key_of(g.logits[(int64_t) row * g.ld + idx[i]]) : 0;
        wt[i] = k && pair_of(k, idx[i]) >= cut ? weight(top, of_key(k), inv_t) : 0.0;
    }
    return pick<4>(sh, wt, idx, sh.base, sh.above);
}

// A row's largest, log normaliser and token from its slices.
template <bool VEC> __global__ void __launch_bounds__(SM_THREADS) sample_pick_kernel(Sample g, SampleWork w) {
    __shared__ PickLds sh;
    const int row = w.row0 + blockIdx.x, tid = threadIdx.x, lane = tid & 63, S = w.slices;
    const SliceStat st = w.stat[(int64_t) blockIdx.x * S + min(lane, S - 1)];
    uint32_t bk = st.key;
    int bi = st.idx;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t ok = __shfl_xor(bk, o);
        const int oi = __shfl_xor(bi, o);
        if (ok > bk || (ok == bk && oi < bi)) bk = ok, bi = oi;
    }
    const double top = (double) of_key(bk);
    const double z = wave_sum_f64(lane < S ? st.z1 * weight(top, of_key(st.key), 1.0) : 0.0);
    if (tid < S) sh.key[tid] = st.key;
    const RowParams rp = params_of(g, row);
    const bool none = bk <= key_of(-__builtin_inff());
    int token = bi;
    if (!none && rp.t > 0.0f) {
        const RowWay way = way_of(rp, g.vocab);
        token = pick_row<VEC>(g, w, row, rp, way, bk, bi, sh);
        if (token < 0) token = sample_general(g, row, bk, rp, sh.general);
    }
    if (tid == 0) {
        g.token[row] = token;
        if (g.logprob != nullptr) {
            const double v = (double) of_key(key_of(g.logits[(int64_t) row * g.ld + token]));
            g.logprob[row] = none ? -__builtin_inff() : (float) ((v == top ? 0.0 : v - top) - log(z));
        }
    }
}

// Rows of more slices than a wave has lanes: the largest and the sum by one workgroup, the rest the general way.
__global__ void __launch_bounds__(SM_THREADS) sample_long_kernel(Sample g) {
    __shared__ GeneralLds sh;
    __shared__ int widx[SM_WAVES];
    __shared__ uint32_t wkey[SM_WAVES];
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = g.vocab;
    const float* x = g.logits + (int64_t) row * g.ld;
    uint32_t bk = 0;
    int bi = 0;
    for (int i = tid; i < n; i += SM_THREADS) {
        const uint32_t k = key_of(x[i]);
        if (k > bk) bk = k, bi = i;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t ok = __shfl_xor(bk, o);
        const int oi = __shfl_xor(bi, o);
        if (ok > bk || (ok == bk && oi < bi)) bk = ok, bi = oi;
    }
    if (lane == 0) wkey[wave] = bk, widx[wave] = bi;
    __syncthreads();
    bk = wkey[0], bi = widx[0];
    for (int w = 1; w < SM_WAVES; w++)
        if (wkey[w] > bk || (wkey[w] == bk && widx[w] < bi)) bk = wkey[w], bi = widx[w];
    const double top = (double) of_key(bk);
    double z = 0.0;
    for (int i = tid; i < n; i += SM_THREADS) z += weight(top, of_key(key_of(x[i])), 1.0);
    z = wave_sum_f64(z);
    if (lane == 0) sh.wsum[wave] = z;
    __syncthreads();
    z = 0.0;
    for (int w = 0; w < SM_WAVES; w++) z += sh.wsum[w];
    __syncthreads();
    const RowParams rp = params_of(g, row);
    const bool none = bk <= key_of(-__builtin_inff());
    int token = bi;
    if (!none && rp.t > 0.0f) token = sample_general(g, row, bk, rp, sh);
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
    const bool vec = (reinterpret_cast<uintptr_t>(g.logits) & 15) == 0 && g.ld % 4 == 0;
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
