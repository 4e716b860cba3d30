// The next token of each row of logits from a given random number: temperature, top-k, top-p, min-p.
//
// With x sorted by value, largest first and equal ones by index, and w = exp((x - max) / t) in 64 bits:
//   top-k keeps the first k; top-p, of those, the ones before which less than p · (their sum) has been summed, the first in
//   any case; min-p those with w >= min_p. The token is the first in the vocabulary's order whose running sum of kept weights
//   exceeds u · (their sum). Temperature 0: the first of the largest. logprob = x - max - log(sum of exp(x - max)), over all.
//
// Nothing is sorted. The kept set is {x > T} and the first of those equal to T, and T is found digit by digit of the values'
// order-preserving 32-bit keys from histograms of counts (top-k) and of weights (top-p). Weights are summed there as 64-bit
// integers, so that the order of the atomics does not matter.
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

JAMHIP_DEV double wave_sum_f64(double v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    return v;
}

// exp(-(top - x) / t); equal to 1 at the top whatever its value, 0 for -Inf below it
JAMHIP_DEV double weight(double top, float x, double inv_t) {
    const double d = top - (double) x;
    return (double) x == top ? 1.0 : d == d ? exp(-d * inv_t) : 0.0;
}

struct Kept {          // the kept set: keys above `key`, and the first `ties` with that key
    uint32_t key;
    int64_t ties;
};

__global__ void __launch_bounds__(SM_THREADS) sample_kernel(Sample g) {
    __shared__ unsigned long long hist[256];
    __shared__ double wsum[SM_WAVES];
    __shared__ int wtie[SM_WAVES], widx[SM_WAVES];
    __shared__ uint32_t wkey[SM_WAVES];
    __shared__ uint32_t s_digit;
    __shared__ unsigned long long s_rest;
    __shared__ int s_token;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = g.vocab;
    const float* x = g.logits + (int64_t) row * g.ld;

    // the largest and its first index
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

    // the sum at temperature 1
    double z = 0.0;
    for (int i = tid; i < n; i += SM_THREADS) z += weight(top, x[i], 1.0);
    z = wave_sum_f64(z);
    if (lane == 0) wsum[wave] = z;
    __syncthreads();
    z = 0.0;
    for (int w = 0; w < SM_WAVES; w++) z += wsum[w];
    __syncthreads();

    const float temp = g.temperature ? g.temperature[row] : 1.0f;
    int token = bi;
    if (temp > 0.0f && bk > key_of(-__builtin_inff())) {
        const double inv_t = 1.0 / (double) temp;
        Kept kept = {0, (int64_t) n};
        int bits = 0;   // 2^bits >= n: the fixed-point weights' sum stays below 2^63
        while ((int64_t(1) << bits) < n) bits++;
        const double unit = __builtin_ldexp(1.0, 62 - bits);
        // T from a histogram of the next 8 bits below `prefix`, four times: the digit in whose bin the running sum, from the
        // top, first reaches `want`
        auto select = [&](auto&& add, unsigned long long want) -> Kept {
            uint32_t prefix = 0;
            for (int shift = 24; shift >= 0; shift -= 8) {
                for (int b = tid; b < 256; b += SM_THREADS) hist[b] = 0;
                __syncthreads();
                for (int i = tid; i < n; i += SM_THREADS) {
                    const uint32_t k = key_of(x[i]);
                    if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) {
                        const unsigned long long a = add(i, k);
                        if (a) atomicAdd(&hist[(k >> shift) & 255], a);
                    }
                }
                __syncthreads();
                if (tid == 0) {
                    unsigned long long run = 0;
                    int b = 255;
                    for (; b > 0 && run + hist[b] < want; b--) run += hist[b];
                    s_digit = b;
                    s_rest = want - run;
                }
                __syncthreads();
                prefix |= s_digit << shift;
                want = s_rest;
                __syncthreads();
            }
            return Kept{prefix, (int64_t) want};   // want: what is still wanted of the bin of this one key
        };
        const int64_t k = g.top_k ? g.top_k[row] : 0;
        if (k > 0 && k < n) kept = select([&](int, uint32_t) { return 1ull; }, (unsigned long long) k);
        const double p = g.top_p ? (double) g.top_p[row] : 1.0;
        auto fixed = [&](uint32_t key) { return (unsigned long long) (weight(top, of_key(key), inv_t) * unit); };
        if (p < 1.0) {
            // the sum of what top-k left, its ties by their number
            if (tid == 0) s_rest = 0;
            __syncthreads();
            unsigned long long mine = 0;
            for (int i = tid; i < n; i += SM_THREADS) {
                const uint32_t key = key_of(x[i]);
                if (key > kept.key) mine += fixed(key);
            }
            atomicAdd(&s_rest, mine);
            __syncthreads();
            const unsigned long long at = fixed(kept.key);
            const unsigned long long total = s_rest + (kept.key ? at * (unsigned long long) kept.ties : 0ull);
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
        const double minp = g.min_p ? (double) g.min_p[row] : 0.0;
        // wave w takes the run [w · span, (w + 1) · span) of the vocabulary
        const int span = (n + SM_WAVES - 1) / SM_WAVES, lo = min(n, wave * span), hi = min(n, lo + span);
        int ties = 0;
        for (int i0 = lo; i0 < hi; i0 += 64) {
            const int i = i0 + lane;
            ties += __popcll(__ballot(i < hi && key_of(x[min(i, n - 1)]) == kept.key));
        }
        if (lane == 0) wtie[wave] = ties;
        __syncthreads();
        int64_t before = 0;
        for (int w = 0; w < wave; w++) before += wtie[w];
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
        if (lane == 0) wsum[wave] = mine;
        if (tid == 0) s_token = -1;
        __syncthreads();
        double total = 0.0;
        for (int w = 0; w < SM_WAVES; w++) total += wsum[w];
        const double goal = (double) g.u[row] * total;
        double run = 0.0;
        int at = -1, last = 0;
        for (int w = 0; w < SM_WAVES; w++) {
            if (wsum[w] > 0.0) last = w;
            if (at < 0) {
                if (run + wsum[w] > goal) at = w;
                else run += wsum[w];
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
            if (lane == 0) s_token = found >= 0 ? found : final_one;
        }
        __syncthreads();
        token = s_token;
    }
    if (tid == 0) {
        g.token[row] = token;
        if (g.logprob != nullptr) {
            const double v = (double) of_key(key_of(x[token]));
            g.logprob[row] = top == -__builtin_inf() ? -__builtin_inff() : (float) ((v == top ? 0.0 : v - top) - log(z));
        }
    }
}

}  // namespace

hipError_t launch_sample(const Sample& g, hipStream_t st) {
    if (g.rows <= 0) return hipSuccess;
    sample_kernel<<<g.rows, SM_THREADS, 0, st>>>(g);
    return hipGetLastError();
}

}  // namespace jamhip
