// The lists of the sampling kernel's second launch and how a workgroup sorts them (also compiles for the host where threadIdx,
// __syncthreads and JAMHIP_DEV are given).
#pragma once

#include <stdint.h>

namespace jamhip {

// The second launch is a chain of short steps: four waves, one a SIMD, take it at half the time of sixteen, which all repeat
// what each step does for its wave.
constexpr int SM_THREADS = 256, SM_WAVES = SM_THREADS / 64;

// An element of a list: larger values first, the lower index first among equal ones.
JAMHIP_DEV unsigned long long pair_of(uint32_t key, int idx) { return (unsigned long long) key << 32 | (uint32_t) ~idx; }
JAMHIP_DEV uint32_t pair_key(unsigned long long p) { return (uint32_t) (p >> 32); }
JAMHIP_DEV int pair_idx(unsigned long long p) { return (int) ~(uint32_t) p; }

// list[0 .. n), written before the last barrier, in falling order; above 256 elements it is filled up to a power of two with zeros.
JAMHIP_DEV void sort_falling(unsigned long long* list, int n) {
    const int tid = threadIdx.x;
    if (n <= SM_THREADS) {   // an element's place is the number of larger ones
        const unsigned long long v = tid < n ? list[tid] : 0;
        int place = 0;
        if (tid < n)
            for (int i = 0; i < n; i++) place += list[i] > v;
        __syncthreads();
        if (tid < n) list[place] = v;
        __syncthreads();
        return;
    }
    int size = 2 * SM_THREADS;
    while (size < n) size <<= 1;
    for (int i = n + tid; i < size; i += SM_THREADS) list[i] = 0;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1)   // a bitonic network
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int p = tid; p < size / 2; p += SM_THREADS) {
                const int a = 2 * p - (p & (j - 1)), b = a + j;   // bit j of a is 0
                const unsigned long long u = list[a], v = list[b];
                if ((u < v) == ((a & k) == 0)) list[a] = v, list[b] = u;
            }
            __syncthreads();
        }
}

// The first m of a sorted list again, in the vocabulary's order: (~index, place in the list before).
JAMHIP_DEV void order_by_index(unsigned long long* list, int m) {
#pragma unroll 1
    for (int e = threadIdx.x; e < m; e += SM_THREADS) list[e] = (list[e] & 0xFFFFFFFFull) << 32 | (unsigned) e;
    __syncthreads();   // sort_falling looks at all of them before its first barrier
    sort_falling(list, m);
}

}  // namespace jamhip
