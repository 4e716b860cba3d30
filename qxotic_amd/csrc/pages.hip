// Pages of the cache handed out and taken back by the sequences' lengths, their slots, and entries moved between slots.
//
//   need_s  = ceil(target_s / page)                       back_s = max(0, held_s - need_s)     take_s = max(0, need_s - held_s)
//   pages given back go on the list of free ones from the last sequence to the first, each one's last page first; then the sequences take
//   theirs off its end in their order, so that giving back at once what was taken restores the list
//   q_offsets = the sums of max(0, target - len) before, slot(p) = seq_pages[p / page] · page + p % page
//
// Small integers in a chain: what counts is the number of launches and of rounds of dependent loads. Lists and counts are device data:
// whatever they hold, no index leaves the arrays.
#include <algorithm>

#include "launch.h"

namespace jamhip {

namespace {

constexpr int T = 1024;   // threads, and sequences at once, of the workgroup that hands out pages

// exclusive sums of v over the workgroup's threads; *total gets the whole. `lds`: T / 64 + 1 entries, free again after the next barrier
JAMHIP_DEV int64_t block_scan(int64_t v, int64_t* lds, int64_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) lds[wave] = x;
    __syncthreads();
    int64_t before = 0, all = 0;
    for (int i = 0; i < T / 64; i++) {
        before += i < wave ? lds[i] : 0;
        all += lds[i];
    }
    *total = all;
    return before + x - v;
}

struct Want {
    int len, target, held, need;
    int64_t fresh;   // new tokens
};
JAMHIP_DEV Want want_of(const Pages& g, int s) {
    Want w{};
    if (s < g.n_seqs) {
        w.len = max(g.lens[s], 0);
        w.target = max(g.targets[s], 0);
        w.held = min(max(g.held[s], 0), g.ld);
        w.need = g.page.div(w.target) + (g.page.div(w.target) * g.page.d < w.target);
        w.fresh = max(0, w.target - w.len);
    }
    return w;
}

// the last i in [0, n) with a[i] <= v, a rising from a[0] <= v
JAMHIP_DEV int find_last(const int64_t* a, int n, int64_t v) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= v) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(T) kv_resize_kernel(Pages g) {
    __shared__ int64_t scan[T / 64 + 1];
    __shared__ int64_t start[T];   // a chunk's sequences: pages given back or taken before each
    __shared__ int first[T];       // and the first page's place in its row
    __shared__ int stop;           // the first sequence of a chunk that does not fit
    const int tid = threadIdx.x;
    const int64_t free0 = min(max(g.n_free[0], 0), g.free_cap);
    int64_t total = 0, sum;
    for (int s0 = 0; s0 < g.n_seqs; s0 += T) {
        const Want w = want_of(g, s0 + tid);
        (void) block_scan(max(0, w.held - w.need), scan, &sum);
        total += sum;
    }
    if (total > 0) {
        int64_t done = 0;
        for (int s0 = 0; s0 < g.n_seqs; s0 += T) {
            const Want w = want_of(g, s0 + tid);
            const int64_t at = block_scan(max(0, w.held - w.need), scan, &sum);
            start[tid] = at, first[tid] = w.need;
            __syncthreads();
            for (int64_t k = tid; k < sum; k += T) {
                const int i = find_last(start, T, k);
                // k counts from the row's first page that goes back; on the list it stands that far from the end
                const int64_t place = free0 + total - 1 - (done + k);
                if (place < g.free_cap) g.free_pages[place] = g.seq_pages[(int64_t) (s0 + i) * g.ld + first[i] + (k - start[i])];
            }
            __syncthreads();
            done += sum;
        }
    }
    __threadfence_block();
    __syncthreads();
    const int64_t have = min(free0 + total, (int64_t) g.free_cap);
    int64_t taken = 0, rows = 0, given = 0;   // pages asked for, tokens, pages handed out by the sequences before
    bool full = false;
    for (int s0 = 0; s0 < g.n_seqs; s0 += T) {
        const int s = s0 + tid;
        const Want w = want_of(g, s);
        const int64_t take = max(0, w.need - w.held);
        int64_t asked, all_rows;
        const int64_t at = block_scan(take, scan, &asked);
        const int64_t row = block_scan(w.fresh, scan, &all_rows);
        const bool grows = take > 0 || w.fresh > 0;
        if (tid == 0) stop = full ? 0 : T;
        __syncthreads();
        if (!full && grows && (taken + at + take > have || rows + row + w.fresh > g.n_tokens || w.need > g.ld)) atomicMin(&stop, tid);
        __syncthreads();
        const bool refused = grows && tid >= stop;
        start[tid] = at, first[tid] = w.held;
        if (s < g.n_seqs) {
            g.lens_out[s] = refused ? w.len : w.target;
            g.held_out[s] = refused ? min(w.held, w.need) : w.need;   // what was too much has been given back
            g.status[s] = refused;
            g.q_offsets[s] = (int) min(rows + row, (int64_t) g.n_tokens);
        }
        __syncthreads();
        const int64_t served = stop < T ? (full ? 0 : start[stop]) : asked;
        for (int64_t k = tid; k < served; k += T) {
            const int i = find_last(start, T, k);
            g.seq_pages[(int64_t) (s0 + i) * g.ld + first[i] + (k - start[i])] = g.free_pages[have - 1 - (taken + k)];
        }
        full = full || stop < T;
        taken += asked, rows += all_rows, given += served;
        __syncthreads();
    }
    if (tid == 0) {
        g.q_offsets[g.n_seqs] = (int) min(rows, (int64_t) g.n_tokens);
        g.n_free_out[0] = (int) (have - given);
    }
}

// ---- up to T sequences, sums in 32 bits: every workgroup adds up all sequences by itself, moves its share of the pages and fills its share of
// the tokens. A page that one sequence gives back and another takes is looked up where it comes from, so no workgroup waits for another's
// writes. What may be written in place (lens, held, n_free) is left to a workgroup that nobody reads beside: the only one, or, where the arrays
// are apart, the first, or a launch of its own behind the others.
constexpr int SHARE_TOKENS = 1024, SHARE_ENTRIES = 16384;   // of a workgroup: new tokens, entries of the table
constexpr int MOST_GROUPS = 128;

// the last i below 2 * half, a power of two up to T, with a[i] <= v, a rising from a[0] <= v
JAMHIP_DEV int find_seq(const int* a, int v, int half) {
    int lo = 0;
    for (int step = half; step > 0; step >>= 1) lo += a[lo + step] <= v ? step : 0;
    return lo;
}

__global__ void __launch_bounds__(T) kv_resize_shared_kernel(Pages g, bool work, bool commit) {
    __shared__ int back_at[T], take_at[T], row_at[T];   // pages given back, pages taken, tokens of the sequences before
    __shared__ int s_need[T], s_held[T], s_len[T];      // s_len: -1 - length of a sequence that was refused
    __shared__ int part[3][T / 64], stops[T / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int free0 = min(max(g.n_free[0], 0), g.free_cap);
    const Want w = want_of(g, tid);
    // what does not fit is cut to where it still does not: the sums stay below 2^31
    const int back = max(0, w.held - w.need), take = min(max(0, w.need - w.held), g.ld + 1), fresh = (int) min(w.fresh, (int64_t) g.n_tokens + 1);
    int at[3] = {wave_exclusive_scan(back), wave_exclusive_scan(take), wave_exclusive_scan(fresh)};
    if (lane == 63) part[0][wave] = at[0] + back, part[1][wave] = at[1] + take, part[2][wave] = at[2] + fresh;
    __syncthreads();
    int total[3];
#pragma unroll
    for (int i = 0; i < 3; i++) {
        const int v = lane < T / 64 ? part[i][lane] : 0, before = wave_exclusive_scan(v);
        total[i] = __builtin_amdgcn_readlane(before, T / 64);
        at[i] += __builtin_amdgcn_readlane(before, wave);
    }
    const int have = (int) min((int64_t) free0 + total[0], (int64_t) g.free_cap);
    const bool grows = take > 0 || fresh > 0;
    const unsigned long long full = __ballot(grows && (at[1] + take > have || at[2] + fresh > g.n_tokens || w.need > g.ld));
    if (lane == 0) stops[wave] = full ? 64 * wave + __ffsll(full) - 1 : T;
    back_at[tid] = at[0], take_at[tid] = at[1], row_at[tid] = at[2];
    s_need[tid] = w.need, s_held[tid] = w.held;
    __syncthreads();
    const int first = lane < T / 64 ? stops[lane] : T;
    int stop = first;   // the first sequence that does not fit
#pragma unroll
    for (int o = 1; o < T / 64; o <<= 1) stop = min(stop, __shfl_xor(stop, o));
    stop = __builtin_amdgcn_readfirstlane(stop);
    const bool refused = grows && tid >= stop;
    s_len[tid] = refused ? -1 - w.len : w.len;
    const int taken = stop < T ? take_at[stop] : total[1];
    __syncthreads();
    const int half = g.n_seqs > 1 ? 1 << (31 - __builtin_clz(g.n_seqs - 1)) : 0;   // 2 * half >= n_seqs
    // the page at place i of the free list once all are given back
    auto page_at = [&](int i) {
        if (i < free0) return g.free_pages[i];
        const int k = free0 + total[0] - 1 - i, s = find_seq(back_at, k, half);
        return g.seq_pages[(int64_t) s * g.ld + s_need[s] + (k - back_at[s])];
    };
    if (work) {
        for (int k = blockIdx.x * T + tid; k < total[0]; k += gridDim.x * T) {
            const int s = find_seq(back_at, k, half), place = free0 + total[0] - 1 - k;
            if (place < g.free_cap) g.free_pages[place] = g.seq_pages[(int64_t) s * g.ld + s_need[s] + (k - back_at[s])];
        }
        for (int k = blockIdx.x * T + tid; k < taken; k += gridDim.x * T) {
            const int s = find_seq(take_at, k, half);
            g.seq_pages[(int64_t) s * g.ld + s_held[s] + (k - take_at[s])] = page_at(have - 1 - k);
        }
        for (int t = blockIdx.x * T + tid; t < g.n_tokens; t += gridDim.x * T) {
            int pos = 0, slot = -1;
            if (t < total[2]) {
                const int s = find_seq(row_at, t, half), p = (s_len[s] < 0 ? -1 - s_len[s] : s_len[s]) + (t - row_at[s]);
                pos = p + (g.base != nullptr ? g.base[s] : 0);
                if (s_len[s] >= 0) {
                    const int c = g.page.div(p), page = c < s_held[s] ? g.seq_pages[(int64_t) s * g.ld + c] : page_at(have - 1 - (take_at[s] + c - s_held[s]));
                    if ((uint32_t) page < (uint32_t) g.n_pages) slot = page * g.page.d + (p - c * g.page.d);
                }
            }
            g.pos[t] = pos;
            g.slots[t] = slot;
        }
    }
    if (!commit || blockIdx.x > 0) return;
    if (tid < g.n_seqs) {
        g.lens_out[tid] = refused ? w.len : w.target;
        g.held_out[tid] = refused ? min(w.held, w.need) : w.need;
        g.status[tid] = refused;
        g.q_offsets[tid] = min(at[2], g.n_tokens);
    }
    if (tid == 0) {
        g.q_offsets[g.n_seqs] = min(total[2], g.n_tokens);
        g.n_free_out[0] = have - taken;
    }
}

constexpr int FILL = 256;

// One token a thread: its sequence, position and slot.
__global__ void __launch_bounds__(FILL) kv_slots_kernel(Pages g) {
    const int t = blockIdx.x * FILL + threadIdx.x;
    if (t >= g.n_tokens) return;
    int lo = 0, hi = g.n_seqs + 1;   // the last offset not above t
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (g.q_offsets[mid] <= t) lo = mid;
        else hi = mid;
    }
    int pos = 0, slot = -1;
    if (lo < g.n_seqs) {
        const int o0 = g.q_offsets[lo], n = g.q_offsets[lo + 1] - o0;
        const bool refused = g.status[lo] != 0;
        const int p = g.lens_out[lo] - (refused ? 0 : n) + (t - o0);   // the length before and on
        pos = p + (g.base != nullptr ? g.base[lo] : 0);
        if (!refused && p >= 0) {
            const int c = g.page.div(p);
            const int page = c < g.ld ? g.seq_pages[(int64_t) lo * g.ld + c] : -1;
            if ((uint32_t) page < (uint32_t) g.n_pages) slot = page * g.page.d + (p - c * g.page.d);
        }
    }
    g.pos[t] = pos;
    g.slots[t] = slot;
}

// ---- entries moved
// A workgroup moves one group's entries in one cache: a thread holds the same pieces of every entry, so that the entries of a group go in their
// order without a barrier between them. Pieces are 16 bytes of codes, and scales one by one (their rows are 2, 4, 6 bytes and so on): keys'
// codes, values' codes, keys' scales, values' scales, numbered through, so that all of an entry is loaded before the first is stored. 64
// sequences' 6 entries in 32 F16 caches, 101 MB read and written: 18.5 us (5.4 TB/s); one sequence's in 4 Q8_0 caches 4.3 us, rounds of dependent
// loads (offsets, slots, entries), 6.3 with a plane of the cache after the other. Scales cost more than their bytes, two of them a thread: calls one
// after another take 21.7 us for the 64 in F16 (101 MB), 20.6 in Q8_0 (54 MB), 15.8 in Q4_0 (28 MB).
constexpr int BATCH = 4;

struct Spot {   // of an entry: its page, and its token of the page
    int page, in;
};

template <int TYPE> __global__ void __launch_bounds__(256) kv_move_kernel(Move g, int block0) {
    const int b = block0 + blockIdx.x, cache = b % g.n_caches, grp = b / g.n_caches;
    const KvView& c = g.cache;
    const int e0 = min(max(g.offsets[grp], 0), g.n), e1 = min(max(g.offsets[grp + 1], e0), g.n);
    const int lane = threadIdx.x & 63;
    const int row = kv_row_bytes(TYPE, c.dim) / 16, codes = c.kv * row, sc = kv_scales(TYPE, c.dim), all = 2 * (codes + c.kv * sc);
    for (int s0 = e0; s0 < e1; s0 += 64) {
        const int e = s0 + lane;
        int f = -1, t = -1;
        if (e < e1) f = g.from[e], t = g.to[e];
        const int64_t slots = c.slots();
        unsigned long long on = __ballot(f >= 0 && t >= 0 && f < slots && t < slots && f != t);
        while (on) {
            // up to BATCH entries whose sources no earlier one of them writes
            Spot from[BATCH], to[BATCH];
            int dst[BATCH], n = 0;
#pragma unroll
            for (int i = 0; i < BATCH; i++) {
                from[i] = to[i] = {0, 0}, dst[i] = -1;
                if (on && n == i) {
                    const int l = __ffsll(on) - 1;
                    const int ff = __builtin_amdgcn_readlane(f, l), tt = __builtin_amdgcn_readlane(t, l);
                    bool clash = false;
#pragma unroll
                    for (int j = 0; j < i; j++) clash |= dst[j] == ff;
                    if (!clash) {
                        from[i].page = c.page.div(ff), from[i].in = ff - from[i].page * c.page.d;
                        to[i].page = c.page.div(tt), to[i].in = tt - to[i].page * c.page.d;
                        dst[i] = tt;
                        n = i + 1;
                        on &= on - 1;
                    }
                }
            }
            for (int u = threadIdx.x; u < all; u += blockDim.x) {
                const bool scale = TYPE != F16 && u >= 2 * codes;
                const int half = scale ? c.kv * sc : codes, v = scale ? u - 2 * codes : u, p = v >= half ? v - half : v, per = scale ? sc : row;
                uint8_t* const buf = (v >= half ? g.v[cache] : g.k[cache]) + (scale ? c.scale_off : 0);
                const int head = p / per, at = p - head * per;
                auto place = [&](const Spot& s) { return (((int64_t) s.page * c.kv + head) * c.page.d + s.in) * per + at; };
                uint4_t x[BATCH];
                uint16_t y[BATCH];
#pragma unroll
                for (int i = 0; i < BATCH; i++)
                    if (i < n) {
                        if (scale) y[i] = reinterpret_cast<const uint16_t*>(buf)[place(from[i])];
                        else x[i] = reinterpret_cast<const uint4_t*>(buf)[place(from[i])];
                    }
#pragma unroll
                for (int i = 0; i < BATCH; i++)
                    if (i < n) {
                        if (scale) reinterpret_cast<uint16_t*>(buf)[place(to[i])] = y[i];
                        else reinterpret_cast<uint4_t*>(buf)[place(to[i])] = x[i];
                    }
            }
        }
    }
}

}  // namespace

hipError_t launch_kv_resize(const Pages& g, hipStream_t st) {
    // us a call: 64 sequences of 32 new tokens 5.3, by the kernels for any number 10.1; 512 with 114594 new tokens and 26000 to 30000 pages moved 8.1, 36.4
    if (g.n_seqs <= T && g.ld < 1 << 20 && g.n_tokens < 1 << 20 && g.free_cap < 1 << 30) {
        const int64_t want = std::max(((int64_t) g.n_tokens + SHARE_TOKENS - 1) / SHARE_TOKENS,
                                      ((int64_t) g.n_seqs * g.ld + SHARE_ENTRIES - 1) / SHARE_ENTRIES);
        const int groups = (int) std::min<int64_t>(std::max<int64_t>(want, 1), MOST_GROUPS);
        bool one = groups == 1;
        if (!one) {   // no array that the first workgroup writes is one that others still read
            auto overlap = [](const int* a, int n, const int* b, int m) { return a < b + m && b < a + n; };
            const struct { const int* p; int n; } in[] = {{g.lens, g.n_seqs}, {g.targets, g.n_seqs}, {g.held, g.n_seqs}, {g.base, g.base ? g.n_seqs : 0}, {g.n_free, 1}};
            const struct { const int* p; int n; } out[] = {{g.lens_out, g.n_seqs}, {g.held_out, g.n_seqs}, {g.n_free_out, 1}, {g.status, g.n_seqs}, {g.q_offsets, g.n_seqs + 1}};
            one = true;
            for (const auto& i : in)
                for (const auto& o : out) one = one && !overlap(i.p, i.n, o.p, o.n);
        }
        kv_resize_shared_kernel<<<groups, T, 0, st>>>(g, true, one);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || one) return e;
        kv_resize_shared_kernel<<<1, T, 0, st>>>(g, false, true);
        return hipGetLastError();
    }
    kv_resize_kernel<<<1, T, 0, st>>>(g);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || g.n_tokens == 0) return e;
    kv_slots_kernel<<<(g.n_tokens + FILL - 1) / FILL, FILL, 0, st>>>(g);
    return hipGetLastError();
}

hipError_t launch_kv_move(int type, const Move& g, hipStream_t st) {
    const int64_t blocks = (int64_t) g.groups * g.n_caches;   // at most 2^20 * MOVE_CACHES
    constexpr int64_t RUN = 1 << 23;   // HIP takes fewer than 2^32 threads a launch
    for (int64_t b = 0; b < blocks; b += RUN) {
        const uint32_t n = (uint32_t) (blocks - b < RUN ? blocks - b : RUN);
        switch (type) {
            case F16: kv_move_kernel<F16><<<n, 256, 0, st>>>(g, (int) b); break;
            case Q8_0: kv_move_kernel<Q8_0><<<n, 256, 0, st>>>(g, (int) b); break;
            case Q4_0: kv_move_kernel<Q4_0><<<n, 256, 0, st>>>(g, (int) b); break;
            default: return hipErrorNotSupported;
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace jamhip
