// Drafted trees: which tokens each token sees, and which of them the model agrees with.
//
//   mask(i) = {i} ∪ mask(parent(i)),  depth(i) = |mask(i)| - 1;   path: from node 0 on to the first child whose token is the model's pick
//
// A wave holds one tree, 64 nodes at a time in their order: a parent is below its child, so what a node needs of the blocks before is
// finished when its block begins. Bound by the launch and rounds of dependent loads: masks of one tree 1.6 us, of 256 3.0.
#include "launch.h"

namespace jamhip {

namespace {

constexpr int WAVES = 4;

struct Range {
    int t0, nq, all;   // its first token, those that are looked at, all of them
};
JAMHIP_DEV Range range_of(const Trees& g, int s) {
    Range r;
    r.t0 = min(max(g.q_offsets[s], 0), g.n_tokens);
    r.all = min(max(g.q_offsets[s + 1], r.t0), g.n_tokens) - r.t0;
    r.nq = min(r.all, g.max_q);
    return r;
}

JAMHIP_DEV uint64_t shfl64(uint64_t v, int l) {
    const uint32_t lo = __shfl((uint32_t) v, l), hi = __shfl((uint32_t) (v >> 32), l);
    return (uint64_t) hi << 32 | lo;
}

__global__ void __launch_bounds__(64 * WAVES) tree_masks_kernel(Trees g, uint64_t* masks, int words, int* pos) {
    const int lane = threadIdx.x & 63, s = blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (s >= g.n_seqs) return;
    const Range r = range_of(g, s);
    if (r.nq <= 0) return;
    const int root = pos != nullptr ? pos[r.t0] : 0;   // position of depth 0: the first token's, which it keeps
    for (int b = 0; 64 * b < r.nq; b++) {
        const int i = 64 * b + lane;
        int p = i < r.nq ? g.parents[r.t0 + i] : -1;
        if (p >= i || p < 0) p = -1;
        // ancestors within the block by doubling: `up` is the first node that the bits do not hold yet
        uint64_t bits = 1ull << lane;
        int up = p;
        while (__any(up >= 64 * b)) {
            const int l = up >= 64 * b ? up - 64 * b : lane;
            const uint64_t more = shfl64(bits, l);
            const int next = __shfl(up, l);
            if (up >= 64 * b) bits |= more, up = next;
        }
        if (i < r.nq) {   // the blocks before: as the first ancestor there has them
            uint64_t* row = masks + (int64_t) (r.t0 + i) * words;
            const uint64_t* of = masks + (int64_t) (r.t0 + max(up, 0)) * words;
            int depth = __builtin_popcountll(bits) - 1;
            for (int w = 0; w < words; w++) {
                const uint64_t v = w == b ? bits : w < b && up >= 0 ? __hip_atomic_load(of + w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) : 0;
                row[w] = v;
                if (w < b) depth += __builtin_popcountll(v);
            }
            if (pos != nullptr) pos[r.t0 + i] = root + depth;
        }
        __threadfence_block();   // the next block's lanes read these rows
    }
}

// What a walk reads of a tree: of up to 64 * BLOCKS nodes in the wave's registers, so that a step is a few comparisons and no load; of more
// (BLOCKS 0) in memory. 256 trees of 64: 3.4 us, with a round of loads for every step 6.4.
template <int BLOCKS> struct Nodes {
    int parent[BLOCKS], token[BLOCKS], pick[BLOCKS];
    JAMHIP_DEV Nodes(const Trees& g, const TreeWalk& w, const Range& r) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int b = 0; b < BLOCKS; b++) {
            const int i = 64 * b + lane;
            parent[b] = -1, token[b] = pick[b] = 0;
            if (i < r.nq) parent[b] = g.parents[r.t0 + i], token[b] = w.tokens[r.t0 + i], pick[b] = w.picked[r.t0 + i];
        }
    }
    JAMHIP_DEV int pick_of(int at) const {
        int v = 0;
#pragma unroll
        for (int b = 0; b < BLOCKS; b++)
            if (at / 64 == b) v = __builtin_amdgcn_readlane(pick[b], at % 64);
        return v;
    }
    // the first child of `at` whose token is v, -1 for none; a child comes after its parent
    JAMHIP_DEV int child(int at, int v) const {
        const int lane = threadIdx.x & 63;
        int found = -1;
#pragma unroll
        for (int b = BLOCKS - 1; b >= 0; b--) {
            const unsigned long long hit = __ballot(parent[b] == at && token[b] == v && 64 * b + lane > at);
            if (hit) found = 64 * b + __ffsll(hit) - 1;
        }
        return found;
    }
};
template <> struct Nodes<0> {
    const Trees& g;
    const TreeWalk& w;
    const Range& r;
    JAMHIP_DEV Nodes(const Trees& g, const TreeWalk& w, const Range& r) : g(g), w(w), r(r) {}
    JAMHIP_DEV int pick_of(int at) const { return w.picked[r.t0 + at]; }
    JAMHIP_DEV int child(int at, int v) const {
        const int lane = threadIdx.x & 63;
        for (int b = (at + 1) / 64; 64 * b < r.nq; b++) {
            const int i = 64 * b + lane;
            const unsigned long long hit = __ballot(i > at && i < r.nq && g.parents[r.t0 + i] == at && w.tokens[r.t0 + i] == v);
            if (hit) return 64 * b + __ffsll(hit) - 1;
        }
        return -1;
    }
};

template <int BLOCKS> __global__ void __launch_bounds__(64 * WAVES) tree_accept_kernel(Trees g, TreeWalk w) {
    const int lane = threadIdx.x & 63, s = blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (s >= g.n_seqs) return;
    const Range r = range_of(g, s);
    const Nodes<BLOCKS> nodes(g, w, r);
    int* path = w.path + (int64_t) s * w.ld_path;
    // a root without a slot: the sequence was refused its pages, its drafted tokens have no entries and it stays where it was
    const bool refused = r.nq > 0 && w.slots != nullptr && w.slots[r.t0] < 0;
    int at = r.nq > 0 && w.ld_path > 0 && !refused ? 0 : -1, n = 0, pick = refused ? w.tokens[r.t0] : -1;
    int mine = -1;   // lane k holds the walk's place k of each 64
    auto write = [&](int k0, int k1) {   // places [k0, k1) of the path, those past its end as none
        for (int k = k0 + lane; k < k1; k += 64) {
            const int c = k < n ? mine : -1;
            if (k < w.ld_path) path[k] = c;
            if (w.from != nullptr && k < r.all) {
                w.from[r.t0 + k] = c > k ? w.slots[r.t0 + c] : -1;   // a place is never below its number; at it nothing moves
                w.to[r.t0 + k] = c > k ? w.slots[r.t0 + k] : -1;
            }
        }
    };
    while (at >= 0) {
        pick = nodes.pick_of(at);
        if (lane == n % 64) mine = at;
        n++;
        if (n % 64 == 0) write(n - 64, n);
        at = n < w.ld_path ? nodes.child(at, pick) : -1;
    }
    const int done = n / 64 * 64, end = max(w.ld_path, r.all);
    write(done, end);   // past the first 64 of them all are none: n < done + 64
    if (lane == 0) {
        w.accepted[s] = n;
        w.next[s] = pick;
        if (w.lens_out != nullptr) w.lens_out[s] = w.lens[s] + n;
    }
}

}  // namespace

hipError_t launch_tree_masks(const Trees& g, uint64_t* masks, int words, int* pos, hipStream_t st) {
    tree_masks_kernel<<<(uint32_t) (((int64_t) g.n_seqs + WAVES - 1) / WAVES), 64 * WAVES, 0, st>>>(g, masks, words, pos);
    return hipGetLastError();
}

hipError_t launch_tree_accept(const Trees& g, const TreeWalk& w, hipStream_t st) {
    const uint32_t blocks = (uint32_t) (((int64_t) g.n_seqs + WAVES - 1) / WAVES);
    if (g.max_q <= 64) tree_accept_kernel<1><<<blocks, 64 * WAVES, 0, st>>>(g, w);
    else if (g.max_q <= 256) tree_accept_kernel<4><<<blocks, 64 * WAVES, 0, st>>>(g, w);
    else tree_accept_kernel<0><<<blocks, 64 * WAVES, 0, st>>>(g, w);
    return hipGetLastError();
}

}  // namespace jamhip
