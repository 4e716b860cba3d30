// Drafted trees: which tokens each token sees, and which of them the model agrees with.
//
//   mask(i) = {i} ∪ mask(parent(i)),  depth(i) = |mask(i)| - 1;   path: from node 0 on to the first child whose token is the model's pick
//
// A wave holds one tree, 64 nodes at a time in their order: a parent is below its child, so what a node needs of the blocks before is
// finished when its block begins. Bound by the launch and three rounds of loads.
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

__global__ void __launch_bounds__(64 * WAVES) tree_accept_kernel(Trees g, TreeWalk w) {
    const int lane = threadIdx.x & 63, s = blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (s >= g.n_seqs) return;
    const Range r = range_of(g, s);
    int* path = w.path + (int64_t) s * w.ld_path;
    int at = 0, n = 0, pick = -1;
    bool on = r.nq > 0 && w.ld_path > 0;
    while (on) {
        pick = w.picked[r.t0 + at];
        if (lane == 0) {
            path[n] = at;
            if (w.from != nullptr) {
                const bool move = at != n;
                w.from[r.t0 + n] = move ? w.slots[r.t0 + at] : -1;
                w.to[r.t0 + n] = move ? w.slots[r.t0 + n] : -1;
            }
        }
        n++;
        on = false;
        if (n >= w.ld_path) break;
        for (int b = (at + 1) / 64; 64 * b < r.nq; b++) {   // a child comes after its parent
            const int i = 64 * b + lane;
            const bool fits = i > at && i < r.nq && g.parents[r.t0 + i] == at && w.tokens[r.t0 + i] == pick;
            const unsigned long long hit = __ballot(fits);
            if (hit) {
                at = 64 * b + __ffsll(hit) - 1;
                on = true;
                break;
            }
        }
    }
    for (int k = n + lane; k < w.ld_path; k += 64) path[k] = -1;
    if (w.from != nullptr)
        for (int k = n + lane; k < r.all; k += 64) w.from[r.t0 + k] = w.to[r.t0 + k] = -1;
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
    tree_accept_kernel<<<(uint32_t) (((int64_t) g.n_seqs + WAVES - 1) / WAVES), 64 * WAVES, 0, st>>>(g, w);
    return hipGetLastError();
}

}  // namespace jamhip
