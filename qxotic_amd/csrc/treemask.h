// Which keys a query token of a drafted tree sees (compiles without HIP).
//
// A sequence's keys are its context, `ctx` tokens, and its `nq` query tokens behind it, whose entries are the last of its own. A query
// token sees the context and the query tokens whose bits are set in its row of the mask; with a window only the last `window` keys of
// that list. So the context that it sees is one range, and the rest are the bits in [b0, b1) of its row: the window drops the lowest.
#pragma once

#include <stdint.h>

#include "fastdiv.h"

#ifdef __HIPCC__
#define JAMHIP_MASK_DEV __host__ __device__ __forceinline__
#else
#define JAMHIP_MASK_DEV inline
#endif

namespace jamhip {

struct TreeMask {
    const uint64_t* row;
    int words;
};

struct TreeSpan {
    int ctx_lo, ctx_hi;   // the context's keys that it sees: [ctx_lo, ctx_hi)
    int tree0, b0, b1;    // and keys tree0 + j of the bits j in [b0, b1)
};

JAMHIP_MASK_DEV int mask_max(int a, int b) { return a > b ? a : b; }
JAMHIP_MASK_DEV int mask_min(int a, int b) { return a < b ? a : b; }

// word w of the row, the bits in [b0, b1) alone; zero for a word that the row does not have
JAMHIP_MASK_DEV uint64_t mask_word(const TreeMask& m, int w, int b0, int b1) {
    if (w < 0 || w >= m.words || b1 <= 64 * w || b0 >= 64 * w + 64 || b0 >= b1) return 0;
    uint64_t v = m.row[w];
    if (b0 > 64 * w) v &= ~0ull << (b0 - 64 * w);
    if (b1 < 64 * w + 64) v &= ~(~0ull << (b1 - 64 * w));
    return v;
}

// base: tokens of the prefix; first: the first query token's place among the own tokens, below zero where there are more query
// tokens than own ones (those in front have no entry); words · 64 fits 32 bits
JAMHIP_MASK_DEV TreeSpan tree_span(const TreeMask& m, int base, int first, int nq, int window) {
    TreeSpan s;
    s.ctx_lo = 0, s.ctx_hi = base + mask_max(first, 0);
    s.tree0 = base + first, s.b0 = mask_max(0, -first), s.b1 = mask_min(nq, 64 * m.words);
    if (window > 0) {
        int n = 0;
        for (int w = s.b0 / 64; 64 * w < s.b1; w++) n += __builtin_popcountll(mask_word(m, w, s.b0, s.b1));
        if (n < window) {
            s.ctx_lo = mask_max(0, s.ctx_hi - (window - n));
        } else {
            s.ctx_lo = s.ctx_hi;
            int drop = n - window;
            for (int w = s.b0 / 64; 64 * w < s.b1; w++) {
                uint64_t v = mask_word(m, w, s.b0, s.b1);
                const int here = __builtin_popcountll(v);
                if (drop >= here) {
                    drop -= here;
                    continue;
                }
                for (; drop > 0; drop--) v &= v - 1;
                s.b0 = 64 * w + __builtin_ctzll(v);
                break;
            }
        }
    }
    return s;
}

// the part of a span in the run of keys [c0, c1), whose numbers have `skip` keys fewer in front
JAMHIP_MASK_DEV TreeSpan span_cut(TreeSpan s, int skip, int c0, int c1) {
    s.ctx_lo = mask_max(s.ctx_lo - skip, c0), s.ctx_hi = mask_min(s.ctx_hi - skip, c1);
    s.tree0 -= skip;
    s.b0 = mask_max(s.b0, c0 - s.tree0), s.b1 = mask_min(s.b1, c1 - s.tree0);
    return s;
}

// a range that holds every key of a span, [span_lo, span_hi), without a look at the bits
JAMHIP_MASK_DEV int span_lo(const TreeSpan& s) { return s.ctx_lo < s.ctx_hi ? s.ctx_lo : s.tree0 + s.b0; }
JAMHIP_MASK_DEV int span_hi(const TreeSpan& s) { return s.b0 < s.b1 ? s.tree0 + s.b1 : s.ctx_lo < s.ctx_hi ? s.ctx_hi : s.tree0 + s.b0; }

JAMHIP_MASK_DEV bool span_sees(const TreeMask& m, const TreeSpan& s, int key) {
    if (key >= s.ctx_lo && key < s.ctx_hi) return true;
    const int j = key - s.tree0;
    return j >= s.b0 && j < s.b1 && (m.row[j / 64] >> (j % 64) & 1);
}

// bit i: the key k0 + i is seen, for the 64 keys from k0 on
JAMHIP_MASK_DEV uint64_t span_tile(const TreeMask& m, const TreeSpan& s, int k0) {
    uint64_t v = 0;
    const int lo = mask_max(s.ctx_lo - k0, 0), hi = mask_min(s.ctx_hi - k0, 64);
    if (lo < hi) v = (~0ull >> (64 - (hi - lo))) << lo;
    const int d = k0 - s.tree0;   // the bit that key k0 has
    if (d < s.b1 && d > s.b0 - 64) {
        if (d >= 0) {
            const int w = d / 64, sh = d % 64;
            v |= mask_word(m, w, s.b0, s.b1) >> sh;
            if (sh) v |= mask_word(m, w + 1, s.b0, s.b1) << (64 - sh);
        } else {
            v |= mask_word(m, 0, s.b0, s.b1) << -d;
        }
    }
    return v;
}

}  // namespace jamhip
