// How an attention call is cut into workgroups: plain arithmetic on the call's sizes, shared by the launcher, by the sizing of
// its workspace and by the tests (compiles without HIP).
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "plan.h"

namespace jamhip {

// The tiles of a workgroup of four waves: `rows` query rows (a row is a token's head of one key head), `keys` keys at a time.
//   0: 16 rows in every wave,   1: 32 rows in every wave: 32 keys a wave (attn_wave.h)
//   2: 32 rows a wave, the same 64 keys for all (head_dim over 128: 32) (attn_tile.h)
constexpr int attn_rows(int cfg) { return cfg == 0 ? 16 : cfg == 1 ? 32 : 128; }
constexpr int attn_keys(int cfg, int dim) { return cfg < 2 ? 128 : dim > 128 ? 32 : 64; }
constexpr int ATTN_WIDE_DIM = 192;   // the largest head_dim whose 32 rows fit a wave's registers beside the codes
// Rows of two 32-row tiles: their own reads of the keys against a 128-row tile half empty, 30.5 / 32.8 us for 36 rows behind 8000
// tokens in Q8_0, 32.4 / 34.4 for 64, F16 35.8 / 37.6.
inline int attn_cfg(int64_t rows, int dim) { return rows <= 16 ? 0 : rows <= 64 && dim <= ATTN_WIDE_DIM ? 1 : 2; }

// One launch: `tiles` row tiles and `splits` runs of `chunk` keys of each, whose results go to workspace slots from slot0 on,
// or straight to the output (direct).
struct AttnPart {
    int mode;   // 0: every sequence's whole row of keys; 1: the groups' prefixes; 2: the sequences' own keys
    int cfg, tiles, chunk, splits, slot0;
    bool direct;
};

// HIP takes fewer than 2^32 threads a launch: a part's workgroups, of 256 each, go out in runs of at most this many.
constexpr int64_t ATTN_RUN = 1 << 23;

// Tiles and runs follow the call's maxima, not the device's lengths, so a call fits what it is told and no more. A max_seq_len far above the
// lengths leaves few workgroups with keys: one sequence of 1000 tokens 11.5 us at 1000, 12.8 at 16384, 23.5 at 131072; of 8000 16.7 at 8000,
// 43.7 at 131072. A max_q far above most sequences' query tokens gives each mostly empty tiles and its prefix no group: 63 sequences'
// next tokens and a prompt of 1024, behind 8192 shared tokens, 2030 us in one call, 408 in one for the decoding and one for the prompt.
struct AttnPlan {
    int n;          // launches; 0: more workgroups than are numbered in 32 bits
    AttnPart part[2];
    int slots;      // workspace results per output row
};

// Splits of up to `longest` keys for `groups` workgroups with work: as many workgroups as are resident at once, two to a CU, whole
// tiles each. More do not help where sequences differ in length: a run of keys costs its start and end (64 sequences of 33 to
// 1024 keys, 8 key heads: 27 us as one run each, 31 as two, 36 as four).
inline int attn_splits(int cfg, int64_t groups, int keys, int longest, int* chunk) {
    const int tiles = longest > 0 ? up_div(longest, keys) : 1, least = cfg < 2 ? 1 : 2;
    const int64_t want = groups >= 512 ? 1 : 512 / groups;
    int splits = (int) (want < tiles / least ? want : tiles / least);
    if (splits < 1) splits = 1;
    const int per = up_div(tiles, splits);
    *chunk = per * keys;
    return up_div(tiles, per);
}

inline AttnPlan attn_plan(int dim, int kv, int grp, int n_tokens, int n_seqs, int n_prefixes, int max_q, int max_seq, int max_prefix) {
    AttnPlan p{};
    bool fits = true;
    const int64_t rows = (int64_t) max_q * grp;
    // A prefix read once for its group costs a second launch, the joining of every sequence and emptier tiles, 8 us for 16 sequences
    // and 16 for 64; what it saves grows with the keys that the group's other sequences do not walk again, less where a sequence's
    // own rows fill a 16-row tile, since their products stay. In us, grouped against sequence by sequence, Q8_0, heads of 128, 8 key
    // heads and 4 rows unless said: 64 sequences behind 400 tokens 32 / 20, 800 32 / 27, 2000 34 / 49; 16 behind 800 22 / 16, 2000
    // 24 / 24; 4 behind 6000 25 / 19; 64 behind 2000 with 2 key heads 28 / 24, with 1 27 / 19, of 16 rows 60 / 50; 16 of 32 rows
    // behind 3000 45 / 35, 16000 95 / 105; 64 of 32 rows behind 4000 109 / 101, 16000 288 / 357.
    const int64_t saved = (n_seqs - 4 * (int64_t) n_prefixes) * kv * max_prefix, cost = (60000 + 7500 * (int64_t) n_seqs) * (rows <= 8 ? 1 : 4);
    const bool grouped = n_prefixes > 0 && rows < attn_rows(2) && saved >= cost;
    auto add = [&](int mode, int cfg, int64_t tiles, int64_t busy, int longest) {   // busy: tiles with rows
        AttnPart& a = p.part[p.n++];
        a.mode = mode, a.cfg = cfg, a.tiles = (int) tiles, a.slot0 = p.slots;
        a.splits = attn_splits(cfg, busy * kv, attn_keys(cfg, dim), longest, &a.chunk);
        p.slots += a.splits;
        fits = fits && tiles <= INT32_MAX / kv / a.splits;
    };
    const int cfg = attn_cfg(rows, dim);
    const int64_t per = (rows + attn_rows(cfg) - 1) / attn_rows(cfg);
    if (!grouped) {
        add(0, cfg, per * n_seqs, per * n_seqs, max_seq + max_prefix);
        if (p.slots == 1) p.part[0].direct = true, p.slots = 0;
        return fits ? p : AttnPlan{};
    }
    const int64_t all = (int64_t) n_tokens * grp;
    const int gcfg = attn_cfg((all + n_prefixes - 1) / n_prefixes, dim), r = attn_rows(gcfg);
    add(1, gcfg, all / r + n_prefixes, ((all + n_prefixes - 1) / n_prefixes + r - 1) / r * n_prefixes, max_prefix);
    add(2, cfg, per * n_seqs, per * n_seqs, max_seq);
    return fits ? p : AttnPlan{};
}

}  // namespace jamhip
