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
inline int attn_cfg(int64_t rows, int dim) { return rows <= 16 ? 0 : rows <= 64 && dim <= ATTN_WIDE_DIM ? 1 : 2; }

// One launch: `tiles` row tiles and `splits` runs of `chunk` keys of each, whose results go to workspace slots from slot0 on,
// or straight to the output (direct).
struct AttnPart {
    int mode;   // 0: every sequence's whole row of keys; 1: the groups' prefixes; 2: the sequences' own keys
    int cfg, tiles, chunk, splits, slot0;
    bool direct;
};

struct AttnPlan {
    int n;          // launches
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
    const int64_t rows = (int64_t) max_q * grp;
    // A prefix is worth reading once for its group while one sequence's rows leave a tile partly empty, and something is shared.
    const bool grouped = n_prefixes > 0 && n_seqs > n_prefixes && rows < attn_rows(2) && max_prefix > 128;
    auto add = [&](int mode, int cfg, int64_t tiles, int64_t busy, int longest) {   // busy: tiles with rows
        AttnPart& a = p.part[p.n++];
        a.mode = mode, a.cfg = cfg, a.tiles = (int) tiles, a.slot0 = p.slots;
        a.splits = attn_splits(cfg, busy * kv, attn_keys(cfg, dim), longest, &a.chunk);
        p.slots += a.splits;
    };
    const int cfg = attn_cfg(rows, dim);
    const int64_t per = (rows + attn_rows(cfg) - 1) / attn_rows(cfg);
    if (!grouped) {
        add(0, cfg, per * n_seqs, per * n_seqs, max_seq + max_prefix);
        if (p.slots == 1) p.part[0].direct = true, p.slots = 0;
        return p;
    }
    const int64_t all = (int64_t) n_tokens * grp;
    const int gcfg = attn_cfg((all + n_prefixes - 1) / n_prefixes, dim), r = attn_rows(gcfg);
    add(1, gcfg, all / r + n_prefixes, ((all + n_prefixes - 1) / n_prefixes + r - 1) / r * n_prefixes, max_prefix);
    add(2, cfg, per * n_seqs, per * n_seqs, max_seq);
    return p;
}

}  // namespace jamhip
