// What the calls around drafted trees refuse (compiles without HIP).
#pragma once

#include <stdint.h>

#include "jamhip.h"

namespace jamhip {

struct Refusal {
    jamhip_status status;   // JAMHIP_OK: the call is taken
    const char* why;
};
constexpr Refusal TAKEN = {JAMHIP_OK, ""};
constexpr int MAX_SEQS = 1 << 20;
constexpr int MAX_TOKENS = INT32_MAX - 4096;

inline Refusal refuse_pages(const jamhip_kv_pages* p) {
    if (!p) return {JAMHIP_EINVAL, "kv_resize: null description"};
    if (p->n_seqs < 0 || p->n_tokens < 0 || p->page_tokens <= 0 || p->n_pages < 0 || p->free_cap < 0 || p->ld_seq_pages < 0)
        return {JAMHIP_EINVAL, "kv_resize: bad shape"};
    const bool seqs = p->lens && p->targets && p->held && p->lens_out && p->held_out && p->status && (p->seq_pages || p->ld_seq_pages == 0);
    if ((p->n_seqs > 0 && !seqs) || !p->n_free || !p->n_free_out || !p->q_offsets || (p->free_cap > 0 && !p->free_pages) ||
        (p->n_tokens > 0 && (!p->pos || !p->slots)))
        return {JAMHIP_EINVAL, "kv_resize: null array"};
    if (p->n_seqs > MAX_SEQS || p->n_tokens > MAX_TOKENS || (int64_t) p->n_pages * p->page_tokens > INT32_MAX)
        return {JAMHIP_EUNSUPPORTED, "kv_resize: more than 2^20 sequences, or tokens or slots beyond 32 bits"};
    return TAKEN;
}

inline Refusal refuse_tree(const jamhip_tree* t) {
    if (!t) return {JAMHIP_EINVAL, "tree: null description"};
    if (t->n_tokens < 0 || t->n_seqs < 0 || t->max_q < 0) return {JAMHIP_EINVAL, "tree: bad shape"};
    if (t->n_seqs > 0 && t->n_tokens > 0 && (!t->q_offsets || !t->parents)) return {JAMHIP_EINVAL, "tree: null array"};
    if (t->n_seqs > MAX_SEQS || t->n_tokens > MAX_TOKENS) return {JAMHIP_EUNSUPPORTED, "tree: more than 2^20 sequences, or tokens beyond 32 bits"};
    return TAKEN;
}

// rows of `words` 64-bit words, for up to max_q drafted tokens a sequence
inline Refusal refuse_masks(const void* masks, int words, int max_q) {
    if (!masks || (reinterpret_cast<uintptr_t>(masks) & 7)) return {JAMHIP_EINVAL, "tree masks: null or not 8-byte aligned"};
    if (words <= 0 || max_q > (int64_t) words * 64) return {JAMHIP_EINVAL, "tree masks: fewer bits than max_q"};
    if (words > MAX_TOKENS / 64) return {JAMHIP_EUNSUPPORTED, "tree masks: bits beyond 32 bits"};
    return TAKEN;
}

inline Refusal refuse_path(const jamhip_tree* t, const void* tokens, const void* picked, const jamhip_tree_path* p) {
    if (!p) return {JAMHIP_EINVAL, "tree_accept: null path"};
    if (p->ld_path < 0 || (p->ld_path > 0 && !p->path)) return {JAMHIP_EINVAL, "tree_accept: null or negative path"};
    if (!p->accepted || !p->next || (t->n_tokens > 0 && (!tokens || !picked))) return {JAMHIP_EINVAL, "tree_accept: null array"};
    if ((p->lens_out != nullptr) && !p->lens) return {JAMHIP_EINVAL, "tree_accept: lens_out without lens"};
    if ((p->move_from != nullptr) != (p->move_to != nullptr) || (p->move_from && !p->slots))
        return {JAMHIP_EINVAL, "tree_accept: move_from and move_to go together, with slots"};
    if (p->ld_path > MAX_TOKENS) return {JAMHIP_EUNSUPPORTED, "tree_accept: paths beyond 32 bits"};
    return TAKEN;
}

// `caches` of one shape, which the caller has looked at one by one
inline Refusal refuse_move(const jamhip_kv_cache* caches, int n_caches, const void* offsets, int n_groups, const void* from, const void* to, int n) {
    if (n_caches < 0 || n_groups < 0 || n < 0 || (n_caches > 0 && !caches)) return {JAMHIP_EINVAL, "kv_move: null caches or negative count"};
    if (n > 0 && n_groups > 0 && (!offsets || !from || !to)) return {JAMHIP_EINVAL, "kv_move: null array"};
    for (int i = 1; i < n_caches; i++)
        if (caches[i].type != caches[0].type || caches[i].kv_heads != caches[0].kv_heads || caches[i].head_dim != caches[0].head_dim ||
            caches[i].page_tokens != caches[0].page_tokens || caches[i].n_pages != caches[0].n_pages)
            return {JAMHIP_EINVAL, "kv_move: caches of different shapes"};
    if (n > MAX_TOKENS || n_groups > MAX_SEQS) return {JAMHIP_EUNSUPPORTED, "kv_move: more than 2^20 groups, or entries beyond 32 bits"};
    return TAKEN;
}

}  // namespace jamhip
