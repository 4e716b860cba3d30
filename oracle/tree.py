"""A step with drafted trees from its definitions (numpy, lists): page tables and slots, masks, attention, the accepted path."""
from __future__ import annotations

import numpy as np


def resize(page, lens, targets, base, held, free, table, n_tokens):
    """`free` a list of pages, `table` lists of pages (ld entries each, changed). Returns what jamhip_kv_resize writes, and the list."""
    free, table = list(free), [list(r) for r in table]
    ld, n = len(table[0]) if table else 0, len(lens)
    lens, targets, held = [max(v, 0) for v in lens], [max(v, 0) for v in targets], [min(max(v, 0), ld) for v in held]
    need = [-(-t // page) for t in targets]
    for s in reversed(range(n)):
        for c in reversed(range(need[s], held[s])):
            free.append(table[s][c])
    rows, full = 0, False
    out = dict(lens=[], held=[], status=[], q_offsets=[0], pos=[], slots=[])
    for s in range(n):
        new, take = max(0, targets[s] - lens[s]), max(0, need[s] - held[s])
        rows += new
        full = full or ((new > 0 or take > 0) and (take > len(free) or rows > n_tokens or need[s] > ld))
        refused = full and (new > 0 or take > 0)
        if not refused:
            for c in range(held[s], need[s]):
                table[s][c] = free.pop()
        out["lens"].append(lens[s] if refused else targets[s])
        out["held"].append(min(held[s], need[s]) if refused else need[s])
        out["status"].append(int(refused))
        out["q_offsets"].append(min(rows, n_tokens))
        for p in range(lens[s], lens[s] + min(new, n_tokens)):
            out["pos"].append(base[s] + p)
            out["slots"].append(-1 if refused else table[s][p // page] * page + p % page)
    out["pos"], out["slots"] = out["pos"][:n_tokens], out["slots"][:n_tokens]
    pad = n_tokens - len(out["pos"])
    out["pos"] += [0] * pad
    out["slots"] += [-1] * pad
    out.update(n_free=[len(free)], seq_pages=table)
    return out, free


def clean(parents):
    """Parents of one tree with those that are none as -1."""
    return [p if 0 <= p < i else -1 for i, p in enumerate(parents)]


def ancestors(parents):
    """For each token the set of those that it sees: itself and its ancestors."""
    out = []
    for i, p in enumerate(clean(parents)):
        out.append(({i} | out[p]) if p >= 0 else {i})
    return out


def words(sets, n_words):
    """Rows of 64-bit words."""
    out = np.zeros((len(sets), n_words), np.uint64)
    for i, s in enumerate(sets):
        for j in s:
            out[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out


def walk(parents, tokens, picked, longest):
    """Accepted places, and what is picked after the last."""
    if not len(parents) or not longest:
        return [], -1
    parents, path = clean(parents), [0]
    while len(path) < longest:
        more = [c for c in range(path[-1] + 1, len(parents)) if parents[c] == path[-1] and tokens[c] == picked[path[-1]]]
        if not more:
            break
        path.append(more[0])
    return path, int(picked[path[-1]])


def accept(parents, tokens, picked, slots, longest):
    """walk, of a sequence whose tokens have these slots: one without a slot for its root was refused, and stays as it was."""
    if len(parents) and slots[0] < 0:
        return [], int(tokens[0])
    return walk(parents, tokens, picked, longest)


def seen(ctx, nq, bits, window=0):
    """The keys, in order, that a query token sees whose row has these bits: `ctx` context keys, then nq drafted ones."""
    keys = list(range(ctx)) + [ctx + j for j in sorted(bits) if 0 <= j < nq]
    return keys[-window:] if window else keys


def attention(q, k, v, keys, scale, sinks=None):
    """One sequence and key head: q [n, grp, dim], k, v [keys, dim], keys[i] what token i sees. Returns (out [n, grp, dim], the largest
    scale * sum |q k| of a visible key [n, grp], largest |v|)."""
    n, grp, dim = q.shape
    out, mass, big = np.zeros((n, grp, dim)), np.zeros((n, grp)), np.zeros((n, grp))
    q, k, v = (a.astype(np.float64) for a in (q, k, v))
    for i in range(n):
        if not keys[i]:
            continue
        kk, vv = k[keys[i]], v[keys[i]]
        s = scale * (q[i] @ kk.T)
        top = s.max(-1, keepdims=True)
        if sinks is not None:
            top = np.maximum(top, sinks[:, None])
        w = np.exp(s - top)
        total = w.sum(-1, keepdims=True) + (np.exp(sinks[:, None] - top) if sinks is not None else 0)
        out[i] = (w @ vv) / total
        mass[i] = scale * (np.abs(q[i]) @ np.abs(kk).T).max(-1)
        big[i] = np.abs(vv).max()
    return out, mass, big
