"""A step of decoding with drafted trees, as cases that can be timed and checked.

A caller is an inference engine on one MI355X that keeps its keys and values in the paged cache of ``qxotic_amd.jam.HipJAM`` and drafts a
small tree of tokens for every sequence, which the model then looks at in one pass. Each kind of case is one operator of that step:

* ``resize``: pages are handed out and taken back so that every sequence holds its new length, and every new token gets its slot.
* ``masks``: which drafted tokens each drafted token sees (itself and its ancestors), and the positions to rotate it by.
* ``attn``: attention of the drafted tokens over the cache: the whole context, and of the drafted ones those that the mask holds.
* ``accept``: the drafted tokens that agree with what the model picked at their parents, a path from each tree's root.
* ``move``: the accepted tokens' entries copied to their places, in the caches of all layers (and read back where they are codes).

A drafted token's parent is its place among its sequence's drafted tokens, below its own, -1 for none. Token 0 of a sequence is the tree's
root: the token that the step before picked. Masks are 64-bit words, bit j of a row: the token sees its sequence's drafted token j.

A cache type is F16, Q8_0 or Q4_0 (blocks of 32 elements of one head of one token, an f16 scale each). What a quantised element stands for
is scale * code rounded to f16. A buffer has two planes: codes [page][kv head][token of the page][row], then scales
[page][kv head][token of the page][head_dim / 32].
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False


def listed():
    return [
        # a server's step: 64 sequences in mid-conversation get room for a tree of 32 tokens each
        {"name": "resize_64_trees", "kind": "resize", "seqs": 64, "grow": 32, "held": 4096, "page": 16, "ends": False},
        # prompts come in, others end: 512 sequences, about 130000 new tokens
        {"name": "resize_512_prompts", "kind": "resize", "seqs": 512, "grow": 640, "held": 8192, "page": 16, "ends": True},
        # the smallest call: one tree of 8 tokens
        {"name": "masks_1", "kind": "masks", "seqs": 1, "nodes": 8},
        # a large batch of full trees
        {"name": "masks_256_trees", "kind": "masks", "seqs": 256, "nodes": 64},
        # one conversation's tree of odd size, a short context: what counts is latency
        {"name": "attn_tree_1", "kind": "attn", "type": "F16", "heads": 32, "kv": 8, "dim": 128, "page": 16, "prefixes": 0, "prefix": 0, "seqs": 1,
         "nodes": 25, "own_min": 745, "own_max": 745, "window": 0, "sinks": False},
        # gpt-oss-shaped heads with their sinks, 32 sequences behind a shared prompt
        {"name": "attn_tree_shared_f16", "kind": "attn", "type": "F16", "heads": 64, "kv": 8, "dim": 64, "page": 16, "prefixes": 1, "prefix": 2048,
         "seqs": 32, "nodes": 16, "own_min": 40, "own_max": 700, "window": 0, "sinks": True},
        # a server's step: 64 conversations of up to 4096 tokens, 8-bit cache
        {"name": "attn_tree_64_q8_0", "kind": "attn", "type": "Q8_0", "heads": 32, "kv": 8, "dim": 128, "page": 16, "prefixes": 0, "prefix": 0,
         "seqs": 64, "nodes": 32, "own_min": 200, "own_max": 4096, "window": 0, "sinks": False},
        # four long documents, large trees, 4-bit cache
        {"name": "attn_tree_long_q4_0", "kind": "attn", "type": "Q4_0", "heads": 32, "kv": 8, "dim": 128, "page": 64, "prefixes": 0, "prefix": 0,
         "seqs": 4, "nodes": 63, "own_min": 20011, "own_max": 32771, "window": 0, "sinks": False},
        # one conversation's tree, as its step needs it
        {"name": "accept_1", "kind": "accept", "seqs": 1, "nodes": 25},
        # a large batch of full trees
        {"name": "accept_256_trees", "kind": "accept", "seqs": 256, "nodes": 64},
        # the entries of one sequence in the 8-bit caches of four layers
        {"name": "move_1_q8_0", "kind": "move", "type": "Q8_0", "layers": 4, "seqs": 1, "entries": 5, "kv": 8, "dim": 128, "page": 16},
        # those of 64 sequences in the f16 caches of a model's 32 layers
        {"name": "move_64_f16", "kind": "move", "type": "F16", "layers": 32, "seqs": 64, "entries": 6, "kv": 8, "dim": 128, "page": 16},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["resize", "masks", "attn", "accept", "move"], [3, 2, 8, 2, 3])[0]
    page = rng.choice([16, 16, 32, 64, 128])
    if kind == "resize":
        seqs = _log(rng, 1, 512)
        return {"kind": kind, "seqs": seqs, "grow": _log(rng, 1, min(32768, 512 * 640 // seqs)), "held": _log(rng, 16, 8192), "page": page,
                "ends": rng.random() < 0.5}
    if kind in ("masks", "accept"):
        nodes = _log(rng, 1, 200)
        return {"kind": kind, "seqs": _log(rng, 1, min(256, 256 * 64 * 64 // (nodes * nodes))), "nodes": nodes}
    dim, kv = rng.choice([64, 64, 128, 128, 128, 96, 256]), rng.choice([1, 2, 4, 8])
    kind_of = rng.choice(["F16", "Q8_0", "Q8_0", "Q4_0"])
    if kind == "move":
        seqs, entries = _log(rng, 1, 64), rng.randint(1, 8)
        layers = 1 if kind_of != "F16" else _log(rng, 1, max(1, min(32, 32 * 64 * 1024 // (seqs * kv * dim))))
        return {"kind": kind, "type": kind_of, "layers": layers if kind_of == "F16" else rng.randint(1, 4), "seqs": seqs, "entries": entries,
                "kv": kv, "dim": dim, "page": min(page, 32)}
    heads = kv * rng.choice([1, 2, 4, 4, 7, 8])
    nodes, seqs = _log(rng, 1, 130), _log(rng, 1, 64)
    prefixes = min(seqs, rng.choice([0, 0, 1, 1, 2, 4]))
    # the plain form keeps a score for every query, head and key: at most what the largest listed case keeps
    keys = max(32, 64 * 32 * 32 * 4096 // (seqs * nodes * heads) - nodes)
    own_max = _log(rng, 1, min(32768 if seqs <= 4 else 4096, keys))
    prefix = _log(rng, 16, max(17, min(8192, keys - own_max))) if prefixes else 0
    return {"kind": kind, "type": kind_of, "heads": heads, "kv": kv, "dim": dim, "page": page, "prefixes": prefixes, "prefix": prefix,
            "seqs": seqs, "nodes": nodes, "own_min": nodes, "own_max": own_max + nodes, "window": rng.choice([0, 0, 0, 128, 1000]),
            "sinks": rng.random() < 0.25}


# ---------------------------------------------------------------------------------------------- shapes
BLOCK = 32


def _row_bytes(kind, dim):
    return {"F16": 2 * dim, "Q8_0": dim, "Q4_0": dim // 2}[kind]


def _entry_bytes(case):
    """Bytes of one token's keys (or values) in the cache."""
    scales = 0 if case["type"] == "F16" else 2 * case["dim"] // BLOCK
    return case["kv"] * (_row_bytes(case["type"], case["dim"]) + scales)


def _words(case):
    return -(-case["nodes"] // 64)


def _lengths(case):
    """Drafted tokens and own tokens (those among them) of each sequence, and each prefix's sequences and length."""
    s, g = case["seqs"], case["prefixes"]
    at = [(i * 7919) % s for i in range(s)]   # 0 .. s - 1 in a mixed order where s is no multiple of 7919
    q = [case["nodes"] - (case["nodes"] * a) // (4 * s) for a in at]
    mine = [max(q[i], case["own_min"] + (case["own_max"] - case["own_min"]) * (a + 1) // s) for i, a in enumerate(at)]
    cuts = [s * j // g for j in range(g + 1)] if g else []
    lens = [case["prefix"] - 13 * j if case["prefix"] > 13 * j else case["prefix"] for j in range(g)]
    return q, mine, cuts, lens


def _tree(nodes, r):
    """Parents of one tree: a few children a node, most of them low in the order, as drafts from a model's favourites are."""
    parents = np.full(nodes, -1, np.int32)
    if nodes > 1:
        u = r.random(nodes - 1)
        i = np.arange(1, nodes)
        parents[1:] = np.where(r.random(nodes - 1) < 0.3, i - 1, np.floor(i * u * u)).astype(np.int32)
    return parents


def _batch_offsets(case):
    """Drafted tokens of each sequence, in a mixed order of sizes, summed."""
    s, n = case["seqs"], case["nodes"]
    return np.cumsum([0] + [n - (n * ((i * 7919) % s)) // (4 * s) for i in range(s)])


ENDS, CUT = -2, -1


def _growth(case):
    """What becomes of the batch's sequences, in some order: new tokens, all given back, or the last few cut (drafts that did not hold)."""
    i = np.arange(case["seqs"])
    grow = np.full(case["seqs"], case["grow"]) if case["grow"] < 64 else (i + 1) * case["grow"] // case["seqs"]
    return np.where(i % 20 < 3, ENDS, np.where(i % 20 < 6, CUT, grow)) if case["ends"] and case["seqs"] > 6 else grow


def _visible(case):
    """Query and key pairs over one head: what every tree's mask and the window leave."""
    q, mine, cuts, lens = _lengths(case)
    n = 0
    for i in range(case["seqs"]):
        ctx = mine[i] - q[i] + next((lens[j] for j in range(case["prefixes"]) if cuts[j] <= i < cuts[j + 1]), 0)
        depth = max(1, round(math.log2(q[i] + 1)))   # about what a tree of that many tokens has
        n += q[i] * (min(ctx + depth, case["window"]) if case["window"] else ctx + depth)
    return n


def work(case):
    kind = case["kind"]
    if kind == "resize":
        tokens = int(np.maximum(_growth(case), 0).sum())
        return {"bytes": case["seqs"] * 10 * 4 + tokens * 8 + tokens // case["page"] * 8, "flops": 8 * (tokens + case["seqs"])}
    if kind in ("masks", "accept"):
        n = int(_batch_offsets(case)[-1])
        if kind == "masks":
            return {"bytes": n * (4 + 8 + 8 * _words(case)) + 4 * case["seqs"], "flops": 8 * n}
        return {"bytes": n * (3 * 4 + 4 + 8) + case["seqs"] * 4 * (5 + case["nodes"]), "flops": 8 * n}
    if kind == "move":
        moved = 2 * 2 * case["layers"] * case["seqs"] * case["entries"] * _entry_bytes(case)
        if case["type"] != "F16":   # read again as f32
            moved += 2 * case["layers"] * case["seqs"] * case["entries"] * (_entry_bytes(case) + 4 * case["kv"] * case["dim"])
        return {"bytes": moved, "flops": 0}
    q, mine, cuts, lens = _lengths(case)
    tokens = sum(min(m, case["window"] + n) if case["window"] else m for n, m in zip(q, mine)) + sum(
        min(p, case["window"]) if case["window"] else p for p in lens)
    return {"bytes": 2 * tokens * _entry_bytes(case) + 2 * 4 * sum(q) * case["heads"] * case["dim"] + 8 * sum(q) * _words(case),
            "flops": 4 * _visible(case) * case["heads"] * case["dim"]}


# ----------------------------------------------------------------------------------------------- cache
def _decode(kind, codes, scales):
    """What the codes stand for, f32."""
    if kind == "F16":
        return codes.view(torch.float16).float()
    if kind == "Q8_0":
        q = codes.view(torch.int8).float().reshape(*scales.shape, BLOCK)
    else:
        b = codes.reshape(*scales.shape, 16)
        q = torch.cat([b & 15, b >> 4], -1).float() - 8
    return (q * scales.float()[..., None]).to(torch.float16).float().flatten(-2)


def _planes(buf, case):
    """Views of a cache buffer: codes [page, kv, token, row], scales [page, kv, token, dim / 32] or None."""
    row, p, kv = _row_bytes(case["type"], case["dim"]), case["page"], case["kv"]
    cut = case["pages"] * kv * p * row
    codes = buf[:cut].view(case["pages"], kv, p, row)
    return codes, None if case["type"] == "F16" else buf[cut:].view(torch.float16).view(case["pages"], kv, p, case["dim"] // BLOCK)


def _get(buf, case, slots):
    """[*slots, kv, dim] f32."""
    codes, scales = _planes(buf, case)
    page, at = slots // case["page"], slots % case["page"]
    return _decode(case["type"], codes[page, :, at], None if scales is None else scales[page, :, at])


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _i32(v):
    return torch.as_tensor(np.asarray(v, dtype=np.int32)).cuda()


def _new_buffer(case, g):
    """A cache buffer with entries in every slot: normal heads with a few strong elements, as codes and scales."""
    pages, kv, p, d = case["pages"], case["kv"], case["page"], case["dim"]
    rows = pages * kv * p
    strong = torch.where(torch.rand(d, generator=g, device="cuda") < 0.02, 3.0, 1.0)
    if case["type"] == "F16":
        out = torch.empty((rows, d), dtype=torch.float16, device="cuda")
        for part in out.split(1 << 18):
            part.copy_(torch.randn(part.shape, generator=g, device="cuda") * strong)
        return out.view(torch.uint8).flatten()
    blocks = d // BLOCK
    top = strong.view(blocks, BLOCK).amax(-1) * (2 + torch.rand((rows, blocks), generator=g, device="cuda"))
    share = 45 * strong / strong.view(blocks, BLOCK).amax(-1).repeat_interleave(BLOCK)
    codes = torch.empty((rows, _row_bytes(case["type"], d)), dtype=torch.uint8, device="cuda")
    for part in codes.split(1 << 18):
        if case["type"] == "Q8_0":
            x = torch.randn((part.shape[0], d), generator=g, device="cuda") * share
            part.copy_(x.round().clamp(-127, 127).to(torch.int8).view(torch.uint8))
        else:
            x = torch.randn((2, part.shape[0], d // 2), generator=g, device="cuda") * 2.8
            x = (x.round().clamp(-8, 7) + 8).to(torch.uint8)
            part.copy_(x[0] | (x[1] << 4))
    return torch.cat([codes.flatten(), (top / (127 if case["type"] == "Q8_0" else 8)).to(torch.float16).view(torch.uint8).flatten()])


# --------------------------------------------------------------------------------------------- prepare
def _prepare_resize(case, s, r):
    n, page = case["seqs"], case["page"]
    lens = r.integers(0, case["held"] + 1, n)
    rank = r.permutation(n)
    grow = _growth(case)[rank]
    target = lens + np.maximum(grow, 0)
    target = np.where(grow == ENDS, 0, np.where(grow == CUT, np.maximum(lens - r.integers(0, 40, n), 0), target))
    held = -(-lens // page) + (r.random(n) < 0.2)   # now and then a page more than the length needs
    most = -(-(case["held"] + case["grow"]) // page) + 1
    case["pages"], case["width"] = n * most + 7, most + 1
    case["tokens"] = int(np.maximum(grow, 0).sum()) + 5   # a batch padded by a few rows
    order = r.permutation(case["pages"]).astype(np.int32)
    table, used = np.full((n, case["width"]), -1, np.int32), 0
    for i, h in enumerate(held):
        table[i, :h] = order[used:used + h]
        used += h
    free = np.full(case["pages"], -1, np.int32)
    free[:case["pages"] - used] = order[used:]
    s.update(lens=_i32(lens), targets=_i32(target), held=_i32(held), n_free=_i32([case["pages"] - used]), free_pages=_i32(free),
             seq_pages=_i32(table), base=_i32(r.integers(0, 3000, n)))
    empty = lambda k: torch.empty(k, dtype=torch.int32, device="cuda")   # noqa: E731
    s.update(lens_out=empty(n), held_out=empty(n), n_free_out=empty(1), status=empty(n), q_offsets=empty(n + 1), pos=empty(case["tokens"]),
             slots=empty(case["tokens"]))


def _prepare_trees(case, s, r):
    off = _batch_offsets(case)
    n = int(off[-1])
    parents = np.concatenate([_tree(b - a, r) for a, b in zip(off, off[1:])])
    s.update(q_offsets=_i32(off), parents=_i32(parents))
    case["tokens"] = n
    seq = np.repeat(np.arange(case["seqs"]), np.diff(off))
    if case["kind"] == "masks":
        first = r.integers(0, 130000, case["seqs"])
        s["pos_in"] = _i32((first[seq] + np.arange(n) - off[seq]))
        s["pos"], s["masks"] = s["pos_in"].clone(), torch.empty((n, _words(case)), dtype=torch.int64, device="cuda")
        return
    tokens = r.integers(0, 128256, n)
    picked = r.integers(0, 128256, n)
    for t in range(n - 1, -1, -1):   # the model agrees with one of a node's children more often than not
        if parents[t] >= 0 and r.random() < 0.45:
            picked[off[seq[t]] + parents[t]] = tokens[t]
    s.update(tokens=_i32(tokens), picked=_i32(picked), lens=_i32(r.integers(0, 30000, case["seqs"])), slots=_i32(r.permutation(4 * n)[:n]))
    empty = lambda *k: torch.empty(k, dtype=torch.int32, device="cuda")   # noqa: E731
    s.update(path=empty(case["seqs"], case["nodes"]), accepted=empty(case["seqs"]), next=empty(case["seqs"]), lens_out=empty(case["seqs"]),
             move_from=empty(n), move_to=empty(n))


def _prepare_move(case, s, r, g):
    n, page = case["seqs"], case["page"]
    per = -(-16 // page)   # pages of a tree's drafted tokens, apart from the sequence's own
    case["pages"] = n * (per + 2) + 3
    order = r.permutation(case["pages"])
    counts = [max(1, case["entries"] - i % 3) for i in range(n)]
    src, dst = [], []
    for i, c in enumerate(counts):
        draft, mine = order[i * (per + 2):i * (per + 2) + per], order[i * (per + 2) + per:(i + 1) * (per + 2)]
        node = np.sort(r.permutation(16)[:c])
        at = r.integers(0, page) + np.arange(c)   # behind the sequence's last token, over a page's end now and then
        src += list(draft[node // page] * page + node % page)
        dst += list(mine[at // page] * page + at % page)
    s.update(offsets=_i32(np.cumsum([0] + counts)), move_from=_i32(src), move_to=_i32(dst))
    case["moved"] = len(src)
    s["k"] = [_new_buffer(case, g) for _ in range(case["layers"])]
    s["v"] = [_new_buffer(case, g) for _ in range(case["layers"])]
    if case["type"] != "F16":
        s["out"] = torch.empty((case["layers"], 2, len(src), case["kv"] * case["dim"]), device="cuda")


def _prepare_attn(case, s, r, g):
    q, mine, cuts, lens = _lengths(case)
    p, h, d = case["page"], case["heads"], case["dim"]
    need = [-(-v // p) for v in mine + lens]
    case["pages"] = sum(need) + 3
    s["k"], s["v"] = _new_buffer(case, g), _new_buffer(case, g)
    order = list(r.permutation(case["pages"]))

    def table(counts):
        t = np.zeros((max(1, len(counts)), max(counts, default=0) + 1), np.int32)
        for i, c in enumerate(counts):
            t[i, :c] = [order.pop() for _ in range(c)]
        return _i32(t)

    s["seq_pages"], s["prefix_pages"] = table(need[:len(mine)]), table(need[len(mine):])
    s["q_offsets"] = _i32([0] + list(np.cumsum(q)))
    s["seq_lens"], s["prefix_lens"], s["prefix_seqs"] = _i32(mine), _i32(lens or [0]), _i32(cuts or [0])
    s["tokens"], s["max_q"], s["max_seq"], s["max_prefix"] = sum(q), max(q), max(mine), max(lens, default=0)
    masks = np.zeros((sum(q), _words(case)), np.uint64)
    at = 0
    for n in q:
        parents = _tree(n, r)
        for i in range(n):
            if parents[i] >= 0:
                masks[at + i] = masks[at + parents[i]]
            masks[at + i, i // 64] |= np.uint64(1 << (i % 64))
        at += n
    s["masks"] = torch.from_numpy(masks.view(np.int64)).cuda()
    s["q"] = torch.randn((sum(q), h * d), generator=g, device="cuda") * 1.5
    s["scale"] = 1 / math.sqrt(d)
    s["sinks"] = torch.randn(h, generator=g, device="cuda") if case["sinks"] else None
    s["out"] = torch.empty((sum(q), h * d), device="cuda")


def prepare(case, seed):
    g, r = _gen(seed), np.random.default_rng(int(seed) & 0x7FFFFFFF)
    case = dict(case)
    s = {"case": case}
    if case["kind"] == "resize":
        _prepare_resize(case, s, r)
    elif case["kind"] in ("masks", "accept"):
        _prepare_trees(case, s, r)
    elif case["kind"] == "move":
        _prepare_move(case, s, r, g)
    else:
        _prepare_attn(case, s, r, g)
    torch.cuda.synchronize()   # the inputs were made on torch's own stream
    return s


# ---------------------------------------------------------------------------------------- plain forms
def _scan(x):
    """0 and the running sums of x, int64."""
    return torch.cat([torch.zeros(1, dtype=torch.int64, device=x.device), x.long().cumsum(0)])


def _plain_resize(s):
    case = s["case"]
    n, page, width, cap = case["seqs"], case["page"], case["width"], case["tokens"]
    lens, target, held, free_n = s["lens"].long(), s["targets"].long(), s["held"].long(), s["n_free"].long()
    table, free = s["seq_pages"].long(), s["free_pages"].long()
    dev, col = lens.device, torch.arange(width, device=lens.device)[None]
    need = (target + page - 1) // page
    back, take = (held - need).clamp(min=0), (need - held).clamp(min=0)
    new = (target - lens).clamp(min=0)
    off, taken = _scan(new), _scan(take)
    pushed = back.sum()
    # pages come back from the last sequence to the first, each one's last page first
    after = pushed - _scan(back)[1:]                             # pages given back by the sequences behind
    gone = (col >= need[:, None]) & (col < held[:, None])
    place = free_n + after[:, None] + (held[:, None] - 1 - col)
    size = free.numel()
    pool = torch.cat([free, free.new_zeros(1)])
    pool = pool.scatter(0, torch.where(gone, place, torch.full_like(place, size)).flatten(), table.flatten())
    have = free_n + pushed
    grows = (new > 0) | (take > 0)
    bad = grows & ((taken[1:] > have) | (off[1:] > cap) | (need > width))
    bad = grows & (bad.cumsum(0) > 0)                             # from the first that does not fit on, none grows
    got = torch.where(bad, torch.zeros_like(take), take)
    fresh = (col >= held[:, None]) & (col < (held + got)[:, None])
    which = have - 1 - (taken[:-1, None] + col - held[:, None])
    table = torch.where(fresh, pool[which.clamp(0, size)], table)
    t = torch.arange(cap, device=dev)
    seq = torch.searchsorted(off[1:].contiguous(), t, right=True)
    live, seq = seq < n, seq.clamp(max=n - 1)
    at = lens[seq] + t - off[seq]
    slot = table[seq, (at // page).clamp(0, width - 1)] * page + at % page
    i32 = lambda x: x.to(torch.int32)   # noqa: E731
    zero = torch.zeros_like(at)
    return {"lens": i32(torch.where(bad, lens, target)), "held": i32(torch.where(bad, held, need)),
            "n_free": i32(have - torch.where(bad, torch.zeros_like(take), take).sum()), "status": i32(bad), "q_offsets": i32(off.clamp(max=cap)),
            "pos": i32(torch.where(live, at + s["base"].long()[seq], zero)), "slots": i32(torch.where(live & ~bad[seq], slot, zero - 1)),
            "seq_pages": i32(table), "free_pages": i32(pool[:size])}


def _forest(s):
    """Tokens of the batch's trees side by side: (sequence, place) of each token, and parents [seqs, nodes] (-1 past the end)."""
    case, off = s["case"], s["q_offsets"].long()
    t = torch.arange(case["tokens"], device="cuda")
    seq = torch.searchsorted(off[1:].contiguous(), t, right=True)
    place = t - off[seq]
    parents = torch.full((case["seqs"], case["nodes"]), -1, dtype=torch.int64, device="cuda")
    parents[seq, place] = s["parents"].long()
    return seq, place, parents


def _plain_masks(s):
    case = s["case"]
    seq, place, jump = _forest(s)
    n = case["nodes"]
    sees = torch.eye(n, dtype=torch.bool, device="cuda").repeat(case["seqs"], 1, 1)
    for _ in range(max(1, (n - 1).bit_length())):   # what a token sees and what the token at its jump's end does
        to = jump.clamp(min=0)
        sees = sees | (sees.gather(1, to[..., None].expand(-1, -1, n)) & (jump >= 0)[..., None])
        jump = torch.where(jump >= 0, jump.gather(1, to), jump)
    rows = sees[seq, place]
    words = []
    for w in range(_words(case)):
        bits = rows[:, 64 * w:64 * (w + 1)].long()
        words.append((bits << torch.arange(bits.shape[1], device="cuda")).sum(-1))
    first = s["pos_in"].long()[s["q_offsets"].long()[seq]]
    return {"masks": torch.stack(words, -1), "pos": (first + rows.sum(-1) - 1).to(torch.int32)}


def _plain_accept(s):
    case = s["case"]
    seq, place, parents = _forest(s)
    n, m = case["seqs"], case["nodes"]
    tokens, picked = (torch.full((n, m), -1, dtype=torch.int64, device="cuda") for _ in range(2))
    tokens[seq, place], picked[seq, place] = s["tokens"].long(), s["picked"].long()
    off = s["q_offsets"].long()
    at, live = torch.zeros(n, dtype=torch.int64, device="cuda"), off[1:] > off[:-1]
    path = torch.full((n, m), -1, dtype=torch.int64, device="cuda")
    count, col = torch.zeros_like(at), torch.arange(m, device="cuda")[None]
    last = torch.full_like(at, -1)
    for i in range(m):
        path[:, i] = torch.where(live, at, path[:, i])
        count = count + live
        pick = picked.gather(1, at[:, None])
        last = torch.where(live, pick[:, 0], last)
        fits = (parents == at[:, None]) & (tokens == pick) & (col > 0) & live[:, None]
        live = fits.any(-1)
        at = torch.where(live, fits.int().argmax(-1), at)
    on = place < count[seq]
    slots = s["slots"].long()
    src = slots[(off[seq] + path[seq, place].clamp(min=0)).clamp(max=case["tokens"] - 1)]
    on = on & (path[seq, place] != place)
    i32 = lambda x: x.to(torch.int32)   # noqa: E731
    none = torch.full_like(slots, -1)
    return {"path": i32(path), "accepted": i32(count), "next": i32(last), "lens": i32(s["lens"].long() + count),
            "from": i32(torch.where(on, src, none)), "to": i32(torch.where(on, slots, none))}


def _plain_move(s):
    case = s["case"]
    src, dst = s["move_from"].long(), s["move_to"].long()
    p = case["page"]
    for buf in s["k"] + s["v"]:
        for plane in _planes(buf, case):
            if plane is not None:
                plane[dst // p, :, dst % p] = plane[src // p, :, src % p]
    return _moved(s, [torch.stack([_get(b[i], case, dst).flatten(1) for b in (s["k"], s["v"])]) for i in range(case["layers"])]
                  if case["type"] != "F16" else None)


def _moved(s, read):
    """The caches as they are (f16 values), or what their moved entries stand for."""
    if s["case"]["type"] == "F16":
        return {name: [b.view(torch.float16) for b in s[name]] for name in ("k", "v")}
    return torch.stack(read)


def _bits(masks, n):
    """[tokens, n] truth values of 64-bit words."""
    at = torch.arange(n, device=masks.device)
    return (masks[:, at // 64] >> (at % 64)) & 1 == 1


def _plain_attn(s):
    case = s["case"]
    n_seqs, kv, d, grp, page = case["seqs"], case["kv"], case["dim"], case["heads"] // case["kv"], case["page"]
    n, dev, width = s["tokens"], "cuda", s["max_q"]
    off, lens = s["q_offsets"].long(), s["seq_lens"].long()
    tok = torch.arange(n, device=dev)
    seq = torch.searchsorted(off[1:].contiguous(), tok, right=True)
    row = tok - off[seq]
    cap_p, cap_o = s["max_prefix"], s["max_seq"]
    slots_of = lambda t, cap: t.long()[:, torch.arange(cap, device=dev) // page] * page + torch.arange(cap, device=dev) % page   # noqa: E731
    own_slots = slots_of(s["seq_pages"], cap_o)
    base = torch.zeros(n_seqs, dtype=torch.int64, device=dev)
    parts = [(own_slots, False)]
    if case["prefixes"]:
        of = torch.searchsorted(s["prefix_seqs"].long()[1:].contiguous(), torch.arange(n_seqs, device=dev), right=True)
        base = s["prefix_lens"].long()[of]
        parts.insert(0, (slots_of(s["prefix_pages"], cap_p)[of], True))
    q = torch.zeros((n_seqs, width, kv, grp, d), device=dev)
    q[seq, row] = s["q"].view(n, kv, grp, d) * s["scale"]
    q = q.permute(0, 2, 1, 3, 4).reshape(n_seqs, kv, width * grp, d)
    ctx = lens - (off[1:] - off[:-1])                             # own tokens before the drafted ones
    seen = []
    for slots, shared in parts:
        at = torch.arange(slots.shape[1], device=dev)[None]
        if shared:
            seen.append((at < base[:, None])[:, None].expand(-1, width, -1))
            continue
        tree = torch.zeros((n_seqs, width, width), dtype=torch.bool, device=dev)
        tree[seq, row] = _bits(s["masks"], width)
        j = (at - ctx[:, None]).clamp(0, width - 1)
        inside = (at >= ctx[:, None]) & (at < lens[:, None])
        seen.append((at < ctx[:, None])[:, None] | (inside[:, None] & tree.gather(2, j[:, None].expand(-1, width, -1))))
    vis = torch.cat(seen, -1)
    if case["window"]:   # the last `window` of the keys that it sees
        vis = vis & (vis.flip(-1).cumsum(-1, dtype=torch.int32).flip(-1) <= case["window"])
    keys = torch.cat([_get(s["k"], case, slots) for slots, _ in parts], 1).transpose(1, 2)   # [seq, kv, keys, dim]
    x = (q @ keys.transpose(2, 3)).view(n_seqs, kv, width, grp, -1)
    del keys
    x.masked_fill_(~vis[:, None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        top = torch.maximum(top, s["sinks"].view(1, kv, 1, grp, 1))
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(s["sinks"].view(1, kv, 1, grp, 1) - top)
    values = torch.cat([_get(s["v"], case, slots) for slots, _ in parts], 1).transpose(1, 2).contiguous()
    out = (x.flatten(2, 3) @ values).view(n_seqs, kv, width, grp, d)
    out = torch.where(total > 0, out / total, torch.zeros_like(out)).permute(0, 2, 1, 3, 4)
    return out[seq, row].reshape(n, -1)


# ------------------------------------------------------------------------------------------------- run
_JAM = None


def _jam():
    """The program's one context."""
    global _JAM
    if _JAM is None:
        from qxotic_amd.jam import HipJAM
        _JAM = HipJAM(0)
    return _JAM


def _ok(status):
    if status:
        raise RuntimeError(_jam().last_error())


def _handles(s):
    """The descriptors that a program keeps beside its buffers, made once for a state."""
    if "handles" not in s:
        from qxotic_amd.jam import JAM, AttnBatch, KvCache, KvPages, Tree, TreePath
        case, h = s["case"], {}
        ptr = lambda name: None if s.get(name) is None else s[name].data_ptr()   # noqa: E731
        kind = case["kind"]
        if kind == "resize":
            h["pages"] = KvPages(n_seqs=case["seqs"], n_tokens=case["tokens"], page_tokens=case["page"], n_pages=case["pages"],
                                 free_cap=case["pages"], ld_seq_pages=case["width"],
                                 **{k: ptr(k) for k in ("lens", "targets", "base", "held", "n_free", "free_pages", "seq_pages", "lens_out",
                                                        "held_out", "n_free_out", "status", "q_offsets", "pos", "slots")})
        if kind in ("masks", "accept"):
            h["tree"] = Tree(n_tokens=case["tokens"], n_seqs=case["seqs"], max_q=case["nodes"], q_offsets=ptr("q_offsets"), parents=ptr("parents"))
        if kind == "accept":
            h["path"] = TreePath(ld_path=case["nodes"], path=ptr("path"), accepted=ptr("accepted"), next=ptr("next"), lens=ptr("lens"),
                                 lens_out=ptr("lens_out"), slots=ptr("slots"), move_from=ptr("move_from"), move_to=ptr("move_to"))
        if "type" in case:
            cache = lambda k, v: KvCache(type=getattr(JAM, case["type"]), kv_heads=case["kv"], head_dim=case["dim"],   # noqa: E731
                                         page_tokens=case["page"], n_pages=case["pages"], k=k.data_ptr(), v=v.data_ptr())
            if kind == "move":
                h["caches"] = (KvCache * case["layers"])(*(cache(k, v) for k, v in zip(s["k"], s["v"])))
            else:
                h["cache"] = cache(s["k"], s["v"])
                h["batch"] = AttnBatch(n_tokens=s["tokens"], n_seqs=case["seqs"], n_prefixes=case["prefixes"], max_q=s["max_q"],
                                       max_seq_len=s["max_seq"], max_prefix_len=s["max_prefix"], q_offsets=ptr("q_offsets"),
                                       seq_lens=ptr("seq_lens"), seq_pages=ptr("seq_pages"), ld_seq_pages=s["seq_pages"].shape[1],
                                       prefix_seqs=ptr("prefix_seqs"), prefix_lens=ptr("prefix_lens"), prefix_pages=ptr("prefix_pages"),
                                       ld_prefix_pages=s["prefix_pages"].shape[1])
        s["handles"] = h
    return s["handles"]


def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        return {"resize": _plain_resize, "masks": _plain_masks, "attn": _plain_attn, "accept": _plain_accept, "move": _plain_move}[kind](s)
    jam, h = _jam(), _handles(s)
    if kind == "resize":
        _ok(jam.kv_resize(h["pages"]))
        return {"lens": s["lens_out"], "held": s["held_out"], "n_free": s["n_free_out"], "status": s["status"], "q_offsets": s["q_offsets"],
                "pos": s["pos"], "slots": s["slots"], "seq_pages": s["seq_pages"], "free_pages": s["free_pages"]}
    if kind == "masks":
        _ok(jam.tree_masks(h["tree"], s["masks"].data_ptr(), _words(case), s["pos"].data_ptr()))
        return {"masks": s["masks"], "pos": s["pos"]}
    if kind == "accept":
        _ok(jam.tree_accept(h["tree"], s["tokens"].data_ptr(), s["picked"].data_ptr(), h["path"]))
        return {"path": s["path"], "accepted": s["accepted"], "next": s["next"], "lens": s["lens_out"], "from": s["move_from"], "to": s["move_to"]}
    if kind == "move":
        _ok(jam.kv_move(h["caches"], case["layers"], s["offsets"].data_ptr(), case["seqs"], s["move_from"].data_ptr(), s["move_to"].data_ptr(),
                        case["moved"]))
        if case["type"] == "F16":
            return _moved(s, None)
        kd = case["kv"] * case["dim"]
        for i in range(case["layers"]):
            _ok(jam.kv_read(h["caches"][i], s["move_to"].data_ptr(), case["moved"], s["out"][i, 0].data_ptr(), kd, s["out"][i, 1].data_ptr(), kd))
        return s["out"]
    ld = case["heads"] * case["dim"]
    _ok(jam.attn_tree(h["cache"], h["batch"], s["masks"].data_ptr(), _words(case), s["q"].data_ptr(), ld, case["heads"], s["scale"],
                      s["out"].data_ptr(), ld, window=case["window"], sinks_dev=None if s["sinks"] is None else s["sinks"].data_ptr()))
    return s["out"]


# --------------------------------------------------------------------------------------------- exact
def _np(t):
    return t.cpu().numpy()


RESIZED = ("lens", "held", "n_free", "status", "q_offsets", "pos", "slots", "seq_pages", "free_pages")   # the outputs in their order


def _exact_resize(s):
    """Sequence by sequence on the host, the pages on a list."""
    case, page = s["case"], s["case"]["page"]
    lens, target, held, base = (_np(s[k]).astype(int).tolist() for k in ("lens", "targets", "held", "base"))
    pool, table = _np(s["free_pages"]).tolist(), _np(s["seq_pages"]).copy()
    top = int(s["n_free"][0])
    for i in reversed(range(case["seqs"])):
        for c in range(held[i] - 1, -(-target[i] // page) - 1, -1):
            pool[top] = int(table[i, c])
            top += 1
    asked, rows, out, full = 0, 0, {k: [] for k in ("lens", "held", "status", "pos", "slots")}, False
    have, offs = top, [0]
    for i in range(case["seqs"]):
        need, new = -(-target[i] // page), max(0, target[i] - lens[i])
        more = max(0, need - held[i])
        asked, rows = asked + more, rows + new
        full = full or (max(new, more) > 0 and (asked > have or rows > case["tokens"] or need > case["width"]))
        refused = full and max(new, more) > 0
        if not refused:
            for c in range(more):
                table[i, held[i] + c] = pool[have - 1 - (asked - more + c)]
            top -= more
        for p in range(lens[i], lens[i] + new):
            out["pos"].append(base[i] + p)
            out["slots"].append(-1 if refused else int(table[i, p // page]) * page + p % page)
        out["lens"].append(lens[i] if refused else target[i])
        out["held"].append(held[i] if refused else need)
        out["status"].append(int(refused))
        offs.append(min(rows, case["tokens"]))
    pad = case["tokens"] - len(out["pos"])
    out["pos"] += [0] * pad
    out["slots"] += [-1] * pad
    out.update(n_free=[top], q_offsets=offs, seq_pages=table, free_pages=pool)
    return {k: torch.as_tensor(np.asarray(out[k], np.int32)) for k in RESIZED}


def _exact_trees(s):
    case = s["case"]
    off, parents = _np(s["q_offsets"]), _np(s["parents"])
    if case["kind"] == "masks":
        pos, first = np.zeros(case["tokens"], np.int32), _np(s["pos_in"])
        masks = np.zeros((case["tokens"], _words(case)), np.uint64)
        for a, b in zip(off, off[1:]):
            for t in range(a, b):
                at, steps = t - a, 0
                while at >= 0:
                    masks[t, at // 64] |= np.uint64(1) << np.uint64(at % 64)
                    at, steps = parents[a + at], steps + 1
                pos[t] = first[a] + steps - 1
        return {"masks": torch.from_numpy(masks.view(np.int64)), "pos": torch.from_numpy(pos)}
    tokens, picked, slots, lens = (_np(s[k]) for k in ("tokens", "picked", "slots", "lens"))
    n = case["seqs"]
    path, accepted, after = np.full((n, case["nodes"]), -1, np.int32), np.zeros(n, np.int32), np.full(n, -1, np.int32)
    src, dst = np.full(case["tokens"], -1, np.int32), np.full(case["tokens"], -1, np.int32)
    for i, (a, b) in enumerate(zip(off, off[1:])):
        walk = [0] if b > a else []
        while walk:
            after[i] = picked[a + walk[-1]]
            more = [c for c in range(walk[-1] + 1, b - a) if parents[a + c] == walk[-1] and tokens[a + c] == after[i]]
            if not more:
                break
            walk.append(more[0])
        for k, c in enumerate(walk):
            path[i, k] = c
            if c != k:
                src[a + k], dst[a + k] = slots[a + c], slots[a + k]
        accepted[i] = len(walk)
    out = {"path": path, "accepted": accepted, "next": after, "lens": lens + accepted, "from": src, "to": dst}
    return {k: torch.from_numpy(v) for k, v in out.items()}


def _exact_entries(buf, case, slots):
    """The cache's entries at `slots` from the layout's definition, element by element: [slots, kv, dim] in 64 bits."""
    kv, d, page, row = case["kv"], case["dim"], case["page"], _row_bytes(case["type"], case["dim"])
    at = ((slots // page)[:, None] * kv + torch.arange(kv, device="cuda")) * page + (slots % page)[:, None]
    e = torch.arange(d, device="cuda")
    if case["type"] == "F16":
        return buf.view(torch.float16)[at[..., None] * d + e].double()
    if case["type"] == "Q8_0":
        code = buf.view(torch.int8)[at[..., None] * row + e].double()
    else:
        code = ((buf[at[..., None] * row + e // BLOCK * 16 + e % 16] >> (e % BLOCK // 16 * 4)) & 15).double() - 8
    scale = buf[case["pages"] * kv * page * row:].view(torch.float16)[at[..., None] * (d // BLOCK) + e // BLOCK]
    return (code * scale.double()).half().double()


def _exact_move(s):
    case = s["case"]
    src, dst = s["move_from"].long(), s["move_to"].long()
    if case["type"] != "F16":
        return torch.stack([torch.stack([_exact_entries(b[i], case, src).flatten(1) for b in (s["k"], s["v"])]) for i in range(case["layers"])])
    out = {"k": [], "v": []}
    head = torch.arange(case["kv"], device="cuda")
    line = lambda slots: ((slots // case["page"])[:, None] * case["kv"] + head) * case["page"] + (slots % case["page"])[:, None]   # noqa: E731
    for name in out:
        for b in s[name]:
            x = b.view(torch.float16).clone().view(-1, case["dim"])
            x[line(dst).flatten()] = x[line(src).flatten()]
            out[name].append(x.flatten())
    return out


def _exact_attn(s):
    """One sequence and key head at a time, its visible keys by name."""
    case = s["case"]
    q, mine, cuts, lens = _lengths(case)
    kv, d, grp, page = case["kv"], case["dim"], case["heads"] // case["kv"], case["page"]
    out = torch.zeros((sum(q), kv, grp, d), dtype=torch.float64, device="cuda")
    rows, masks = s["q"].double().view(sum(q), kv, grp, d), _np(s["masks"]).view(np.uint64)
    start = 0

    def entries(pages, length):
        slots = (pages.long()[:, None] * page + torch.arange(page, device="cuda")).flatten()[:length]
        return _exact_entries(s["k"], case, slots), _exact_entries(s["v"], case, slots)

    held = [entries(s["prefix_pages"][j], lens[j]) for j in range(case["prefixes"])]
    for i in range(case["seqs"]):
        k, v = entries(s["seq_pages"][i], mine[i])
        j = next((j for j in range(case["prefixes"]) if cuts[j] <= i < cuts[j + 1]), None)
        if j is not None:
            k, v = torch.cat([held[j][0], k]), torch.cat([held[j][1], v])
        length = k.shape[0]
        ctx = length - q[i]
        ok = np.zeros((q[i], length), bool)
        for t in range(q[i]):
            words = masks[start + t]
            see = list(range(ctx)) if not case["window"] else list(range(max(0, ctx - case["window"]), ctx))
            see += [ctx + b for b in range(q[i]) if int(words[b // 64]) >> (b % 64) & 1]
            ok[t, see[-case["window"]:] if case["window"] else see] = True
        ok = torch.from_numpy(ok).cuda()
        for c in range(kv):
            x = (rows[start:start + q[i], c].reshape(-1, d) @ k[:, c].T).view(q[i], grp, length) * s["scale"]
            x = torch.where(ok[:, None], x, torch.full_like(x, -math.inf))
            if s["sinks"] is not None:
                sink = s["sinks"].double().view(kv, grp)[c].view(1, grp, 1).expand(q[i], grp, 1)
                w = torch.softmax(torch.cat([x, sink], -1), -1)[..., :-1]
            else:
                w = torch.softmax(x, -1)
            out[start:start + q[i], c] = (w.reshape(-1, length) @ v[:, c]).view(q[i], grp, d)
        start += q[i]
    return out.reshape(sum(q), -1)


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["case"]["kind"]
    return {"resize": _exact_resize, "masks": _exact_trees, "accept": _exact_trees, "move": _exact_move, "attn": _exact_attn}[kind](s)
