"""The decode-side operators around the matmuls, as cases that can be timed and checked.

A caller is an inference engine on one MI355X whose projections run through ``qxotic_amd.jam.HipJAM``. Between the q|k|v
projection and the output projection, and after the output head, it needs four more things, and each is a kind of case:

* ``rope``: RMS norm of every query and key head and the position rotation, in one pass over the projection's rows.
* ``write``: the same, with keys and values quantised into the paged cache as they are made, and the new entries read back
  (what an engine does that keeps a prompt's cache on the host too).
* ``read``: a stretch of the cache read back.
* ``attn``: attention of a ragged batch over the cache: groups of sequences share a prefix, which is read once for the
  whole group, and each sequence has tokens of its own after it. One query token per sequence (decode) or many (prompt).
* ``sample``: the next token of each row of logits: temperature, top-k, top-p and min-p, from a given random number.

A cache type is F16, Q8_0 or Q4_0 (blocks of 32 elements of one head of one token, an f16 scale each). What a quantised
element stands for is scale * code rounded to f16. The cache is two planes in one buffer, for keys and for values each:
codes [page][kv head][token of the page][row], then scales [page][kv head][token of the page][head_dim / 32].
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False


def listed():
    return [
        # the smallest call: one token's heads normed and rotated (32 query and 8 key heads of 128)
        {"name": "rope_decode_1", "kind": "rope", "n": 1, "heads": 32, "kv": 8, "dim": 128, "rot": 128, "pairs": "halves", "norm": True},
        # a long prompt of gpt-oss-shaped heads, no head norm, far positions
        {"name": "rope_prompt_4096", "kind": "rope", "n": 4096, "heads": 64, "kv": 8, "dim": 64, "rot": 64, "pairs": "halves", "norm": False},
        # a decode step of 64 sequences into an 8-bit cache
        {"name": "write_q8_0_64", "kind": "write", "type": "Q8_0", "n": 64, "heads": 32, "kv": 8, "dim": 128, "rot": 128,
         "pairs": "halves", "norm": True, "page": 16},
        # a prompt into a 4-bit cache
        {"name": "write_q4_0_2048", "kind": "write", "type": "Q4_0", "n": 2048, "heads": 32, "kv": 8, "dim": 128, "rot": 128,
         "pairs": "halves", "norm": True, "page": 64},
        # a prompt of odd length into an f16 cache, a quarter of wide heads rotated, neighbours paired
        {"name": "write_f16_333", "kind": "write", "type": "F16", "n": 333, "heads": 16, "kv": 2, "dim": 256, "rot": 64,
         "pairs": "neighbours", "norm": True, "page": 32},
        # a 16k-token prompt's 8-bit cache read back
        {"name": "read_q8_0_16384", "kind": "read", "type": "Q8_0", "n": 16384, "kv": 8, "dim": 128, "page": 16},
        # one sequence's next token, a short context: what counts is latency
        {"name": "attn_one_sequence", "kind": "attn", "type": "F16", "heads": 32, "kv": 8, "dim": 128, "page": 16, "prefixes": 1,
         "prefix": 700, "seqs": 1, "q": 1, "own_min": 45, "own_max": 45, "window": 0, "sinks": False},
        # a server's decode step: 64 conversations behind one long system prompt
        {"name": "attn_decode_64_prefix_8192", "kind": "attn", "type": "Q8_0", "heads": 32, "kv": 8, "dim": 128, "page": 16,
         "prefixes": 1, "prefix": 8192, "seqs": 64, "q": 1, "own_min": 33, "own_max": 1024, "window": 0, "sinks": False},
        # four long documents with eight questions each, 4-bit cache
        {"name": "attn_documents_q4_0", "kind": "attn", "type": "Q4_0", "heads": 32, "kv": 8, "dim": 128, "page": 64, "prefixes": 4,
         "prefix": 24001, "seqs": 32, "q": 1, "own_min": 5, "own_max": 300, "window": 0, "sinks": False},
        # eight prompts of up to 256 tokens behind a shared one, gpt-oss-shaped heads with their sinks
        {"name": "attn_prompts_256", "kind": "attn", "type": "F16", "heads": 64, "kv": 8, "dim": 64, "page": 16, "prefixes": 1,
         "prefix": 4096, "seqs": 8, "q": 256, "own_min": 256, "own_max": 256, "window": 0, "sinks": True},
        # one row of a Llama-3 vocabulary, as one conversation's step needs it
        {"name": "sample_1", "kind": "sample", "rows": 1, "vocab": 128256, "spread": 2.5, "filters": "all"},
        # 64 rows whose requests ask for different filters
        {"name": "sample_64", "kind": "sample", "rows": 64, "vocab": 128256, "spread": 2.5, "filters": "mixed"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    dim = rng.choice([64, 64, 128, 128, 128, 96, 256])
    kv = rng.choice([1, 2, 4, 8])
    return dim, kv, kv * rng.choice([1, 2, 4, 4, 7, 8])


def draw(rng):
    kind = rng.choices(["rope", "write", "read", "attn", "sample"], [2, 4, 2, 7, 4])[0]
    if kind in ("rope", "write"):
        dim, kv, heads = _heads(rng)
        case = {"kind": kind, "n": _log(rng, 1, min(4096, 4096 * 4608 // ((heads + kv) * dim))), "heads": heads, "kv": kv, "dim": dim,
                "rot": rng.choice([dim, dim, dim // 2]), "pairs": rng.choice(["halves", "halves", "neighbours"]), "norm": rng.random() < 0.7}
        if kind == "write":
            case.update({"type": rng.choice(["F16", "Q8_0", "Q8_0", "Q4_0"]), "page": rng.choice([16, 32, 64, 128])})
        return case
    if kind == "read":
        dim, kv, _ = _heads(rng)
        return {"kind": kind, "type": rng.choice(["F16", "Q8_0", "Q4_0"]), "n": _log(rng, 1, 16384 * 1024 // (kv * dim)), "kv": kv, "dim": dim,
                "page": rng.choice([16, 32, 64, 128])}
    if kind == "sample":
        rows = _log(rng, 1, 64)
        return {"kind": kind, "rows": rows, "vocab": _log(rng, 1000, min(262144, 64 * 128256 // rows)), "spread": rng.choice([1.0, 2.5, 4.0]),
                "filters": rng.choice(["none", "all", "top_k", "top_p", "min_p", "mixed", "mixed"])}
    dim, kv, heads = _heads(rng)
    q = rng.choice([1, 1, 1, _log(rng, 2, 8), _log(rng, 16, 512)])
    seqs = _log(rng, 1, 64 if q < 16 else 8)
    prefixes = min(seqs, rng.choice([0, 1, 1, 1, 2, 4]))
    # the plain form keeps a score for every query, head and key: at most what the largest listed prompt case keeps
    keys = 256 * 8 * 64 * 4352 // (seqs * q * heads)
    own_max = q + _log(rng, 1, max(2, min(2048 if seqs <= 16 else 1024, keys // 2 - q)))
    keys -= own_max
    prefix = _log(rng, 16, max(17, min(32768 // max(1, prefixes), keys))) if prefixes else 0
    return {"kind": kind, "type": rng.choice(["F16", "Q8_0", "Q8_0", "Q4_0"]), "heads": heads, "kv": kv, "dim": dim,
            "page": rng.choice([16, 32, 64, 128]), "prefixes": prefixes, "prefix": prefix, "seqs": seqs, "q": q, "own_min": q,
            "own_max": own_max, "window": rng.choice([0, 0, 0, 128, 1000]), "sinks": rng.random() < 0.25}


# ---------------------------------------------------------------------------------------------- shapes
BLOCK = 32


def _row_bytes(kind, dim):
    return {"F16": 2 * dim, "Q8_0": dim, "Q4_0": dim // 2}[kind]


def _entry_bytes(case):
    """Bytes of one token's keys (or values) in the cache."""
    scales = 0 if case["type"] == "F16" else 2 * case["dim"] // BLOCK
    return case["kv"] * (_row_bytes(case["type"], case["dim"]) + scales)


def _lengths(case):
    """Query tokens and own tokens of each sequence, and each prefix's sequences and length."""
    s, g = case["seqs"], case["prefixes"]
    at = [(i * 7919) % s for i in range(s)]   # 0 .. s - 1 in a mixed order where s is no multiple of 7919
    q = [case["q"] if case["q"] < 16 else case["q"] - (case["q"] * a) // (4 * s) for a in at]
    mine = [max(q[i], case["own_min"] + (case["own_max"] - case["own_min"]) * (a + 1) // s) for i, a in enumerate(at)]
    cuts = [s * j // g for j in range(g + 1)] if g else []
    lens = [case["prefix"] - 13 * j if case["prefix"] > 13 * j else case["prefix"] for j in range(g)]
    return q, mine, cuts, lens


def _pairs_seen(case):
    """Query and key pairs that the mask leaves, over one head."""
    q, mine, cuts, lens = _lengths(case)
    n = 0
    for i in range(case["seqs"]):
        before = next((lens[j] for j in range(case["prefixes"]) if cuts[j] <= i < cuts[j + 1]), 0)
        for t in range(q[i]):
            seen = before + mine[i] - q[i] + t + 1
            n += min(seen, case["window"]) if case["window"] else seen
    return n


def work(case):
    kind = case["kind"]
    if kind == "sample":
        return {"bytes": 4 * case["rows"] * (case["vocab"] + 7), "flops": 3 * case["rows"] * case["vocab"]}
    if kind in ("rope", "write"):
        n, d, qd, kd = case["n"], case["dim"], case["heads"] * case["dim"], case["kv"] * case["dim"]
        moved = 2 * 4 * n * (qd + kd)
        if kind == "write":   # keys go to the cache only, values are read and written, both read again and returned
            moved = 4 * n * (2 * qd + 2 * kd) + 4 * n * _entry_bytes(case) + 2 * 4 * n * kd
        return {"bytes": moved + 4 * n + 8 * d + 2 * case["rot"], "flops": 8 * n * (qd + kd)}
    if kind == "read":
        return {"bytes": case["n"] * 2 * (_entry_bytes(case) + 4 * case["kv"] * case["dim"] + 2), "flops": 2 * case["n"] * case["kv"] * case["dim"]}
    q, mine, cuts, lens = _lengths(case)
    reach = lambda length, first: length if not case["window"] else min(length, max(0, length - first + case["window"] - 1))   # noqa: E731
    tokens = 0
    for i in range(case["seqs"]):   # own tokens that some query sees
        tokens += reach(mine[i], mine[i] - q[i] + 1 if case["window"] else 0)
    for j in range(case["prefixes"]):   # prefix tokens that some sequence of the group sees
        first = min(lens[j] + mine[i] - q[i] + 1 for i in range(cuts[j], cuts[j + 1]))
        tokens += lens[j] if not case["window"] else min(lens[j], max(0, lens[j] - first + case["window"]))
    return {"bytes": 2 * tokens * _entry_bytes(case) + 2 * 4 * sum(q) * case["heads"] * case["dim"],
            "flops": 4 * _pairs_seen(case) * case["heads"] * case["dim"]}


# ----------------------------------------------------------------------------------------------- cache
def _encode(kind, x):
    """x [..., dim] f32 -> (codes [..., row bytes] uint8, scales [..., dim / 32] f16 or None)."""
    if kind == "F16":
        return x.to(torch.float16).view(torch.uint8), None
    b = x.reshape(*x.shape[:-1], -1, BLOCK)
    if kind == "Q8_0":
        top = b.abs().amax(-1)
        d = top / torch.full_like(top, 127)   # tensor by tensor: a true division
        inv = torch.where(d > 0, 1 / d, torch.zeros_like(d))
        q = (b * inv[..., None]).round().clamp(-127, 127).to(torch.int8)
        return q.reshape(x.shape).view(torch.uint8), d.to(torch.float16)
    at = b.abs().argmax(-1, keepdim=True)
    d = b.gather(-1, at)[..., 0] / -8
    inv = torch.where(d != 0, 1 / d, torch.zeros_like(d))
    q = (b * inv[..., None] + 8.5).floor().clamp(0, 15).to(torch.uint8)
    return (q[..., :16] | (q[..., 16:] << 4)).reshape(*x.shape[:-1], -1), d.to(torch.float16)


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
    pages = case["pages"]
    cut = pages * kv * p * row
    codes = buf[:cut].view(pages, kv, p, row)
    return codes, None if case["type"] == "F16" else buf[cut:].view(torch.float16).view(pages, kv, p, case["dim"] // BLOCK)


def _put(buf, case, slots, x):
    codes, scales = _planes(buf, case)
    page, at = slots // case["page"], slots % case["page"]
    c, s = _encode(case["type"], x)
    codes[page, :, at] = c
    if s is not None:
        scales[page, :, at] = s


def _get(buf, case, slots):
    """[*slots, kv, dim] f32."""
    codes, scales = _planes(buf, case)
    page, at = slots // case["page"], slots % case["page"]
    return _decode(case["type"], codes[page, :, at], None if scales is None else scales[page, :, at])


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _i32(v):
    return torch.as_tensor(v, dtype=torch.int32).cuda()


def _new_cache(case, tokens, g):
    """An empty cache of a few more pages than `tokens` need, and the pages in a random order."""
    case["pages"] = -(-tokens // case["page"]) + 3
    size = case["pages"] * case["page"] * _entry_bytes(case)
    make = lambda: torch.zeros(size, dtype=torch.uint8, device="cuda")   # noqa: E731
    return make(), make(), torch.randperm(case["pages"], generator=g, device="cuda")


def _fill(buf, case, g, scale):
    """Entries in every slot, made as the path's own values are: normal heads with a few strong elements."""
    slots = torch.arange(case["pages"] * case["page"], device="cuda")
    for part in slots.split(1 << 15):
        x = torch.randn((part.numel(), case["kv"], case["dim"]), generator=g, device="cuda") * scale
        strong = torch.rand((case["kv"], case["dim"]), generator=g, device="cuda") < 0.02
        _put(buf, case, part, torch.where(strong, 3 * x, x))


# --------------------------------------------------------------------------------------------- prepare
def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    case = dict(case)
    s = {"case": case}
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda")   # noqa: E731
    empty = lambda *shape: torch.empty(shape, dtype=torch.float32, device="cuda")   # noqa: E731
    if kind in ("rope", "write"):
        n, h, kv, d = (case[v] for v in ("n", "heads", "kv", "dim"))
        s["qkv"] = randn(n, (h + 2 * kv) * d) * torch.exp(0.5 * randn(n, 1))   # the projection's rows, q | k | v
        s["wq"], s["wk"] = (1 + 0.1 * randn(d), 1 + 0.1 * randn(d)) if case["norm"] else (None, None)
        base = 500000.0
        s["freq"] = torch.tensor([base ** (-2 * i / case["rot"]) for i in range(case["rot"] // 2)], dtype=torch.float32, device="cuda")
        if n > 64:   # a prompt: positions in a row, from somewhere
            first = int(torch.randint(0, 131072 - n, (1,), generator=g, device="cuda"))
            s["pos"] = torch.arange(first, first + n, dtype=torch.int32, device="cuda")
        else:
            s["pos"] = torch.randint(0, 131072, (n,), generator=g, device="cuda", dtype=torch.int32)
        s["q_out"], s["k_out"] = empty(n, h * d), empty(n, kv * d)
        if kind == "write":
            s["v_out"] = empty(n, kv * d)
            s["k"], s["v"], order = _new_cache(case, n, g)
            at = torch.arange(n, device="cuda") + 5   # the sequence goes on inside a page
            s["slots"] = (order[at // case["page"]] * case["page"] + at % case["page"]).to(torch.int32)
    elif kind == "read":
        n, kv, d = case["n"], case["kv"], case["dim"]
        s["k"], s["v"], order = _new_cache(case, n, g)
        _fill(s["k"], case, g, 1.0)
        _fill(s["v"], case, g, 1.0)
        at = torch.arange(n, device="cuda")
        s["slots"] = (order[at // case["page"]] * case["page"] + at % case["page"]).to(torch.int32)
        s["k_out"], s["v_out"] = empty(n, kv * d), empty(n, kv * d)
    elif kind == "attn":
        q, mine, cuts, lens = _lengths(case)
        p, h, d = case["page"], case["heads"], case["dim"]
        need = [-(-v // p) for v in mine + lens]
        s["k"], s["v"], order = _new_cache(case, sum(need) * p, g)
        _fill(s["k"], case, g, 1.0)
        _fill(s["v"], case, g, 1.0)
        order = order.tolist()

        def table(counts):
            t = torch.zeros((max(1, len(counts)), max(counts, default=0) + 1), dtype=torch.int32)
            for i, c in enumerate(counts):
                t[i, :c] = torch.tensor([order.pop() for _ in range(c)], dtype=torch.int32)
            return t.cuda()

        s["seq_pages"], s["prefix_pages"] = table(need[:len(mine)]), table(need[len(mine):])
        s["q_offsets"] = _i32([0] + list(np.cumsum(q)))
        s["seq_lens"], s["prefix_lens"], s["prefix_seqs"] = _i32(mine), _i32(lens or [0]), _i32(cuts or [0])
        s["tokens"], s["max_q"], s["max_seq"], s["max_prefix"] = sum(q), max(q), max(mine), max(lens, default=0)
        s["q"] = randn(sum(q), h * d) * 1.5
        s["scale"] = 1 / math.sqrt(d)
        s["sinks"] = randn(h) if case["sinks"] else None
        s["out"] = empty(sum(q), h * d)
    else:
        rows, v = case["rows"], case["vocab"]
        s["logits"] = randn(rows, v) * case["spread"]
        peak = torch.randint(0, v, (rows, 8), generator=g, device="cuda")   # a few tokens that the model favours
        s["logits"].scatter_add_(1, peak, 4 * case["spread"] * torch.rand((rows, 8), generator=g, device="cuda"))
        s["logits"] = s["logits"].bfloat16().float() if seed % 2 else s["logits"]   # of a 16-bit head: many ties
        r = torch.rand((4, rows), generator=g, device="cuda")
        f = case["filters"]
        pick = torch.randint(0, 4, (rows,), generator=g, device="cuda")
        on = lambda name, k: torch.full((rows,), f in (name, "all"), device="cuda") | ((f == "mixed") & (pick == k))   # noqa: E731
        s["temperature"] = 0.5 + r[0]
        if f == "mixed":
            s["temperature"] = torch.where(r[0] < 0.1, torch.zeros_like(r[0]), s["temperature"])   # some are greedy
        k = torch.randint(1, 100, (rows,), generator=g, device="cuda")
        s["top_k"] = torch.where(on("top_k", 1), k, torch.zeros_like(k)).to(torch.int32)
        s["top_p"] = torch.where(on("top_p", 2), 0.5 + 0.49 * r[1], torch.ones_like(r[1]))
        s["min_p"] = torch.where(on("min_p", 3), 0.02 + 0.1 * r[2], torch.zeros_like(r[2]))
        s["u"] = r[3].clamp(max=1 - 2.0 ** -24)
        s["token"], s["logprob"] = torch.empty(rows, dtype=torch.int32, device="cuda"), empty(rows)
    torch.cuda.synchronize()   # the inputs were made on torch's own stream
    return s


# ---------------------------------------------------------------------------------------- plain forms
def _rotate(x, cos, sin, rot, pairs):
    a, rest = x[..., :rot], x[..., rot:]
    if pairs == "halves":
        lo, hi = a[..., : rot // 2], a[..., rot // 2:]
        a = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
    else:
        lo, hi = a[..., 0::2], a[..., 1::2]
        a = torch.stack([lo * cos - hi * sin, hi * cos + lo * sin], -1).flatten(-2)
    return torch.cat([a, rest], -1)


EPS = 1e-6


def _plain_heads(s, x, w, wide):
    """Norm and rotation of heads x [n, heads, dim], f32; in 64 bits where they are rounded to codes afterwards."""
    case = s["case"]
    angle = s["pos"].double()[:, None] * s["freq"].double()
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    if wide:
        x = x.double()
    else:
        cos, sin = cos.float(), sin.float()
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
    return _rotate(x, cos, sin, case["rot"], case["pairs"]).float()


def _plain_attn(s):
    case = s["case"]
    kv, d, grp = case["kv"], case["dim"], case["heads"] // case["kv"]
    n, dev = s["tokens"], "cuda"
    off, lens, page = s["q_offsets"].long(), s["seq_lens"].long(), case["page"]
    tok = torch.arange(n, device=dev)
    seq = torch.searchsorted(off[1:].contiguous(), tok, right=True)
    row = tok - off[seq]                                         # the token's place among its sequence's queries
    base = torch.zeros_like(lens)                                # length of each sequence's prefix
    q = s["q"].view(n, kv, grp, d) * s["scale"]

    def keys(buf, pages, cap):
        at = torch.arange(cap, device=dev)
        return _get(buf, case, pages.long()[:, at // page] * page + at % page).transpose(1, 2)   # [set, kv, cap, dim]

    def fold(x, which, place, sets, width):                      # tokens -> [set, kv, width * grp, .]
        t = torch.zeros((sets, width) + x.shape[1:], device=dev)
        t[which, place] = x
        return t.transpose(1, 2).reshape(sets, kv, width * grp, -1)

    def unfold(x, which, place, width):
        return x.reshape(x.shape[0], kv, width, grp, -1).transpose(1, 2)[which, place]

    parts = []
    if case["prefixes"]:
        cuts = s["prefix_seqs"].long()
        of = torch.searchsorted(cuts[1:].contiguous(), torch.arange(len(lens), device=dev), right=True)
        base = s["prefix_lens"].long()[of]
        grp_of, first = of[seq], off[cuts[:-1]]
        place = tok - first[grp_of]
        parts.append((s["prefix_pages"], s["max_prefix"], grp_of, place, case["prefixes"], _widest(case)))
    parts.append((s["seq_pages"], s["max_seq"], seq, row, case["seqs"], s["max_q"]))
    at = base[seq] + lens[seq] - (off[1:] - off[:-1])[seq] + row   # position of each query
    scores, folded = [], []
    for i, (pages, cap, which, place, sets, width) in enumerate(parts):
        k = keys(s["k"], pages, cap)
        x = unfold(fold(q, which, place, sets, width) @ k.transpose(2, 3), which, place, width)   # [token, kv, grp, cap]
        pos = torch.arange(cap, device=dev)[None] + (base[seq][:, None] if i == len(parts) - 1 else 0)
        held = s["prefix_lens"].long()[which] if i < len(parts) - 1 else base[seq] + lens[seq]
        ok = (pos < held[:, None]) & (pos <= at[:, None])
        if case["window"]:
            ok &= pos > at[:, None] - case["window"]
        scores.append(x.masked_fill_(~ok[:, None, None], -math.inf))
        folded.append((pages, cap, which, place, sets, width))
    top = scores[0].amax(-1)
    for x in scores[1:]:
        top = torch.maximum(top, x.amax(-1))
    if s["sinks"] is not None:
        top = torch.maximum(top, s["sinks"].view(kv, grp))
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    total = torch.exp(s["sinks"].view(kv, grp) - top) if s["sinks"] is not None else torch.zeros_like(top)
    out = 0
    for x, (pages, cap, which, place, sets, width) in zip(scores, folded):
        x = x.sub_(top[..., None]).exp_()
        total = total + x.sum(-1)
        out = out + unfold(fold(x, which, place, sets, width) @ keys(s["v"], pages, cap), which, place, width)
    return torch.where(total[..., None] > 0, out / total[..., None], torch.zeros_like(out)).reshape(n, -1)


def _widest(case):
    """Query tokens of the prefix group that has most."""
    q, _, cuts, _ = _lengths(case)
    return max(sum(q[cuts[j]:cuts[j + 1]]) for j in range(case["prefixes"]))


def _plain_sample(s):
    x = s["logits"].double()
    n = x.shape[1]
    t = s["temperature"].double()[:, None]
    val, idx = x.sort(dim=-1, descending=True, stable=True)   # equal ones keep the order of their indices
    top = val[:, :1]
    rank = torch.arange(n, device=x.device)[None]
    k = s["top_k"].long()[:, None]
    w = torch.exp((val - top) / torch.where(t > 0, t, torch.ones_like(t)))
    w = torch.where((k <= 0) | (rank < k), w, torch.zeros_like(w))
    run_ = w.cumsum(-1)
    before = torch.cat([torch.zeros_like(top), run_[:, :-1]], -1)
    p = s["top_p"].double()[:, None]
    keep = (w > 0) & ((p >= 1) | (rank == 0) | (before < p * run_[:, -1:])) & (w >= s["min_p"].double()[:, None])
    keep &= (t > 0) | (rank == 0)
    w = torch.zeros_like(w).scatter_(1, idx, torch.where(keep, w, torch.zeros_like(w)))   # back in the vocabulary's order
    run_ = w.cumsum(-1)
    hit = (run_ > s["u"].double()[:, None] * run_[:, -1:]) & (w > 0)
    last = n - 1 - (w > 0).flip(-1).int().argmax(-1)
    token = torch.where(hit.any(-1), hit.int().argmax(-1), last)
    prob = x.gather(1, token[:, None]) - top - torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    return {"token": token.to(torch.int32), "logprob": prob[:, 0].float()}


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
        from qxotic_amd.jam import JAM, AttnBatch, KvCache, QkSpec, Sampling
        case, h = s["case"], {}
        ptr = lambda t: None if t is None else t.data_ptr()   # noqa: E731
        if "type" in case:
            h["cache"] = KvCache(type=getattr(JAM, case["type"]), kv_heads=case["kv"], head_dim=case["dim"], page_tokens=case["page"],
                                 n_pages=case["pages"], k=ptr(s["k"]), v=ptr(s["v"]))
        if "freq" in s:
            h["spec"] = QkSpec(q_heads=case["heads"], kv_heads=case["kv"], head_dim=case["dim"], rope_dim=case["rot"],
                               neighbours=int(case["pairs"] == "neighbours"), eps=EPS, scale=1.0, q_weight=ptr(s["wq"]), k_weight=ptr(s["wk"]),
                               inv_freq=ptr(s["freq"]))
        if case["kind"] == "attn":
            h["batch"] = AttnBatch(n_tokens=s["tokens"], n_seqs=case["seqs"], n_prefixes=case["prefixes"], max_q=s["max_q"],
                                   max_seq_len=s["max_seq"], max_prefix_len=s["max_prefix"], q_offsets=ptr(s["q_offsets"]),
                                   seq_lens=ptr(s["seq_lens"]), seq_pages=ptr(s["seq_pages"]), ld_seq_pages=s["seq_pages"].shape[1],
                                   prefix_seqs=ptr(s["prefix_seqs"]), prefix_lens=ptr(s["prefix_lens"]), prefix_pages=ptr(s["prefix_pages"]),
                                   ld_prefix_pages=s["prefix_pages"].shape[1])
        if case["kind"] == "sample":
            h["params"] = Sampling(temperature=ptr(s["temperature"]), top_k=ptr(s["top_k"]), top_p=ptr(s["top_p"]), min_p=ptr(s["min_p"]),
                                   u=ptr(s["u"]))
        s["handles"] = h
    return s["handles"]


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        jam, h = _jam(), _handles(s)
        if kind == "sample":
            _ok(jam.sample(s["logits"].data_ptr(), case["vocab"], case["rows"], case["vocab"], h["params"], s["token"].data_ptr(),
                           s["logprob"].data_ptr()))
            return {"token": s["token"], "logprob": s["logprob"]}
        if kind == "attn":
            ld = case["heads"] * case["dim"]
            _ok(jam.attn_shared_prefix(h["cache"], h["batch"], s["q"].data_ptr(), ld, case["heads"], s["scale"], s["out"].data_ptr(), ld,
                                       window=case["window"], sinks_dev=None if s["sinks"] is None else s["sinks"].data_ptr()))
            return s["out"]
        n, kd = case["n"], case["kv"] * case["dim"]
        if kind == "read":
            _ok(jam.kv_read(h["cache"], s["slots"].data_ptr(), n, s["k_out"].data_ptr(), kd, s["v_out"].data_ptr(), kd))
            return {"k": s["k_out"], "v": s["v_out"]}
        qd = case["heads"] * case["dim"]
        ld, q = qd + 2 * kd, s["qkv"].data_ptr()
        k, v = q + 4 * qd, q + 4 * (qd + kd)
        if kind == "rope":
            _ok(jam.qk_norm_rope(h["spec"], q, ld, s["q_out"].data_ptr(), qd, k, ld, s["k_out"].data_ptr(), kd, s["pos"].data_ptr(), n))
            return {"q": s["q_out"], "k": s["k_out"]}
        _ok(jam.qkv_norm_rope_write(h["spec"], h["cache"], q, ld, s["q_out"].data_ptr(), qd, k, ld, v, ld, s["pos"].data_ptr(),
                                    s["slots"].data_ptr(), n))
        _ok(jam.kv_read(h["cache"], s["slots"].data_ptr(), n, s["k_out"].data_ptr(), kd, s["v_out"].data_ptr(), kd))
        return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}
    if kind == "sample":
        return _plain_sample(s)
    if kind == "attn":
        return _plain_attn(s)
    n, kv, d = case["n"], case["kv"], case["dim"]
    if kind == "read":
        slots = s["slots"].long()
        return {"k": _get(s["k"], case, slots).reshape(n, -1), "v": _get(s["v"], case, slots).reshape(n, -1)}
    q, k, v = s["qkv"].view(n, -1, d).split([case["heads"], kv, kv], 1)
    q, k = _plain_heads(s, q, s["wq"], False), _plain_heads(s, k, s["wk"], kind == "write")
    if kind == "rope":
        return {"q": q.reshape(n, -1), "k": k.reshape(n, -1)}
    slots = s["slots"].long()
    _put(s["k"], case, slots, k)
    _put(s["v"], case, slots, v)
    return {"q": q.reshape(n, -1), "k": _get(s["k"], case, slots).reshape(n, -1), "v": _get(s["v"], case, slots).reshape(n, -1)}


# --------------------------------------------------------------------------------------------- exact
def _exact_values(kind, x):
    """What the cache holds for the f32 values x [.., dim] once written, in 64 bits."""
    if kind == "F16":
        return x.to(torch.float16).double()
    b = x.view(*x.shape[:-1], x.shape[-1] // BLOCK, BLOCK)
    if kind == "Q8_0":
        d = torch.div(b.abs().max(-1).values, torch.tensor(127.0, device=x.device).expand(b.shape[:-1]))
        code = torch.round(b * torch.where(d == 0, d, d.reciprocal())[..., None])
    else:
        big = b.abs().max(-1, keepdim=True).values
        first = (b.abs() == big).int().argmax(-1, keepdim=True)
        d = torch.take_along_dim(b, first, -1)[..., 0] * -0.125
        code = torch.floor(b * torch.where(d == 0, d, d.reciprocal())[..., None] + 8.5).clamp(max=15) - 8
    return (code.double() * d.half().double()[..., None]).half().double().reshape(x.shape)


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


def _exact_heads(s, x, w):
    case, half = s["case"], s["case"]["rot"] // 2
    x = x.double().clone()
    if w is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + EPS) * w.double()
    at = torch.arange(half, device=x.device)
    i, j = (at, at + half) if case["pairs"] == "halves" else (2 * at, 2 * at + 1)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), s["pos"].double()[:, None] * s["freq"].double()[None])[:, None]
    z = torch.complex(x[..., i], x[..., j]) * turn
    x[..., i], x[..., j] = z.real, z.imag
    return x


def exact(case, seed):
    s = prepare(case, seed)
    case = s["case"]
    kind = case["kind"]
    if kind == "sample":
        x, out = s["logits"].cpu().numpy().astype(np.float64), []
        par = {k: s[k].cpu().numpy().astype(np.float64) for k in ("temperature", "top_k", "top_p", "min_p", "u")}
        prob = np.empty(len(x))
        for r, row in enumerate(x):
            t, k = par["temperature"][r], int(par["top_k"][r])
            order = np.lexsort((np.arange(row.size), -row))
            if t == 0:
                pick = order[0]
            else:
                if k > 0:
                    order = order[:k]
                w = np.exp((row[order] - row[order[0]]) / t)
                if par["top_p"][r] < 1:
                    ahead = np.concatenate([[0.0], np.cumsum(w)])[:-1]
                    cut = max(1, int((ahead < par["top_p"][r] * w.sum()).sum()))
                    order, w = order[:cut], w[:cut]
                some = w >= par["min_p"][r]
                order, w = order[some], w[some]
                by = np.argsort(order)
                order, run_ = order[by], np.cumsum(w[by])
                pick = order[min(np.searchsorted(run_, par["u"][r] * run_[-1], side="right"), order.size - 1)]
            out.append(pick)
            prob[r] = row[pick] - row.max() - math.log(math.fsum(np.exp(row - row.max())))
        return {"token": torch.tensor(np.array(out), dtype=torch.int32), "logprob": torch.from_numpy(prob)}
    if kind == "read":
        return {name: _exact_entries(s[name], case, s["slots"].long()).reshape(case["n"], -1) for name in ("k", "v")}
    if kind in ("rope", "write"):
        n, h, kv, d = (case[v] for v in ("n", "heads", "kv", "dim"))
        x = s["qkv"].view(n, h + 2 * kv, d)
        q, k = _exact_heads(s, x[:, :h], s["wq"]), _exact_heads(s, x[:, h:h + kv], s["wk"])
        if kind == "rope":
            return {"q": q.reshape(n, -1), "k": k.reshape(n, -1)}
        return {"q": q.reshape(n, -1), "k": _exact_values(case["type"], k.float()).reshape(n, -1),
                "v": _exact_values(case["type"], x[:, h + kv:].contiguous()).reshape(n, -1)}
    # attention, one sequence and key head at a time
    q, mine, cuts, lens = _lengths(case)
    kv, d, grp, page = case["kv"], case["dim"], case["heads"] // case["kv"], case["page"]
    out = torch.zeros((sum(q), kv, grp, d), dtype=torch.float64, device="cuda")
    rows = s["q"].double().view(sum(q), kv, grp, d)
    at = 0

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
        where = torch.arange(length, device="cuda")
        mine_at = length - q[i] + torch.arange(q[i], device="cuda")
        ok = where[None] <= mine_at[:, None]
        if case["window"]:
            ok &= mine_at[:, None] - where[None] < case["window"]
        for c in range(kv):
            x = (rows[at:at + q[i], c].reshape(-1, d) @ k[:, c].T).view(q[i], grp, length) * s["scale"]
            x = torch.where(ok[:, None], x, torch.full_like(x, -math.inf))
            if s["sinks"] is not None:
                sink = s["sinks"].double().view(kv, grp)[c].view(1, grp, 1).expand(q[i], grp, 1)
                w = torch.softmax(torch.cat([x, sink], -1), -1)[..., :-1]
            else:
                w = torch.softmax(x, -1)
            out[at:at + q[i], c] = (w.reshape(-1, length) @ v[:, c]).view(q[i], grp, d)
        at += q[i]
    return out.reshape(sum(q), -1)
