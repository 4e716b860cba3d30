"""The operators around attention and sampling from their definitions, in 64 bits (numpy): head norm and rotation, the cache's
codes, attention of a ragged batch, the next token of a row of logits."""
from __future__ import annotations

import numpy as np

F16, Q4_0, Q8_0 = 1, 2, 8


def norm_rope(x, weight, pos, freq, rot, neighbours, eps, scale=1.0):
    """x [n, heads, dim] -> f64."""
    x = x.astype(np.float64).copy()
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * weight.astype(np.float64)
    if rot:
        angle = pos.astype(np.float64)[:, None] * freq.astype(np.float64)[None]
        z = np.float64(np.float32(scale)) * np.exp(1j * angle)[:, None]
        p = np.arange(rot // 2)
        a, b = (2 * p, 2 * p + 1) if neighbours else (p, p + rot // 2)
        w = (x[..., a] + 1j * x[..., b]) * z
        x[..., a], x[..., b] = w.real, w.imag
    return x


def entry(kind, x):
    """What the cache holds for f32 rows x [..., dim]: f64 values, by the types' definitions in f32."""
    x = np.ascontiguousarray(x, np.float32)
    if kind == F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16).astype(np.float64)
    b = x.reshape(*x.shape[:-1], -1, 32)
    one = np.float32(1)
    with np.errstate(divide="ignore", over="ignore", invalid="ignore"):
        if kind == Q8_0:
            d = np.abs(b).max(-1, keepdims=True) / np.float32(127)
            code = np.clip(np.rint(b * np.where(d > 0, one / d, np.float32(0))), -127, 127)
        else:
            at = np.abs(b).argmax(-1)[..., None]
            d = np.take_along_axis(b, at, -1) * np.float32(-0.125)
            code = np.clip(np.floor(b * np.where(d != 0, one / d, np.float32(0)) + np.float32(8.5)), 0, 15) - 8
        v = (code.astype(np.float64) * d.astype(np.float16).astype(np.float64)).astype(np.float16)
    return v.astype(np.float64).reshape(x.shape)


def pack(kind, x, kv, page, pages, slots):
    """A cache buffer of `pages` pages with the rows x [n, kv, dim] at `slots`, byte by byte, zeros elsewhere."""
    n, _, dim = x.shape
    row = {F16: 2 * dim, Q8_0: dim, Q4_0: dim // 2}[kind]
    codes = np.zeros((pages, kv, page, row), np.uint8)
    scales = np.zeros((pages, kv, page, dim // 32 if kind != F16 else 0), np.float16)
    x = np.ascontiguousarray(x, np.float32)
    for i, s in enumerate(slots):
        p, t = divmod(int(s), page)
        if kind == F16:
            codes[p, :, t] = x[i].astype(np.float16).view(np.uint8).reshape(kv, row)
            continue
        b = x[i].reshape(kv, -1, 32)
        if kind == Q8_0:
            d = np.abs(b).max(-1, keepdims=True) / np.float32(127)
            inv = np.where(d > 0, np.float32(1) / np.where(d > 0, d, 1), np.float32(0)).astype(np.float32)
            codes[p, :, t] = np.rint(b * inv).astype(np.int8).view(np.uint8).reshape(kv, row)
        else:
            d = np.take_along_axis(b, np.abs(b).argmax(-1)[..., None], -1) * np.float32(-0.125)
            inv = np.where(d != 0, np.float32(1) / np.where(d != 0, d, 1), np.float32(0)).astype(np.float32)
            q = np.clip(np.floor(b * inv + np.float32(8.5)), 0, 15).astype(np.uint8)
            codes[p, :, t] = (q[..., :16] | (q[..., 16:] << 4)).reshape(kv, row)
        scales[p, :, t] = d[..., 0].astype(np.float16)
    return np.concatenate([codes.reshape(-1), scales.reshape(-1).view(np.uint8)])


def attention(q, k, v, pos, scale, window=0, sinks=None):
    """One sequence and key head: q [n, grp, dim], k, v [keys, dim], pos [n] positions among the keys, sinks [grp]. Masked entries
    are left out. Returns (out [n, grp, dim], the largest scale * sum |q k| of a visible key [n, grp], largest |v|)."""
    n, grp, dim = q.shape
    out, mass, big = np.zeros((n, grp, dim)), np.zeros((n, grp)), np.zeros((n, grp))
    q, k, v = (a.astype(np.float64) for a in (q, k, v))
    for i in range(n):
        lo, hi = (max(0, pos[i] - window + 1) if window else 0), min(len(k), pos[i] + 1)
        if hi <= lo:
            continue
        kk, vv = k[lo:hi], v[lo:hi]
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


def sample(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.0):
    """(token, logprob, margin): margin is how far u is from the ends of the token's share of the kept weights."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return 0, -np.inf, 1.0
    with np.errstate(invalid="ignore"):
        d = np.where(x == top, 0.0, x - top)
    logz = np.log(np.exp(d).sum())
    order = np.lexsort((np.arange(x.size), -x))
    if not temperature > 0:
        return int(order[0]), d[order[0]] - logz, 1.0
    if top_k > 0:
        order = order[:top_k]
    w = np.exp(d / temperature)[order]
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        keep = before < top_p * w.sum()
        keep[0] = True
        order, w = order[keep], w[keep]
    keep = w >= min(min_p, 1.0)
    order, w = order[keep], w[keep]
    by = np.argsort(order)
    order, w = order[by], w[by]
    run = np.cumsum(w)
    hit = np.nonzero((run > u * run[-1]) & (w > 0))[0]
    i = hit[0] if hit.size else np.nonzero(w > 0)[0][-1]
    share = run / run[-1]
    margin = min(abs(share[i] - u) if i + 1 < len(share) else 1.0, abs(u - share[i - 1]) if i else 1.0)
    return int(order[i]), d[order[i]] - logz, margin
