"""GPU: head norm and rotation, the cache's codes as they are written, and the cache read back, against their definitions in 64
bits (oracle/decode.py).

What is returned as f32 is computed in f32 from 64-bit angles: the norm's sum of up to 512 squares, a root, a division and four
products, below 16 roundings of 2^-24 (the sum's grow with the depth of its tree, log2 of the lanes plus the 8 elements of one);
the tolerance is 2^-20 of the head's largest element times its weight. What the cache gives back is compared bit by bit."""
import sys

import numpy as np
import pytest

from oracle import decode as D

pytestmark = pytest.mark.gpu
NAMES = {D.F16: "F16", D.Q8_0: "Q8_0", D.Q4_0: "Q4_0"}


def say(*a):
    print(*a, file=sys.stderr, flush=True)


def ptr(t, off=0):
    return None if t is None else t.data_ptr() + 4 * off


def make(n, heads, kv, dim, rot, norm, seed, pad=0):
    """A token's row is q | k | v and `pad` floats more; positions far and near, one of them 0."""
    import torch
    r = np.random.default_rng(seed)
    x = (r.standard_normal((n, (heads + 2 * kv) * dim + pad)) * np.exp(r.standard_normal((n, 1)))).astype(np.float32)
    w = [(1 + 0.1 * r.standard_normal(dim)).astype(np.float32) for _ in range(2)] if norm else [None, None]
    freq = (10000.0 ** (-2 * np.arange(rot // 2) / max(rot, 1))).astype(np.float32)
    pos = r.integers(0, 1 << 20, n).astype(np.int32)
    pos[0] = 0
    dev = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()   # noqa: E731
    return x, w, freq, pos, dev(x), [dev(a) for a in w], dev(freq), dev(pos)


def spec(heads, kv, dim, rot, nbr, w, freq, scale=1.0):
    from qxotic_amd.jam import QkSpec
    return QkSpec(q_heads=heads, kv_heads=kv, head_dim=dim, rope_dim=rot, neighbours=nbr, eps=1e-6, scale=scale, q_weight=ptr(w[0]),
                  k_weight=ptr(w[1]), inv_freq=ptr(freq) if rot else None)


def near(got, want):
    tol = 2.0 ** -20 * np.abs(want).max(-1, keepdims=True)
    bad = np.abs(got - want) > tol
    assert not bad.any(), (int(bad.sum()), float((np.abs(got - want) / tol).max()))


ROPE = [   # (n, heads, kv, dim, rot, neighbours, norm, pad)
    (1, 32, 8, 128, 128, 0, True, 0), (1, 1, 1, 64, 64, 0, False, 0), (3, 7, 1, 96, 96, 0, True, 0), (5, 6, 2, 96, 48, 1, True, 0),
    (2, 4, 2, 256, 64, 1, True, 4), (9, 5, 5, 80, 40, 0, True, 0), (4, 3, 1, 34, 18, 0, True, 1), (4, 3, 1, 34, 34, 1, True, 3),
    (2, 2, 1, 512, 512, 0, True, 0), (3, 2, 2, 6, 2, 0, True, 0), (7, 4, 4, 64, 0, 0, True, 2), (600, 9, 3, 64, 32, 0, False, 0),
    (530, 20, 4, 128, 64, 1, True, 0), (3, 2, 0, 128, 128, 0, True, 0), (3, 0, 2, 128, 128, 0, True, 0),
]


@pytest.mark.parametrize("n,heads,kv,dim,rot,nbr,norm,pad", ROPE)
def test_norm_rope(hip, n, heads, kv, dim, rot, nbr, norm, pad):
    import torch
    say("rope", n, heads, kv, dim, rot, nbr, norm, pad)
    x, w, freq, pos, xd, wd, fd, pd = make(n, heads, kv, dim, rot, norm, 7 * n + dim, pad)
    ld, lq, lk = x.shape[1], heads * dim + pad, kv * dim + pad
    q = torch.full((n, max(lq, 1)), -5.0, device="cuda")
    k = torch.full((n, max(lk, 1)), -5.0, device="cuda")
    torch.cuda.synchronize()
    st = hip.qk_norm_rope(spec(heads, kv, dim, rot, nbr, wd, fd, 0.75), xd.data_ptr(), ld, q.data_ptr(), lq, ptr(xd, heads * dim), ld,
                          k.data_ptr(), lk, pd.data_ptr(), n)
    assert st == 0, hip.last_error()
    hip.synchronize()
    for out, first, h, weight in ((q, 0, heads, w[0]), (k, heads * dim, kv, w[1])):
        if h:
            got = out.cpu().numpy()
            want = D.norm_rope(x[:, first:first + h * dim].reshape(n, h, dim), weight, pos, freq, rot, nbr, 1e-6, 0.75)
            near(got[:, :h * dim].reshape(n, h, dim), want)
            assert (got[:, h * dim:] == -5.0).all()
    # in place, the same bits
    st = hip.qk_norm_rope(spec(heads, kv, dim, rot, nbr, wd, fd, 0.75), xd.data_ptr(), ld, xd.data_ptr(), ld, ptr(xd, heads * dim), ld,
                          ptr(xd, heads * dim), ld, pd.data_ptr(), n)
    assert st == 0
    hip.synchronize()
    assert torch.equal(xd[:, :heads * dim], q[:, :heads * dim])
    assert torch.equal(xd[:, heads * dim:(heads + kv) * dim], k[:, :kv * dim])
    assert np.array_equal(xd.cpu().numpy()[:, (heads + kv) * dim:], x[:, (heads + kv) * dim:])


WRITE = [   # (n, heads, kv, dim, rot, neighbours, norm, page, pad)
    (1, 32, 8, 128, 128, 0, True, 16, 0), (5, 4, 2, 64, 32, 0, True, 16, 0), (40, 7, 1, 96, 96, 0, False, 32, 0),
    (33, 6, 3, 96, 48, 1, True, 5, 0), (700, 4, 4, 128, 64, 1, True, 64, 0), (9, 2, 2, 256, 256, 0, True, 1, 1),
    (6, 3, 3, 32, 0, 0, False, 7, 3), (17, 0, 2, 128, 128, 0, True, 128, 0),
]


@pytest.mark.parametrize("kind", [D.F16, D.Q8_0, D.Q4_0])
@pytest.mark.parametrize("n,heads,kv,dim,rot,nbr,norm,page,pad", WRITE)
def test_write_and_read(hip, kind, n, heads, kv, dim, rot, nbr, norm, page, pad):
    """The buffers byte by byte, the queries, and the read back with slots outside the cache. A block of zeros, one of equal
    magnitudes and both signs, and one of tiny values are among the values."""
    import torch
    from qxotic_amd.jam import KvCache
    say("write", NAMES[kind], n, heads, kv, dim, rot, nbr, norm, page, pad)
    x, w, freq, pos, _, wd, fd, pd = make(n, heads, kv, dim, rot, norm, 3 * n + dim + kind, pad)
    v0 = (heads + kv) * dim
    x[0, v0:v0 + 32] = 0
    x[n - 1, v0:v0 + 32] = np.where(np.arange(32) % 3 == 1, -2.5, 2.5)
    x[n // 2, v0 + dim - 32:v0 + dim] *= 1e-6
    xd = torch.from_numpy(x).cuda()
    ld = x.shape[1]
    pages = -(-n // page) + 2
    slots = np.random.default_rng(n).permutation(pages * page)[:n].astype(np.int32)
    skip = slots.copy()
    if n > 4:
        skip[2], skip[3] = -1, pages * page   # padding tokens: not written
    sd = torch.from_numpy(skip).cuda()
    c = KvCache(type=kind, kv_heads=kv, head_dim=dim, page_tokens=page, n_pages=pages)
    size = hip.kv_cache_bytes(c)
    guard = 256
    bufs = [torch.zeros(size + guard, dtype=torch.uint8, device="cuda") for _ in range(2)]
    c.k, c.v = bufs[0].data_ptr(), bufs[1].data_ptr()
    q = torch.full((n, max(1, heads * dim)), -5.0, device="cuda")
    torch.cuda.synchronize()
    st = hip.qkv_norm_rope_write(spec(heads, kv, dim, rot, nbr, wd, fd), c, xd.data_ptr(), ld, q.data_ptr(), heads * dim,
                                 ptr(xd, heads * dim), ld, ptr(xd, v0), ld, pd.data_ptr(), sd.data_ptr(), n)
    assert st == 0, hip.last_error()
    hip.synchronize()
    if heads:
        near(q.cpu().numpy().reshape(n, heads, dim), D.norm_rope(x[:, :heads * dim].reshape(n, heads, dim), w[0], pos, freq, rot, nbr, 1e-6))
    keys = D.norm_rope(x[:, heads * dim:v0].reshape(n, kv, dim), w[1], pos, freq, rot, nbr, 1e-6).astype(np.float32)
    vals = x[:, v0:v0 + kv * dim].reshape(n, kv, dim)
    live = (skip >= 0) & (skip < pages * page)
    for buf, rows in zip(bufs, (keys, vals)):
        got = buf.cpu().numpy()
        assert np.array_equal(got[:size], D.pack(kind, rows[live], kv, page, pages, skip[live]))
        assert (got[size:] == 0).all()
    want = [np.where(live[:, None, None], D.entry(kind, r), 0).reshape(n, -1).astype(np.float32) for r in (keys, vals)]
    for odd in (0, 1):   # rows at 16-byte and at 4-byte alignment
        lk = kv * dim + odd
        outs = [torch.full((n, lk), -5.0, device="cuda") for _ in range(2)]
        torch.cuda.synchronize()
        assert hip.kv_read(c, sd.data_ptr(), n, outs[0].data_ptr(), lk, outs[1].data_ptr(), lk) == 0, hip.last_error()
        hip.synchronize()
        for o, want_ in zip(outs, want):
            got = o.cpu().numpy()
            assert np.array_equal(got[:, :kv * dim], want_)
            assert (got[:, kv * dim:] == -5.0).all()
    one = torch.full((n, kv * dim), -5.0, device="cuda")
    torch.cuda.synchronize()
    assert hip.kv_read(c, sd.data_ptr(), n, None, 0, one.data_ptr(), kv * dim) == 0
    hip.synchronize()
    assert np.array_equal(one.cpu().numpy(), want[1])


def test_refusals(hip):
    """What is refused is refused before any work: the pointers here lead nowhere."""
    from qxotic_amd.jam import JAM, KvCache, QkSpec
    good = dict(type=JAM.Q8_0, kv_heads=2, head_dim=64, page_tokens=16, n_pages=4, k=1 << 20, v=1 << 20)
    s = QkSpec(q_heads=4, kv_heads=2, head_dim=64, rope_dim=64, eps=1e-6, scale=1.0, inv_freq=1 << 20)
    P = 1 << 20

    def write(c, s=s, ldq=256, ldv=128, pos=P, slots=P, n=1):
        return hip.qkv_norm_rope_write(s, c, P, ldq, P, 256, P, 128, P, ldv, pos, slots, n)

    E, U = JAM.EINVAL, JAM.EUNSUPPORTED
    c = KvCache(**good)
    assert hip.kv_cache_bytes(c) == 4 * 16 * 2 * (64 + 4)
    assert write(None) == E and write(c, None) == E
    assert write(KvCache(**{**good, "k": None})) == E and write(KvCache(**{**good, "v": P + 8})) == E
    assert write(KvCache(**{**good, "page_tokens": 0})) == E and write(KvCache(**{**good, "kv_heads": 4})) == E
    assert write(KvCache(**{**good, "type": JAM.Q4_K})) == U and hip.kv_cache_bytes(KvCache(**{**good, "type": JAM.F32})) == -1
    assert write(KvCache(**{**good, "head_dim": 48}), QkSpec(q_heads=4, kv_heads=2, head_dim=48)) == U
    assert write(KvCache(**{**good, "n_pages": 1 << 30})) == U
    assert write(c, ldq=255) == E and write(c, ldv=127) == E and write(c, pos=None) == E and write(c, slots=None) == E
    assert write(c, n=-1) == E and write(c, n=0) == JAM.OK
    assert write(c, QkSpec(q_heads=4, kv_heads=2, head_dim=64, rope_dim=66)) == E
    assert write(c, QkSpec(q_heads=4, kv_heads=2, head_dim=64, rope_dim=64)) == E   # no inv_freq
    assert write(c, QkSpec(q_heads=4, kv_heads=2, head_dim=64, rope_dim=3)) == E
    assert hip.qk_norm_rope(QkSpec(q_heads=1, kv_heads=1, head_dim=1024), P, 1024, P, 1024, P, 1024, P, 1024, P, 1) == U
    assert hip.qk_norm_rope(s, None, 256, P, 256, P, 128, P, 128, P, 1) == E
    assert hip.qk_norm_rope(s, P, 256, P, 256, P, 128, P, 127, P, 1) == E
    assert hip.kv_read(c, P, 1, None, 0, None, 0) == E and hip.kv_read(c, None, 1, P, 128, None, 0) == E
    assert hip.kv_read(c, P, 1, P, 127, None, 0) == E and hip.kv_read(c, P, 0, P, 128, None, 0) == JAM.OK
    assert "kv_read" in hip.last_error()
