"""GPU: sampling against its definition in 64 bits (oracle/decode.py): the token exactly, its log probability to 2^-22 of 1 + |it|
(one rounding to f32 of a 64-bit value). Random numbers that fall within 1e-9 of the border between two tokens are not used: sums
in another order may round there (each is within 2^-45 of the largest weight)."""
import sys

import numpy as np
import pytest

from oracle import decode as D

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, file=sys.stderr, flush=True)


def run(hip, x, temperature=None, top_k=None, top_p=None, min_p=None, u=None, pad=0, logprob=True):
    import torch
    from qxotic_amd.jam import Sampling
    rows, vocab = x.shape
    xd = torch.from_numpy(np.concatenate([x, np.full((rows, pad), 1e30, np.float32)], 1)).cuda()
    dev = [None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (temperature, top_k, top_p, min_p, u)]
    token = torch.full((rows + 1,), -7, dtype=torch.int32, device="cuda")
    lp = torch.full((rows + 1,), -7.0, device="cuda")
    p = Sampling(*(None if a is None else a.data_ptr() for a in dev))
    torch.cuda.synchronize()
    for _ in range(2):   # the second call finds the first one's workspace
        st = hip.sample(xd.data_ptr(), vocab + pad, rows, vocab, p, token.data_ptr(), lp.data_ptr() if logprob else None)
        assert st == 0, hip.last_error()
    hip.synchronize()
    t, l = token.cpu().numpy(), lp.cpu().numpy()
    assert t[-1] == -7 and l[-1] == -7.0
    return t[:-1], l[:-1]


def check(hip, x, **kw):
    rows = x.shape[0]
    get = lambda k, r, d: d if kw.get(k) is None else kw[k][r]   # noqa: E731
    want = [D.sample(x[r], get("temperature", r, 1.0), int(get("top_k", r, 0)), np.float64(get("top_p", r, 1.0)),
                     np.float64(get("min_p", r, 0.0)), np.float64(kw["u"][r])) for r in range(rows)]
    token, lp = run(hip, x, **kw)
    for r in range(rows):
        t, l, margin = want[r]
        if margin > 1e-9:
            assert token[r] == t, (r, int(token[r]), t, {k: get(k, r, None) for k in ("temperature", "top_k", "top_p", "min_p", "u")})
            assert lp[r] == l or abs(lp[r] - l) <= 2.0 ** -22 * (1 + abs(l)), (r, lp[r], l)


def params(rows, seed, which):
    r = np.random.default_rng(seed)
    on = lambda k: np.full(rows, which in (k, "all")) | ((which == "mixed") & (r.integers(0, 2, rows) == 1))   # noqa: E731
    t = r.uniform(0.3, 1.6, rows).astype(np.float32)
    if which == "mixed":
        t[r.random(rows) < 0.15] = 0
    return dict(temperature=t, top_k=np.where(on("top_k"), r.integers(1, 200, rows), 0).astype(np.int32),
                top_p=np.where(on("top_p"), r.uniform(0.05, 0.999, rows), 1).astype(np.float32),
                min_p=np.where(on("min_p"), r.uniform(0.001, 0.3, rows), 0).astype(np.float32), u=(r.random(rows) * (1 - 2.0 ** -24)).astype(np.float32))


@pytest.mark.parametrize("which", ["none", "top_k", "top_p", "min_p", "all", "mixed"])
@pytest.mark.parametrize("rows,vocab,spread,half", [(1, 1, 1.0, 0), (3, 2, 1.0, 0), (5, 63, 2.0, 0), (4, 64, 3.0, 1), (7, 1000, 2.5, 1),
                                                    (2, 4097, 1.0, 0), (3, 32001, 2.5, 1), (33, 5003, 4.0, 0), (2, 128256, 1.0, 0),
                                                    (2, 262144, 2.5, 1)])
def test_sample(hip, which, rows, vocab, spread, half):
    """half: logits of a 16-bit head, many of them equal."""
    say("sample", which, rows, vocab, spread, half)
    r = np.random.default_rng(vocab + rows)
    x = (r.standard_normal((rows, vocab)) * spread).astype(np.float32)
    x[np.arange(rows), r.integers(0, vocab, rows)] += np.float32(3 * spread)
    if half:
        x = (x.view(np.uint32) & 0xFFFF0000).view(np.float32)
    check(hip, x, pad=vocab % 3, **params(rows, vocab, which))


@pytest.mark.parametrize("name", ["equal", "two values", "tiny range", "wide", "masked", "one left", "infinite", "nan", "zeros", "falling",
                                  "denormal"])
@pytest.mark.parametrize("vocab", [40, 9001])
def test_sample_values(hip, name, vocab):
    """Rows where a threshold falls among equal values, where almost all is masked, or where values are extreme."""
    say("sample values", name, vocab)
    r = np.random.default_rng(vocab)
    rows = 24
    x = r.standard_normal((rows, vocab)).astype(np.float32)
    if name == "equal":
        x[:] = 1.25
    elif name == "two values":
        x = np.where(r.random(x.shape) < 0.3, 2.0, 1.0).astype(np.float32)
    elif name == "tiny range":
        x = (x * 1e-6).astype(np.float32)
    elif name == "wide":
        x = (x * 3e4).astype(np.float32)
    elif name == "masked":
        x[r.random(x.shape) < 0.9] = np.finfo(np.float32).min
        x[:, 7] = 0.5
    elif name == "one left":
        x[:] = -np.inf
        x[np.arange(rows), r.integers(0, vocab, rows)] = -3.0
    elif name == "infinite":
        x[r.random(x.shape) < 0.3] = -np.inf
        x[::2, vocab // 2] = np.inf
        x[::4, vocab // 3] = np.inf
    elif name == "nan":
        x[r.random(x.shape) < 0.2] = np.nan
        x[:, 11] = 2.0
    elif name == "zeros":
        x = np.where(r.random(x.shape) < 0.5, 0.0, -0.0).astype(np.float32)
    elif name == "falling":
        x = np.sort(x, 1)[:, ::-1].copy()
    elif name == "denormal":
        x = (x * 1e-42).astype(np.float32)
    check(hip, x, **params(rows, 5, "all"))
    check(hip, x, **params(rows, 6, "mixed"))
    check(hip, x, u=np.linspace(0, 1 - 2.0 ** -24, rows).astype(np.float32))


def test_sample_edges(hip):
    """The first and last token at the ends of u; top-k at and above the vocabulary; min-p of 1; top-p of 0; no arrays but u; rows
    of nothing; no log probability."""
    r = np.random.default_rng(1)
    x = r.standard_normal((6, 777)).astype(np.float32)
    u = np.array([0, 0, 0.5, 0.5, 1 - 2.0 ** -24, 1 - 2.0 ** -24], np.float32)
    check(hip, x, u=u)
    check(hip, x, top_k=np.array([777, 776, 778, 1, 1, 2], np.int32), u=u)
    check(hip, x, top_p=np.zeros(6, np.float32), u=u)
    check(hip, x, min_p=np.ones(6, np.float32), u=u)
    check(hip, x, temperature=np.array([0, -1, np.nan, 1e-3, 100, 1], np.float32), u=u)
    x[2] = -np.inf
    x[4] = np.nan
    token, lp = run(hip, x, u=u)
    assert token[2] == 0 and token[4] == 0 and not (lp[2] > -np.inf) and not (lp[4] > -np.inf)
    token, lp = run(hip, x, u=u, logprob=False)
    assert (lp == -7.0).all()


def test_sample_largest_k(hip):
    """top-k so large that its threshold lies deep in the row, top-p after it."""
    r = np.random.default_rng(2)
    x = (r.standard_normal((4, 50021)) * 2).astype(np.float32)
    u = r.random(4).astype(np.float32)
    for k in (3000, 20011, 50020):
        check(hip, x, top_k=np.full(4, k, np.int32), u=u)
        check(hip, x, top_k=np.full(4, k, np.int32), top_p=np.array([0.3, 0.9, 0.999, 0.5], np.float32), u=u)
        check(hip, (x.view(np.uint32) & 0xFFFF0000).view(np.float32), top_k=np.full(4, k, np.int32),
              top_p=np.array([0.3, 0.9, 0.999, 0.5], np.float32), u=u)


@pytest.mark.parametrize("vocab", [301, 20000, 128256])
def test_sample_k_of_several_waves(hip, vocab):
    """top-k alone, of 65 to 256: the kept ones are put into the vocabulary's order by several waves in one pass."""
    say("sample k of several waves", vocab)
    r = np.random.default_rng(vocab)
    k = np.concatenate([[64, 65, 66, 127, 128, 129, 191, 192, 193, 255, 256, 257], r.integers(65, 257, 52)]).astype(np.int32)
    x = r.standard_normal((k.size, vocab)).astype(np.float32)
    check(hip, x, temperature=np.full(k.size, 3.0, np.float32), top_k=k, u=(r.random(k.size) * (1 - 2.0 ** -24)).astype(np.float32))


def test_sample_many_rows_and_long_ones(hip):
    """More rows than a pair of launches takes; rows of more slices than a wave has lanes."""
    r = np.random.default_rng(3)
    x = (r.standard_normal((300, 133)) * 2).astype(np.float32)
    check(hip, x, **params(300, 8, "mixed"))
    x = (r.standard_normal((3, 300007)) * 2).astype(np.float32)
    for which in ("none", "all", "top_p"):
        check(hip, x, **params(3, 9, which))


def test_refusals(hip):
    from qxotic_amd.jam import JAM, Sampling
    P, ok = 1 << 20, Sampling(u=1 << 20)
    assert hip.sample(None, 8, 1, 8, ok, P) == JAM.EINVAL and hip.sample(P, 8, 1, 8, ok, None) == JAM.EINVAL
    assert hip.sample(P, 8, 1, 8, None, P) == JAM.EINVAL and hip.sample(P, 8, 1, 8, Sampling(), P) == JAM.EINVAL
    assert hip.sample(P, 7, 1, 8, ok, P) == JAM.EINVAL and hip.sample(P, 8, -1, 8, ok, P) == JAM.EINVAL
    assert hip.sample(P, 8, 1, 0, ok, P) == JAM.EINVAL and hip.sample(P, 8, 0, 8, ok, P) == JAM.OK
    assert "sample" in hip.last_error()
