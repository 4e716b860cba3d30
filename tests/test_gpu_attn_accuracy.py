"""GPU: attention's accuracy where a row's elements or weights differ by many powers of two, with the batches of test_gpu_attn.py."""
import numpy as np
import pytest
from test_gpu_attn import CASES, NAMES, Batch, say

from oracle import decode as D

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [D.F16, D.Q8_0, D.Q4_0])
@pytest.mark.parametrize("name", ["one_sequence", "few_tokens", "prompt", "prompt_64", "decode_256", "prompt_192", "grouped_32", "grouped_128"])
@pytest.mark.parametrize("ratio", [256, 4096, 65536])
def test_query_with_a_strong_channel(hip, kind, name, ratio):
    """One element of every query row is `ratio` times the others and meets keys that are 0 there: it adds nothing to a score, nor to S
    of the tolerance, and must not take bits from the others (at most 2^-38 of it each, ratio * 2^-38 <= 2^-22 of theirs)."""
    kv, grp, dim, page, groups, alone, window, sinks = CASES[name]
    say("attn strong channel", NAMES[kind], name, ratio)
    b = Batch(kind, kv, grp, dim, page, groups, alone, window, sinks, seed=ratio + kind)
    at = 37 % dim
    x = b.vals[0].astype(np.float32)
    x[:, :, at] = 0
    b.vals[0] = D.entry(kind, x)
    b.bufs[0] = D.pack(kind, x, kv, page, b.pages, range(b.pages * page))
    q = b.q.reshape(b.n, kv * grp, dim)
    q[:, :, at] = np.where(q[:, :, at] < 0, -1.5, 1.5) * ratio
    b.check(b.run(hip))


@pytest.mark.parametrize("nq,grp", [(1, 1), (8, 4), (130, 1)])
def test_weights_beside_a_strong_first_key(hip, nq, grp):
    """The first of 3000 keys has nearly all the weight and a value of 0; the others, 2^-6 to 2^-32 of it each, make the output. Queries
    and keys are exact: a score of up to 32 (powers of two) is off by the rounding of scale * log2 e and of the exponents, a weight
    by less than 2^-17.5 of it; the two halves by 2^-21; 3000 products joined to a growing sum at 2^-27 of it by 2^-16.4; the whole
    below 2^-15. A weight's end is at 2^-37 of the largest."""
    n, dim = 3000, 64
    say("attn strong first key", nq, grp)
    b = Batch(D.F16, 8, grp, dim, 16, [], [(n, nq)] * 64, seed=1)
    for s in range(1, 64):
        b.own[s] = b.own[0]   # one sequence's pages for all: as many workgroups as the chip holds, so that a row is walked in one run
    k, v = np.zeros((b.pages * 16, 8, dim), np.float32), np.ones((b.pages * 16, 8, dim), np.float32)
    first = b.slots(0)[0]
    k[first, :, 0], v[first] = 1, 0
    b.bufs = [np.ascontiguousarray(x.reshape(b.pages, 16, 8, dim).swapaxes(1, 2)).astype(np.float16).view(np.uint8).reshape(-1) for x in (k, v)]
    score = (4.25 + np.arange(b.n * 8 * grp) % 23 * 0.8125).reshape(b.n, 8 * grp).astype(np.float32)   # natural logarithms
    b.q[:] = 0
    b.q.reshape(b.n, 8 * grp, dim)[:, :, 0] = score * 8   # scale 1 / 8; 11 bits
    got = b.run(hip).reshape(64, nq, 8 * grp, dim)
    others = (n - nq + np.arange(nq))[None, :, None]
    mass = others * np.exp(-score.astype(np.float64)).reshape(64, nq, 8 * grp)
    want = mass / (mass + 1)
    tol = want * 2.0 ** -15 + n * 2.0 ** -37
    err = np.abs(got - want[..., None]).max(-1)
    say(f"   largest error {float((err / tol).max()):.3f} of the tolerance")
    assert bool((err <= tol).all())
