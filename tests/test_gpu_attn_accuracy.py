"""GPU: attention's accuracy where a row's elements differ by many powers of two, with the batches of test_gpu_attn.py."""
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
