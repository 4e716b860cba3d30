"""GPU: attention calls of more workgroups than one launch takes, and of more than there can be."""
import sys

import numpy as np
import pytest
from test_gpu_attn import CASES, Batch

from oracle import decode as D

pytestmark = pytest.mark.gpu


def test_more_workgroups_than_a_launch_takes(hip):
    """17000 sequences of one query token under a max_q of 16384: 17.4 million workgroups of 256 threads, nearly all without rows."""
    import torch
    from qxotic_amd.jam import JAM, AttnBatch, KvCache
    print("attn workgroups", file=sys.stderr, flush=True)
    kv, dim, page, pages, n = 8, 64, 16, 9, 17000
    r = np.random.default_rng(0)
    x = r.standard_normal((2, pages * page, kv, dim)).astype(np.float32)
    vals = [D.entry(D.F16, a) for a in x]
    table = r.integers(0, pages, (n, 3)).astype(np.int32)   # sequences share pages
    lens = r.integers(1, 48, n).astype(np.int32)
    q = r.standard_normal((n, kv * dim)).astype(np.float32)
    dev = [torch.from_numpy(a).cuda() for a in (*(D.pack(D.F16, a, kv, page, pages, range(pages * page)) for a in x),
                                                np.arange(n + 1, dtype=np.int32), lens, table, q)]
    out = torch.full((n, kv * dim), -5.0, device="cuda")
    torch.cuda.synchronize()
    p = [t.data_ptr() for t in dev]
    c = KvCache(type=JAM.F16, kv_heads=kv, head_dim=dim, page_tokens=page, n_pages=pages, k=p[0], v=p[1])
    b = AttnBatch(n_tokens=n, n_seqs=n, max_q=16384, max_seq_len=48, q_offsets=p[2], seq_lens=p[3], seq_pages=p[4], ld_seq_pages=3)
    assert hip.attn_shared_prefix(c, b, p[5], kv * dim, kv, dim ** -0.5, out.data_ptr(), kv * dim) == 0, hip.last_error()
    hip.synchronize()
    got = out.cpu().numpy().reshape(n, kv, dim)
    assert (got != -5.0).all()
    for i in [*range(0, n, 13), *range(n - 40, n)]:
        at = np.arange(lens[i])
        slots = table[i][at // page].astype(np.int64) * page + at % page
        for h in range(kv):
            want, mass, big = D.attention(q[i].reshape(1, kv, dim)[:, h:h + 1], vals[0][slots, h], vals[1][slots, h], [lens[i] - 1],
                                          np.float64(np.float32(dim ** -0.5)))
            assert (np.abs(got[i, h] - want[0, 0]) <= (big * (2.0 ** -18 * mass + 2.0 ** -19))[0, 0]).all(), (i, h)   # as in test_gpu_attn.py


@pytest.mark.parametrize("name,max_q", [("few_tokens", 5), ("few_tokens_window", 7), ("prompt", 60), ("prompt_64", 100), ("many_sequences_prompts", 2),
                                        ("grouped_tokens", 3), ("grouped_tokens", 1), ("many_groups", 2), ("page_7", 20)])
def test_query_tokens_past_max_q(hip, name, max_q):
    """They are not computed; those before them see the keys up to their own place, not a later one's."""
    kv, grp, dim, page, groups, alone, window, sinks = CASES[name]
    print("attn past max_q", name, max_q, file=sys.stderr, flush=True)
    b = Batch(D.Q8_0, kv, grp, dim, page, groups, alone, window, sinks, seed=max_q)
    assert max(q for _, q in b.seqs) > max_q
    got = b.run(hip, max_q=max_q)
    for i, (_, nq) in enumerate(b.seqs):
        rows = got[b.off[i]:b.off[i + 1]]
        assert (rows[max_q:] == -5.0).all()
        for c in range(kv if nq else 0):
            want, tol = b.want(i, c)
            g = rows[:max_q, c * grp * dim:(c + 1) * grp * dim].reshape(want[:max_q].shape)
            assert (np.abs(g - want[:max_q]) <= tol[:max_q]).all(), (i, c)


def test_more_workgroups_than_there_can_be(hip):
    """Refused before any work: the pointers here lead nowhere."""
    from qxotic_amd.jam import JAM, AttnBatch, KvCache
    P = 1 << 20
    c = KvCache(type=JAM.Q8_0, kv_heads=2, head_dim=64, page_tokens=16, n_pages=4, k=P, v=P)
    for seqs in (1 << 10, 1 << 20):
        b = AttnBatch(n_tokens=1 << 28, n_seqs=seqs, max_q=1 << 28, max_seq_len=33, q_offsets=P, seq_lens=P, seq_pages=P, ld_seq_pages=3)
        assert hip.attn_shared_prefix(c, b, P, 256, 4, 0.125, P, 256) == JAM.EUNSUPPORTED and "attn" in hip.last_error()
