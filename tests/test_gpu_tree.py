"""GPU: masks, attention and acceptance of drafted trees against their definitions (oracle/tree.py). Masks, positions, paths and slots are
whole numbers and equal; the attention's tolerance is that of the linear batches (test_gpu_attn.py): the arithmetic of a visible key is the
same, and a masked one adds nothing."""
import sys

import numpy as np
import pytest

from oracle import decode as D
from oracle import tree as T
from test_gpu_attn import Batch

pytestmark = pytest.mark.gpu
NAMES = {D.F16: "F16", D.Q8_0: "Q8_0", D.Q4_0: "Q4_0"}
KINDS = [D.F16, D.Q8_0, D.Q4_0]


def say(*a):
    print(*a, file=sys.stderr, flush=True)


def draft(r, n, shape="wide"):
    """Parents of one tree."""
    if shape == "chain":
        return [i - 1 for i in range(n)]
    if shape == "flat":
        return [-1] + [0] * (n - 1) if n else []
    if shape == "bad":   # parents that are none
        return [int(r.integers(-3, n + 3)) for _ in range(n)]
    return [-1 if i == 0 else int(i * r.random() ** 2) for i in range(n)]


def i32(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(np.array(a, np.int32).reshape(-1))).cuda()


# ------------------------------------------------------------------------------------------------ masks
@pytest.mark.parametrize("shape", ["wide", "chain", "flat", "bad"])
@pytest.mark.parametrize("sizes,words", [([1], 1), ([8], 1), ([64], 1), ([5, 0, 64, 1, 33], 1), ([65, 3, 128, 0], 2), ([200, 7], 4), ([1000, 64, 130], 16),
                                         ([3] * 300, 1)])
def test_masks(hip, sizes, words, shape):
    import torch
    from qxotic_amd.jam import Tree
    say("masks", sizes[:5], words, shape)
    r = np.random.default_rng(sum(sizes) + words)
    trees = [draft(r, n, shape) for n in sizes]
    off, parents = np.cumsum([0] + sizes), [p for t in trees for p in t]
    n, extra = len(parents), 3
    first = r.integers(0, 100000, len(sizes))
    pos = np.concatenate([f + np.arange(k) for f, k in zip(first, sizes)] + [np.full(extra, -7)])
    d_off, d_par, d_pos = i32(off), i32(parents + [-1] * extra), i32(pos)
    for with_pos in (True, False):
        masks = torch.full((n + extra, words), -6, dtype=torch.int64, device="cuda")
        torch.cuda.synchronize()
        t = Tree(n_tokens=n + extra, n_seqs=len(sizes), max_q=max(sizes), q_offsets=d_off.data_ptr(), parents=d_par.data_ptr())
        assert hip.tree_masks(t, masks.data_ptr(), words, d_pos.data_ptr() if with_pos else None) == 0, hip.last_error()
        hip.synchronize()
        sets = [s for t in trees for s in T.ancestors(t)]
        got = masks.cpu().numpy().view(np.uint64)
        assert np.array_equal(got[:n], T.words(sets, words)) and (masks.cpu().numpy()[n:] == -6).all()
        want = [int(first[i]) + len(s) - 1 for i, t in enumerate(trees) for s in T.ancestors(t)] + [-7] * extra
        assert d_pos.cpu().tolist() == want


def test_masks_of_many_tokens(hip):
    """A sequence's tokens past max_q are left alone; offsets that are out of range stay inside the arrays."""
    import torch
    from qxotic_amd.jam import Tree
    parents, pos = i32([-1, 0, 1, 2, 3, -1, 0]), i32([50, 51, 52, 53, 54, 9, 10])
    masks = torch.full((7, 1), -6, dtype=torch.int64, device="cuda")
    off = i32([0, 5, 7])
    torch.cuda.synchronize()
    t = Tree(n_tokens=7, n_seqs=2, max_q=3, q_offsets=off.data_ptr(), parents=parents.data_ptr())
    assert hip.tree_masks(t, masks.data_ptr(), 1, pos.data_ptr()) == 0
    hip.synchronize()
    assert masks.flatten().cpu().tolist() == [1, 3, 7, -6, -6, 1, 3] and pos.cpu().tolist() == [50, 51, 52, 53, 54, 9, 10]
    for bad in ([-4, 900, 2], [6, 2, 100], [1 << 30, -(1 << 30), 5]):
        off = i32(bad)
        guard = torch.full((9, 1), -6, dtype=torch.int64, device="cuda")
        torch.cuda.synchronize()
        t = Tree(n_tokens=7, n_seqs=2, max_q=64, q_offsets=off.data_ptr(), parents=parents.data_ptr())
        assert hip.tree_masks(t, guard.data_ptr(), 1, None) == 0
        hip.synchronize()
        assert (guard[7:] == -6).all()


# --------------------------------------------------------------------------------------------- acceptance
def accept(hip, trees, tokens, picked, longest, max_q=None, extra=2, move=True, lens=None):
    import torch
    from qxotic_amd.jam import Tree, TreePath
    n, off = len(trees), np.cumsum([0] + [len(t) for t in trees])
    total = int(off[-1]) + extra
    r = np.random.default_rng(total)
    slots = r.permutation(3 * total + 1)[:total].astype(np.int32)
    flat = lambda a: [v for t in a for v in t] + [0] * extra   # noqa: E731
    d = dict(off=i32(off), parents=i32(flat(trees)), tokens=i32(flat(tokens)), picked=i32(flat(picked)), slots=i32(slots),
             lens=i32(r.integers(0, 1000, n)), path=i32([-9] * (n * longest + 1)), accepted=i32([-9] * (n + 1)), next=i32([-9] * (n + 1)),
             move_from=i32([-9] * total), move_to=i32([-9] * total))
    before = d["lens"].cpu().numpy()
    torch.cuda.synchronize()
    t = Tree(n_tokens=total, n_seqs=n, max_q=max_q or max(max(len(t) for t in trees), 1), q_offsets=d["off"].data_ptr(), parents=d["parents"].data_ptr())
    p = TreePath(ld_path=longest, path=d["path"].data_ptr(), accepted=d["accepted"].data_ptr(), next=d["next"].data_ptr())
    if move:   # lens in place
        p.lens = p.lens_out = d["lens"].data_ptr()
        p.slots, p.move_from, p.move_to = (d[k].data_ptr() for k in ("slots", "move_from", "move_to"))
    assert hip.tree_accept(t, d["tokens"].data_ptr(), d["picked"].data_ptr(), p) == 0, hip.last_error()
    hip.synchronize()
    got = {k: v.cpu().numpy() for k, v in d.items()}
    assert got["path"][-1] == got["accepted"][-1] == got["next"][-1] == -9
    src, dst = np.full(total, -9), np.full(total, -9)
    for i in range(n):
        cut = len(trees[i]) if max_q is None else max_q
        path, after = T.walk(trees[i][:cut], tokens[i][:cut], picked[i][:cut], longest)
        assert got["path"][i * longest:(i + 1) * longest].tolist() == path + [-1] * (longest - len(path)), i
        assert got["accepted"][i] == len(path) and got["next"][i] == after, i
        a, b = off[i], off[i + 1]
        src[a:b] = dst[a:b] = -1
        for k, c in enumerate(path):
            if c != k:
                src[a + k], dst[a + k] = slots[a + c], slots[a + k]
        if move:
            assert got["lens"][i] == before[i] + len(path)
    if move:
        assert np.array_equal(got["move_from"], src) and np.array_equal(got["move_to"], dst)
    else:
        assert (got["move_from"] == -9).all()
    return got


def agree(r, trees, vocab=5, share=0.7):
    tokens = [r.integers(0, vocab, len(t)).tolist() for t in trees]
    picked = [r.integers(0, vocab, len(t)).tolist() for t in trees]
    for t, w, p in zip(trees, tokens, picked):
        for i in range(1, len(t)):
            if 0 <= t[i] < i and r.random() < share:
                p[t[i]] = w[i]
    return tokens, picked


@pytest.mark.parametrize("shape", ["wide", "chain", "flat", "bad"])
@pytest.mark.parametrize("sizes,longest", [([1], 1), ([25], 25), ([64, 0, 7, 1], 64), ([65, 130], 8), ([300, 2, 1100], 1100), ([9] * 200, 9), ([40], 3)])
def test_accept(hip, sizes, longest, shape):
    say("accept", sizes[:4], longest, shape)
    r = np.random.default_rng(sum(sizes))
    trees = [draft(r, n, shape) for n in sizes]
    tokens, picked = agree(r, trees)
    accept(hip, trees, tokens, picked, longest)
    accept(hip, trees, tokens, picked, longest, move=False)


def test_accept_edges(hip):
    """The lowest of equal children; every token accepted; tokens past max_q; a path of no length; large token ids."""
    got = accept(hip, [[-1, 0, 0, 0, 2, 1]], [[7, 4, 4, 4, 5, 6]], [[4, 6, 5, 1, 2, 9]], 6)
    assert got["path"][:6].tolist() == [0, 1, 5, -1, -1, -1] and got["next"][0] == 9
    n = 150
    accept(hip, [draft(None, n, "chain")], [list(range(n))], [list(range(1, n + 1))], n)
    accept(hip, [draft(None, n, "chain")], [list(range(n))], [list(range(1, n + 1))], n, max_q=70)
    accept(hip, [[-1, 0]], [[1, (1 << 31) - 1]], [[(1 << 31) - 1, -(1 << 31)]], 2)
    got = accept(hip, [[-1, 0], []], [[1, 2], []], [[2, 3], []], 0)
    assert got["accepted"][:2].tolist() == [0, 0] and got["next"][:2].tolist() == [-1, -1]


# ---------------------------------------------------------------------------------------------- attention
class Trees(Batch):
    """A Batch whose query tokens are trees: `bits[t]`, the set of a token's drafted ones."""

    def __init__(self, *a, words=None, shape="wide", **kw):
        super().__init__(*a, **kw)
        r = np.random.default_rng(self.n + 1)
        most = max([q for _, q in self.seqs], default=1)
        self.words = words or -(-max(most, 1) // 64)
        self.bits = []
        for _, n in self.seqs:
            if shape == "any":   # bits of earlier and later tokens alike, and past the tokens
                self.bits += [{j for j in range(64 * self.words) if r.random() < 0.4} for _ in range(n)]
            elif shape == "none":
                self.bits += [set() for _ in range(n)]
            else:
                self.bits += T.ancestors(draft(r, n, shape))

    def run(self, hip, times=1, max_q=None, extra=0):
        from qxotic_amd.jam import HipJAM

        class Linear:   # the call of the base class, as a call of attn_tree
            last_error, synchronize = hip.last_error, hip.synchronize

            @staticmethod
            def attn_shared_prefix(c, b, q, ldq, heads, scale, out, ldo, **kw):
                return HipJAM.attn_tree(hip, c, b, self.masks.data_ptr(), self.words, q, ldq, heads, scale, out, ldo, **kw)

        rows = T.words(self.bits, self.words)
        rows = np.concatenate([rows, np.full((extra, self.words), ~np.uint64(0))])
        self.masks = self.torch.from_numpy(rows.view(np.int64)).cuda()
        return super().run(Linear, times, max_q, extra)

    def want(self, i, kv):
        own, nq = self.seqs[i]
        at = self.slots(i)
        first = own - nq
        base = len(at) - own
        keys = []
        for t in range(nq):
            # drafted token j is the sequence's own first + j; those in front of the own ones have no entry
            have = {first + j for j in self.bits[self.off[i] + t] if 0 <= j < nq and first + j >= 0}
            k = list(range(base + max(first, 0))) + [base + p for p in sorted(have)]
            keys.append(k[-self.window:] if self.window else k)
        w = self.grp * self.dim
        q = self.q[self.off[i]:self.off[i + 1], kv * w:(kv + 1) * w].reshape(nq, self.grp, self.dim)
        sinks = None if self.sinks is None else self.sinks[kv * self.grp:(kv + 1) * self.grp].astype(np.float64)
        out, mass, big = T.attention(q, self.vals[0][at, kv], self.vals[1][at, kv], keys, np.float64(np.float32(self.scale)), sinks)
        return out, (big * (2.0 ** -18 * mass + 2.0 ** -19))[..., None]


# name: (kv, grp, dim, page, groups, alone, window, sinks)
CASES = {
    "one_token": (1, 1, 64, 16, [], [(1, 1)], 0, False),
    "one_tree": (2, 4, 128, 16, [], [(245, 25)], 0, False),
    "tree_alone": (1, 4, 64, 16, [], [(13, 13)], 0, True),
    "trees_16": (2, 4, 128, 16, [], [(100, 16), (16, 16), (17, 16), (301, 15)], 0, False),
    "trees_32": (2, 4, 64, 16, [], [(500, 32), (129, 30), (33, 32)], 0, False),
    "trees_64": (1, 4, 128, 16, [], [(1500, 64), (64, 64), (128, 64), (191, 63)], 0, True),
    "trees_130": (1, 2, 64, 16, [], [(1500, 130), (130, 130), (131, 1), (191, 65)], 0, False),
    "trees_300": (1, 1, 96, 64, [], [(700, 300), (300, 257)], 0, False),
    "small_trees": (1, 1, 128, 16, [], [(40 + 17 * i, 1 + i % 8) for i in range(12)], 0, False),
    "small_trees_8": (2, 8, 64, 16, [], [(40 + 17 * i, 1 + i % 5) for i in range(9)], 0, True),
    "shared": (2, 4, 64, 16, [(300, [(20 + 7 * i, 9) for i in range(5)])], [(77, 12)], 0, False),
    "shared_grouped": (8, 1, 64, 16, [(7000, [(20 + 3 * i, 12) for i in range(20)])], [(77, 12)], 0, False),
    "shared_grouped_2": (8, 2, 128, 16, [(5000, [(20 + 3 * i, 4) for i in range(20)]), (4700, [(9, 4), (4, 4), (30, 3)] * 5)], [], 0, True),
    "shared_many": (8, 2, 64, 16, [(1950 - j % 5, [(3 + (i + j) % 20, 1 + i % 3) for i in range(8)]) for j in range(67)], [(7, 1)], 0, False),
    "grouped_window": (8, 2, 64, 16, [(1500, [(4 + 60 * i, 4) for i in range(36)])], [], 1000, True),
    "grouped_window_short": (8, 2, 64, 16, [(1500, [(4 + i, 4) for i in range(36)])], [], 3, True),
    "window": (1, 4, 64, 16, [(90, [(40, 20), (20, 20)])], [(200, 30), (30, 30)], 50, False),
    "window_short": (1, 4, 128, 16, [], [(200, 30), (30, 30), (400, 33)], 4, True),
    "window_1": (1, 2, 64, 16, [(33, [(40, 20)])], [(70, 70)], 1, False),
    "dim_96": (2, 7, 96, 32, [(131, [(33, 5), (95, 20)])], [], 0, True),
    "dim_192": (1, 4, 192, 16, [], [(333, 13), (40, 40)], 0, False),
    "dim_256": (1, 2, 256, 16, [(70, [(90, 33)])], [(33, 33), (300, 7)], 0, False),
    "dim_256_wide": (1, 4, 256, 16, [], [(333, 70)], 0, False),
    "empty": (1, 4, 64, 16, [(40, [(0, 0), (20, 3), (0, 0)]), (0, [(3, 2)])], [(0, 0), (0, 1), (5, 0)], 0, False),
    "empty_sinks": (1, 4, 64, 16, [], [(0, 1), (0, 2), (9, 2)], 0, True),
    "more_queries_than_keys": (1, 2, 64, 16, [(10, [(2, 5), (0, 3)])], [(2, 6), (60, 70)], 0, False),
    "more_queries_window": (1, 2, 64, 16, [(10, [(2, 5), (0, 3)])], [(2, 6), (60, 70)], 3, False),
    "many": (1, 4, 64, 16, [(200, [(8 + i % 37, 1 + i % 8) for i in range(70)])], [(9, 1)], 0, False),
    "page_1": (1, 2, 64, 1, [(33, [(20, 7)])], [(70, 12)], 0, False),
    "page_7": (1, 2, 64, 7, [], [(100, 60), (13, 6)], 0, False),
}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("name", CASES)
def test_attn_tree(hip, kind, name):
    kv, grp, dim, page, groups, alone, window, sinks = CASES[name]
    say("attn_tree", NAMES[kind], name)
    b = Trees(kind, kv, grp, dim, page, groups, alone, window, sinks, seed=len(name) + kind)
    got = b.run(hip)
    b.check(got)
    assert np.array_equal(b.run(hip, times=2), got)   # the same bits again


@pytest.mark.parametrize("shape", ["chain", "any", "none"])
@pytest.mark.parametrize("name", ["one_tree", "tree_alone", "trees_64", "trees_130", "small_trees", "shared_grouped", "grouped_window", "window",
                                  "window_short", "dim_256", "more_queries_than_keys", "more_queries_window", "page_7"])
def test_attn_any_bits(hip, name, shape):
    """Chains (as linear batches), bits of any tokens, later ones and past the sequence's tokens included, no bits at all."""
    kv, grp, dim, page, groups, alone, window, sinks = CASES[name]
    say("attn_tree bits", name, shape)
    b = Trees(D.Q8_0, kv, grp, dim, page, groups, alone, window, sinks, seed=3, shape=shape)
    got = b.run(hip)
    b.check(got)
    # the linear batch, by its own call too; a linear query token in front of the own ones counts back into the prefix, a tree's does not
    if shape == "chain" and "more_queries" not in name:
        b.check(Batch.run(b, hip))


def test_attn_more_words_than_needed(hip):
    kv, grp, dim, page, groups, alone, window, sinks = CASES["trees_16"]
    b = Trees(D.F16, kv, grp, dim, page, groups, alone, window, sinks, seed=3, words=3)
    b.check(b.run(hip))


@pytest.mark.parametrize("name", ["one_tree", "trees_64", "shared", "window_short"])
def test_attn_strides_and_growing_scores(hip, name):
    kv, grp, dim, page, groups, alone, window, sinks = CASES[name]
    for scale in (1.0, 8.0):
        b = Trees(D.Q8_0, kv, grp, dim, page, groups, alone, window, sinks, seed=3, pad=8, loud=True)
        b.q *= np.float32(scale)
        b.check(b.run(hip))
    b = Trees(D.F16, kv, grp, dim, page, groups, alone, window, sinks, seed=4, pad=3)   # rows at 4-byte alignment
    b.check(b.run(hip))


@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("name", ["one_tree", "trees_16", "trees_64", "trees_130", "shared", "shared_grouped", "window", "dim_256", "small_trees"])
def test_attn_masked_entries_change_nothing(hip, name, value):
    """Every entry that no query sees holds NaN or Inf, and so does the last drafted token of each sequence, which only those with its bit
    see: the others' rows are not touched by it."""
    kv, grp, dim, page, groups, alone, window, sinks = CASES[name]
    say("attn_tree masked", name, value)
    b = Trees(D.F16, kv, grp, dim, page, groups, alone, window, sinks, seed=9)
    seen = np.zeros(b.pages * page, bool)
    for i in range(len(b.seqs)):
        seen[b.slots(i)] = True
    for buf in b.bufs:
        h = buf.view(np.float16).reshape(b.pages, kv, page, dim)
        for s in np.nonzero(~seen)[0]:
            h[s // page, :, s % page] = value
        for i, (_, nq) in enumerate(b.seqs):
            if nq > 1:
                s = b.slots(i)[-1]
                h[s // page, :, s % page] = value
    got = b.run(hip)
    for i, (_, nq) in enumerate(b.seqs):
        ok = np.array([nq == 1 or nq - 1 not in b.bits[b.off[i] + t] for t in range(nq)], bool)
        assert nq <= 1 or ok.any()
        for c in range(kv):
            want, tol = b.want(i, c)
            g = got[b.off[i]:b.off[i + 1], c * grp * dim:(c + 1) * grp * dim].reshape(want.shape)
            assert (np.abs(g - want)[ok] <= np.broadcast_to(tol, want.shape)[ok]).all(), (i, c)


def test_attn_device_lengths_past_the_maxima(hip):
    """Pages out of range, tokens of no sequence, tokens past max_q: rows of others keep their results, those rows are not written."""
    b = Trees(D.Q8_0, 1, 4, 64, 16, [(40, [(20, 5), (30, 6), (17, 7)])], [(25, 8), (12, 9)], seed=2)
    b.own[1, 0] = 1 << 30
    b.own[1, 1] = -9
    got = b.run(hip, extra=3)
    b.check(got, skip=(1,))
    assert np.isfinite(got).all() and (got[b.n:] == -5.0).all()
    b = Trees(D.Q8_0, 1, 4, 64, 16, [], [(20, 5), (25, 2)], seed=2)
    got = b.run(hip, max_q=3)
    want, tol = b.want(0, 0)
    assert (np.abs(got[:3].reshape(3, 4, 64) - want[:3]) <= tol[:3]).all() and (got[3:5] == -5.0).all()
    b.check(got, skip=(0,))


@pytest.mark.parametrize("name", ["one_tree", "trees_64", "shared_grouped"])
def test_attn_in_a_graph_and_on_another_stream(hip, name):
    """Captured once, replayed with other queries and masks and after larger eager calls of the same context."""
    import torch
    from qxotic_amd.jam import HipJAM
    kv, grp, dim, page, groups, alone, window, sinks = CASES[name]
    jam = HipJAM()
    try:
        b = Trees(D.Q8_0, kv, grp, dim, page, groups, alone, window, sinks, seed=5)
        eager = b.run(jam)
        stream = torch.cuda.Stream()
        assert jam.set_stream(stream.cuda_stream) == 0
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            assert b.call() == 0
        big = Trees(D.Q8_0, kv, grp, dim, page, [(400, [(200, 3)] * 6)], [], seed=6)
        for k in range(3):
            big.run(jam)
            scaled = (b.q * np.float32(1 + k)).astype(np.float32)
            b.dev["q"].copy_(torch.from_numpy(scaled))
            if k == 2:
                b.bits = [s ^ {0} for s in b.bits]
                b.masks.copy_(torch.from_numpy(T.words(b.bits, b.words).view(np.int64)))
            b.out.fill_(-5.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = b.out.cpu().numpy()
            if k == 0:
                assert np.array_equal(got, eager)
            keep, b.q = b.q, scaled
            b.check(got)
            b.q = keep
    finally:
        jam.close()


def test_refusals(hip):
    """Through the entry points, before any work: the pointers here lead nowhere."""
    from qxotic_amd.jam import JAM, AttnBatch, KvCache, Tree, TreePath
    P, E, U = 1 << 20, JAM.EINVAL, JAM.EUNSUPPORTED
    cache = dict(type=JAM.Q8_0, kv_heads=2, head_dim=64, page_tokens=16, n_pages=4, k=P, v=P)
    batch = dict(n_tokens=2, n_seqs=2, n_prefixes=1, max_q=1, max_seq_len=33, max_prefix_len=17, q_offsets=P, seq_lens=P, seq_pages=P,
                 ld_seq_pages=3, prefix_seqs=P, prefix_lens=P, prefix_pages=P, ld_prefix_pages=2)

    def call(c=None, b=None, masks=P, words=1, q=P, ldq=256, heads=4, scale=0.125, out=P, ldo=256, window=0, no=None):
        return hip.attn_tree(None if no == "c" else KvCache(**{**cache, **(c or {})}),
                             None if no == "b" else AttnBatch(**{**batch, **(b or {})}), masks, words, q, ldq, heads, scale, out, ldo, window=window)

    assert call(no="c") == E and call(no="b") == E and call(q=None) == E and call(out=None) == E
    assert call(masks=None) == E and call(masks=P + 4) == E and call(words=0) == E and call(words=-1) == E
    assert call(b={"max_q": 65}) == E and call(words=1 << 28) == U
    assert call(ldq=255) == E and call(ldo=255) == E and call(heads=3) == E and call(window=-1) == E and call(scale=0.0) == E
    assert call(c={"head_dim": 160}, ldq=1024, ldo=1024) == U and call(c={"type": JAM.BF16}) == U
    assert call(b={"n_tokens": 0}) == JAM.OK and call(b={"n_seqs": 0}) == JAM.OK and call(b={"max_q": 0}) == JAM.OK
    tree = dict(n_tokens=2, n_seqs=2, max_q=1, q_offsets=P, parents=P)
    assert hip.tree_masks(None, P, 1) == E and hip.tree_masks(Tree(**{**tree, "parents": None}), P, 1) == E and "tree" in hip.last_error()
    assert hip.tree_masks(Tree(**tree), None, 1) == E and hip.tree_masks(Tree(**{**tree, "max_q": 65}), P, 1) == E
    assert hip.tree_masks(Tree(**{**tree, "n_tokens": 0}), P, 1) == JAM.OK and hip.tree_masks(Tree(**{**tree, "n_seqs": 0}), P, 1) == JAM.OK
    path = dict(ld_path=4, path=P, accepted=P, next=P)
    assert hip.tree_accept(None, P, P, TreePath(**path)) == E and hip.tree_accept(Tree(**tree), P, P, None) == E
    assert hip.tree_accept(Tree(**tree), None, P, TreePath(**path)) == E and hip.tree_accept(Tree(**tree), P, P, TreePath(**{**path, "lens_out": P})) == E
    assert hip.tree_accept(Tree(**{**tree, "n_tokens": 0, "q_offsets": None}), P, P, TreePath(**path)) == E
    assert hip.tree_accept(Tree(**{**tree, "n_seqs": 0}), P, P, TreePath(**path)) == JAM.OK


def test_attn_long_offsets(hip):
    """Pages whose byte offsets pass 32 bits, in a cache of 4.8 GB."""
    import torch
    from qxotic_amd.jam import AttnBatch, KvCache
    kv, dim, page, pages, nq = 8, 128, 64, 36700, 9
    c = KvCache(type=D.F16, kv_heads=kv, head_dim=dim, page_tokens=page, n_pages=pages)
    size = hip.kv_cache_bytes(c)
    assert size > 1 << 32
    r = np.random.default_rng(0)
    bufs = [torch.zeros(size, dtype=torch.uint8, device="cuda") for _ in range(2)]
    c.k, c.v = (b.data_ptr() for b in bufs)
    n, use = 150, [36699, 3, 36650]
    x = r.standard_normal((2, n, kv, dim)).astype(np.float16)
    for buf, rows in zip(bufs, x):
        h = buf.view(torch.float16).view(pages, kv, page, dim)
        for t in range(n):
            h[use[t // page], :, t % page] = torch.from_numpy(rows[t]).cuda()
    q = r.standard_normal((nq, 32 * dim)).astype(np.float32)
    bits = T.ancestors(draft(r, nq))
    t = [i32([0, nq]), i32([n]), i32(use), torch.from_numpy(q).cuda(), torch.from_numpy(T.words(bits, 1).view(np.int64)).cuda()]
    out = torch.zeros((nq, 32 * dim), device="cuda")
    torch.cuda.synchronize()
    b = AttnBatch(n_tokens=nq, n_seqs=1, max_q=nq, max_seq_len=n, q_offsets=t[0].data_ptr(), seq_lens=t[1].data_ptr(), seq_pages=t[2].data_ptr(),
                  ld_seq_pages=3)
    assert hip.attn_tree(c, b, t[4].data_ptr(), 1, t[3].data_ptr(), 32 * dim, 32, dim ** -0.5, out.data_ptr(), 32 * dim) == 0, hip.last_error()
    hip.synchronize()
    got = out.cpu().numpy().reshape(nq, 32, dim)
    keys = [T.seen(n - nq, nq, s) for s in bits]
    for h in range(kv):
        want, mass, big = T.attention(q.reshape(nq, 32, dim)[:, 4 * h:4 * h + 4], x[0][:, h], x[1][:, h], keys, np.float64(np.float32(dim ** -0.5)))
        assert (np.abs(got[:, 4 * h:4 * h + 4] - want) <= (big * (2.0 ** -18 * mass + 2.0 ** -19))[..., None]).all()


def test_a_captured_step(hip):
    """Pages, masks, acceptance, entries moved and pages given back in one graph: replayed with other trees and picks, and with eager calls of the
    same context in between, it does what the definitions say."""
    import torch
    from qxotic_amd.jam import HipJAM, KvCache, KvPages, Tree, TreePath
    jam = HipJAM()
    try:
        r = np.random.default_rng(8)
        n, nodes, page, pages, ld, kv, dim = 5, 12, 16, 64, 12, 2, 64
        rows = n * nodes
        full = lambda *s: torch.full(s, -9, dtype=torch.int32, device="cuda")   # noqa: E731
        lens0 = r.integers(1, 90, n)
        held0 = -(-lens0 // page)
        order = r.permutation(pages)
        table0, used = np.full((n, ld), -5, np.int32), 0
        for i, h in enumerate(held0):
            table0[i, :h] = order[used:used + h]
            used += h
        d = dict(lens=i32(lens0), held=i32(held0), n_free=i32([pages - used]), free=i32(np.concatenate([order[used:], np.full(used, -7)])),
                 table=i32(table0).view(n, ld), targets=full(n), status=full(n), off=full(n + 1), off2=full(n + 1), pos=full(rows), slots=full(rows),
                 parents=full(rows), tokens=full(rows), picked=full(rows), path=full(n, nodes), accepted=full(n), next=full(n), before=full(n),
                 after=full(n), src=full(rows), dst=full(rows), masks=torch.zeros((rows, 1), dtype=torch.int64, device="cuda"))
        cache = [torch.randint(0, 256, (pages * page * kv * (dim + 4),), dtype=torch.uint8, device="cuda") for _ in range(2)]
        p = {k: t.data_ptr() for k, t in d.items()}
        c = KvCache(type=D.Q8_0, kv_heads=kv, head_dim=dim, page_tokens=page, n_pages=pages, k=cache[0].data_ptr(), v=cache[1].data_ptr())
        common = dict(n_seqs=n, page_tokens=page, n_pages=pages, free_cap=pages, ld_seq_pages=ld, held=p["held"], n_free=p["n_free"], free_pages=p["free"],
                      seq_pages=p["table"], lens_out=p["lens"], held_out=p["held"], n_free_out=p["n_free"], status=p["status"])
        up = KvPages(n_tokens=rows, lens=p["before"], targets=p["targets"], q_offsets=p["off"], pos=p["pos"], slots=p["slots"], **common)
        down = KvPages(n_tokens=0, lens=p["lens"], targets=p["after"], q_offsets=p["off2"], **common)
        tree = Tree(n_tokens=rows, n_seqs=n, max_q=nodes, q_offsets=p["off"], parents=p["parents"])
        path = TreePath(ld_path=nodes, path=p["path"], accepted=p["accepted"], next=p["next"], lens=p["before"], lens_out=p["after"], slots=p["slots"],
                        move_from=p["src"], move_to=p["dst"])
        stream = torch.cuda.Stream()
        assert jam.set_stream(stream.cuda_stream) == 0

        def step():
            with torch.cuda.stream(stream):
                d["before"].copy_(d["lens"])
                torch.add(d["lens"], nodes, out=d["targets"])
                assert jam.kv_resize(up) == 0 and jam.tree_masks(tree, p["masks"], 1, p["pos"]) == 0
                assert jam.tree_accept(tree, p["tokens"], p["picked"], path) == 0
                assert jam.kv_move(c, 1, p["off"], n, p["src"], p["dst"], rows) == 0
                assert jam.kv_resize(down) == 0

        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        lens, held, table = lens0.tolist(), held0.tolist(), table0.tolist()
        free = order[used:].tolist()
        for k in range(5):
            trees = [draft(r, nodes) for _ in range(n)]
            tokens, picked = agree(r, trees, vocab=4, share=0.9)
            for name, v in (("parents", trees), ("tokens", tokens), ("picked", picked)):
                d[name].copy_(i32([x for t in v for x in t]))
            before = [b.cpu().numpy() for b in cache]
            torch.cuda.synchronize()
            if k % 2:
                step()
            else:
                graph.replay()
            torch.cuda.synchronize()
            a, rest = T.resize(page, lens, [v + nodes for v in lens], [0] * n, held, free, table, rows)
            paths = [T.walk(*x, nodes) for x in zip(trees, tokens, picked)]
            moves = [[(a["slots"][i * nodes + v], a["slots"][i * nodes + q]) for q, v in enumerate(w) if v != q] for i, (w, _) in enumerate(paths)]
            b, free = T.resize(page, a["lens"], [v + len(w) for v, (w, _) in zip(lens, paths)], [0] * n, a["held"], rest, a["seq_pages"], 0)
            lens, held, table = b["lens"], b["held"], b["seq_pages"]
            got = {x: t.cpu().numpy() for x, t in d.items()}
            assert got["lens"].tolist() == lens and got["held"].tolist() == held and got["table"].tolist() == table
            assert got["n_free"][0] == len(free) and got["free"][:len(free)].tolist() == free and got["next"].tolist() == [x for _, x in paths]
            sets = [s for t in trees for s in T.ancestors(t)]
            assert np.array_equal(got["masks"].view(np.uint64), T.words(sets, 1))
            start = [v - len(w) for v, (w, _) in zip(lens, paths)]
            assert got["pos"].tolist() == [start[i // nodes] + len(s) - 1 for i, s in enumerate(sets)]
            for buf, was in zip(cache, before):   # codes, then scales
                now, at = buf.cpu().numpy(), 0
                for row in (dim, dim // 16):
                    plane = was[at:at + pages * kv * page * row].reshape(pages, kv, page, row)
                    for g in moves:
                        for f, t in g:
                            plane[t // page, :, t % page] = plane[f // page, :, f % page]
                    at += plane.size
                assert np.array_equal(now, was)
    finally:
        jam.close()
