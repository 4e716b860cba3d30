"""GPU: attention of ragged batches over the paged cache, shared prefixes, against its definition in 64 bits (oracle/decode.py) on the
values that the cache's codes stand for.

Tolerance. With S the largest scale · Σ|q_d k_d| of a row's keys, a score is off by less than 2^-19 · S: the query is carried to 22
bits (2^-22 a product), and the sum of up to 256 products in f32 adds roundings of 2^-24 that partly cancel (16 of them in a row give
2^-20). A weight is off by that relative to itself, the numerator and the sum alike, so an output by twice it times the largest value;
the weights' own rounding (2^-21) and the sums' (a few 2^-23) add 2^-19. So |error| <= max|v| · (2^-18 · S + 2^-19)."""
import sys

import numpy as np
import pytest

from oracle import decode as D

pytestmark = pytest.mark.gpu
NAMES = {D.F16: "F16", D.Q8_0: "Q8_0", D.Q4_0: "Q4_0"}
KINDS = [D.F16, D.Q8_0, D.Q4_0]


def say(*a):
    print(*a, file=sys.stderr, flush=True)


class Batch:
    """groups: [(prefix tokens, [(own tokens, query tokens), ...])]; then sequences without a prefix."""

    def __init__(self, kind, kv, grp, dim, page, groups, alone=(), window=0, sinks=False, seed=0, pad=0, spare_pages=3, loud=False):
        import torch
        r = np.random.default_rng(seed)
        self.kind, self.kv, self.grp, self.dim, self.page, self.window, self.pad = kind, kv, grp, dim, page, window, pad
        seqs = [s for _, m in groups for s in m] + list(alone)
        self.seqs, self.prefixes = seqs, [p for p, _ in groups]
        cuts = np.cumsum([0] + [len(m) for _, m in groups])
        self.of = [next((j for j in range(len(groups)) if cuts[j] <= i < cuts[j + 1]), None) for i in range(len(seqs))]
        need = lambda n: -(-n // page)   # noqa: E731
        total = sum(need(n) for n, _ in seqs) + sum(need(p) for p in self.prefixes)
        self.pages = total + spare_pages
        free = list(r.permutation(self.pages))
        slots = self.pages * page
        x = r.standard_normal((2, slots, kv, dim)).astype(np.float32)
        x[:, :, :, r.integers(0, dim, 3)] *= 3
        if loud:   # scores that grow along the sequence, so that the running maximum moves
            x[0] *= (1 + 3 * r.random((slots, 1, 1))).astype(np.float32)
        self.vals = [D.entry(kind, a) for a in x]
        self.bufs = [D.pack(kind, a, kv, page, self.pages, range(slots)) for a in x]

        def table(lens):
            w = max([need(n) for n in lens], default=0) + 1
            t = np.full((max(1, len(lens)), w), -3, np.int32)   # past a sequence's pages: never looked at
            for i, n in enumerate(lens):
                t[i, :need(n)] = [free.pop() for _ in range(need(n))]
            return t

        self.own, self.shared = table([n for n, _ in seqs]), table(self.prefixes)
        self.used = np.zeros(slots, bool)
        self.sinks = r.standard_normal(kv * grp).astype(np.float32) if sinks else None
        self.scale = 1 / np.sqrt(dim)
        self.off = np.cumsum([0] + [q for _, q in seqs]).astype(np.int32)
        self.n = int(self.off[-1])
        self.q = (r.standard_normal((self.n, kv * grp * dim + pad)) * 1.5).astype(np.float32)
        self.cuts, self.torch = cuts.astype(np.int32), torch

    def slots(self, i):
        """The sequence's slots, prefix first."""
        j = self.of[i]
        out = []
        for t, n in (((self.shared[j], self.prefixes[j]),) if j is not None else ()) + ((self.own[i], self.seqs[i][0]),):
            at = np.arange(n)
            out.append(t[at // self.page].astype(np.int64) * self.page + at % self.page)
        return np.concatenate(out)

    def run(self, hip, times=1, max_q=None, extra=0):
        from qxotic_amd.jam import AttnBatch, KvCache
        torch, dev = self.torch, lambda a: self.torch.from_numpy(np.ascontiguousarray(a)).cuda()   # noqa: E731
        self.dev = dict(k=dev(self.bufs[0]), v=dev(self.bufs[1]), off=dev(self.off), lens=dev(np.array([n for n, _ in self.seqs], np.int32)),
                        own=dev(self.own), cuts=dev(self.cuts), plens=dev(np.array(self.prefixes or [0], np.int32)), shared=dev(self.shared),
                        q=dev(self.q), sinks=None if self.sinks is None else dev(self.sinks))
        d = {k: None if t is None else t.data_ptr() for k, t in self.dev.items()}
        w = self.kv * self.grp * self.dim
        self.out = torch.full((self.n + extra, w + self.pad), -5.0, device="cuda")
        c = KvCache(type=self.kind, kv_heads=self.kv, head_dim=self.dim, page_tokens=self.page, n_pages=self.pages, k=d["k"], v=d["v"])
        b = AttnBatch(n_tokens=self.n + extra, n_seqs=len(self.seqs), n_prefixes=len(self.prefixes),
                      max_q=max_q or max(q for _, q in self.seqs), max_seq_len=max(n for n, _ in self.seqs),
                      max_prefix_len=max(self.prefixes, default=0), q_offsets=d["off"], seq_lens=d["lens"], seq_pages=d["own"],
                      ld_seq_pages=self.own.shape[1], prefix_seqs=d["cuts"], prefix_lens=d["plens"], prefix_pages=d["shared"],
                      ld_prefix_pages=self.shared.shape[1])
        self.call = lambda: hip.attn_shared_prefix(c, b, d["q"], w + self.pad, self.kv * self.grp, self.scale, self.out.data_ptr(),
                                                   w + self.pad, window=self.window, sinks_dev=d["sinks"])   # noqa: E731
        torch.cuda.synchronize()
        for _ in range(times):
            assert self.call() == 0, hip.last_error()
        hip.synchronize()
        return self.out.cpu().numpy()

    def want(self, i, kv):
        """(out, tolerance) of sequence i's queries, key head kv: [q, grp, dim]."""
        own, nq = self.seqs[i]
        at = self.slots(i)
        pos = len(at) - nq + np.arange(nq)
        w = self.grp * self.dim
        q = self.q[self.off[i]:self.off[i + 1], kv * w:(kv + 1) * w].reshape(nq, self.grp, self.dim)
        sinks = None if self.sinks is None else self.sinks[kv * self.grp:(kv + 1) * self.grp].astype(np.float64)
        out, mass, big = D.attention(q, self.vals[0][at, kv], self.vals[1][at, kv], pos, np.float64(np.float32(self.scale)), self.window, sinks)
        return out, (big * (2.0 ** -18 * mass + 2.0 ** -19))[..., None]

    def check(self, got, skip=()):
        w = self.kv * self.grp * self.dim
        worst = 0.0
        for i, (_, nq) in enumerate(self.seqs):
            if i in skip or nq == 0:
                continue
            for c in range(self.kv):
                want, tol = self.want(i, c)
                g = got[self.off[i]:self.off[i + 1], c * self.grp * self.dim:(c + 1) * self.grp * self.dim].reshape(want.shape)
                ok = np.abs(g - want) <= tol
                assert ok.all(), (i, c, np.argwhere(~ok)[:4].tolist(), float(np.nanmax(np.abs(g - want))), float(tol.max()))
                worst = max(worst, float((np.abs(g - want) / np.maximum(tol, 1e-30)).max()))
        if self.pad:
            assert (got[:, w:] == -5.0).all()
        say(f"   largest error {worst:.3f} of the tolerance")


# name: (kv, grp, dim, page, groups, alone, window, sinks)
CASES = {
    "one_token": (1, 1, 64, 16, [], [(1, 1)], 0, False),
    "one_sequence": (2, 4, 128, 16, [(70, [(45, 1)])], [], 0, False),
    "one_sequence_long": (1, 4, 128, 16, [], [(3001, 1)], 0, True),
    "decode_shared": (2, 4, 128, 16, [(300, [(1 + 17 * i, 1) for i in range(9)])], [], 0, False),
    "decode_shared_long": (1, 4, 64, 16, [(2100, [(3 + 5 * i, 1) for i in range(40)])], [], 0, False),
    "decode_groups": (1, 8, 128, 64, [(257, [(5, 1), (130, 1)]), (1, [(9, 1)]), (64, [(64, 1), (1, 1), (63, 1)])], [(77, 1)], 0, False),
    "decode_96": (2, 7, 96, 32, [(131, [(33, 1), (2, 1), (95, 1)])], [], 0, True),
    "decode_256": (1, 2, 256, 16, [(200, [(50, 1), (7, 1), (19, 1), (128, 1)])], [], 0, False),
    "decode_192": (1, 16, 192, 16, [(90, [(50, 1), (7, 1)])], [], 0, False),
    "decode_window": (2, 4, 64, 16, [(500, [(3, 1), (40, 1), (129, 1), (400, 1)])], [(300, 1), (5, 1)], 128, False),
    "decode_window_1": (1, 4, 64, 16, [(50, [(3, 1), (40, 1)])], [], 1, True),
    "few_tokens": (2, 4, 128, 16, [(123, [(7, 5), (40, 8), (3, 3), (64, 1)])], [], 0, False),
    "few_tokens_window": (1, 7, 96, 16, [(200, [(7, 5), (90, 8), (3, 3)])], [(11, 11)], 20, True),
    "prompt": (2, 4, 128, 16, [(100, [(150, 150), (97, 97), (64, 10)])], [], 0, False),
    "prompt_64": (1, 8, 64, 16, [(333, [(129, 129), (77, 77)])], [(40, 40), (1, 1)], 0, True),
    "prompt_window": (1, 4, 128, 16, [(150, [(200, 200)])], [(90, 90)], 50, False),
    "prompt_256": (1, 2, 256, 32, [(70, [(90, 90)])], [(33, 33)], 0, False),
    "prompt_96": (2, 3, 96, 128, [(70, [(190, 190), (2, 2)])], [], 0, False),
    "prompt_192": (1, 1, 192, 16, [], [(140, 140)], 0, False),
    "prompt_alone_long": (1, 1, 64, 16, [], [(700, 700), (20, 3)], 0, False),
    "groups_of_one": (2, 1, 64, 16, [(40, [(20, 1)]), (50, [(30, 1)]), (3, [(3, 1)])], [], 0, False),
    "empty_sequences": (1, 4, 64, 16, [(40, [(0, 0), (20, 1), (0, 0)]), (0, [(3, 1)])], [(0, 0), (0, 1), (5, 0)], 0, False),
    "empty_rows_sinks": (1, 4, 64, 16, [], [(0, 1), (0, 2), (9, 2)], 0, True),
    "more_queries_than_keys": (1, 2, 64, 16, [(10, [(2, 5), (0, 3)])], [(2, 6)], 0, False),
    "group_16": (1, 16, 128, 16, [(130, [(20, 1), (33, 1)])], [(61, 1)], 0, False),
    "group_20": (1, 20, 64, 16, [(130, [(20, 1), (33, 2)])], [(61, 1)], 0, False),
    "many_sequences": (1, 4, 64, 16, [(200, [(1 + i % 37, 1) for i in range(70)])], [(9, 1)], 0, False),
    "many_groups": (1, 2, 64, 16, [(130 + j % 9, [(3, 1), (20, 1 + j % 3)]) for j in range(66)], [], 0, False),
    "many_sequences_prompts": (1, 1, 64, 16, [(140, [(9, 3) for _ in range(40)]), (150, [(30 + i, 30) for i in range(3)])],
                               [(5, 2) for _ in range(30)], 17, False),
    # prefixes that are read once for their group: 128-, 32- and 16-row tiles, groups beyond a wave's lanes
    "grouped_128": (8, 4, 64, 16, [(1301, [(1 + 3 * i, 1) for i in range(40)])], [(9, 1)], 0, False),
    "grouped_128_dim_128": (8, 4, 128, 16, [(1300, [(1 + 2 * i, 1) for i in range(40)])], [], 0, True),
    "grouped_32": (8, 3, 64, 16, [(2000, [(3 + i, 1) for i in range(20)]), (1931, [(1 + i, 1) for i in range(12)])], [], 0, False),
    "grouped_16": (8, 1, 96, 16, [(4100, [(1 + i, 1) for i in range(15)])], [], 0, False),
    "grouped_window": (8, 2, 64, 16, [(1500, [(1 + 60 * i, 1) for i in range(36)])], [], 1000, True),
    "grouped_tokens": (8, 2, 64, 64, [(1400, [(3 + i, 1 + i % 4) for i in range(38)])], [(30, 4)], 0, False),
    "grouped_many": (8, 2, 64, 16, [(1950 - j % 5, [(1 + (i + j) % 20, 1) for i in range(8)]) for j in range(67)], [(7, 1)], 0, False),
    "grouped_256": (8, 1, 256, 16, [(2300, [(1 + i, 1) for i in range(24)])], [], 0, False),
    "grouped_192": (8, 2, 192, 16, [(2300, [(1 + i, 1) for i in range(24)])], [], 0, False),
    "page_1": (1, 2, 64, 1, [(33, [(20, 1), (70, 2)])], [], 0, False),
    "page_7": (1, 2, 64, 7, [(133, [(20, 1), (70, 2)])], [(100, 60)], 0, False),
    "page_1000": (1, 2, 64, 1000, [(133, [(20, 1), (70, 2)])], [(1001, 60)], 0, False),
}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("name", CASES)
def test_attn(hip, kind, name):
    kv, grp, dim, page, groups, alone, window, sinks = CASES[name]
    say("attn", NAMES[kind], name)
    b = Batch(kind, kv, grp, dim, page, groups, alone, window, sinks, seed=len(name) + kind)
    got = b.run(hip)
    b.check(got)
    assert np.array_equal(b.run(hip, times=2), got)   # the same bits again


@pytest.mark.parametrize("name", ["decode_shared", "few_tokens", "prompt", "one_sequence_long"])
def test_attn_strides_and_growing_scores(hip, name):
    """Rows further apart than their elements; scores whose running maximum moves along the keys; sharp ones."""
    kv, grp, dim, page, groups, alone, window, sinks = CASES[name]
    for scale in (1.0, 8.0):
        say("attn strides", name, scale)
        b = Batch(D.Q8_0, kv, grp, dim, page, groups, alone, window, sinks, seed=3, pad=8, loud=True)
        b.q *= np.float32(scale)
        b.check(b.run(hip))
    b = Batch(D.F16, kv, grp, dim, page, groups, alone, window, sinks, seed=4, pad=3)   # rows at 4-byte alignment
    b.check(b.run(hip))


@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("name", ["one_sequence", "decode_shared", "decode_window", "few_tokens_window", "prompt", "prompt_64", "decode_256",
                                  "grouped_128", "grouped_16", "grouped_window", "grouped_tokens"])
def test_attn_masked_entries_change_nothing(hip, name, value):
    """Every entry that no query sees holds NaN or Inf: what lies past the lengths in a page, and, with queries in the middle of a
    prompt, keys and values that later ones see. Rows that do see such an entry are not looked at."""
    kv, grp, dim, page, groups, alone, window, sinks = CASES[name]
    say("attn masked", name, value)
    b = Batch(D.F16, kv, grp, dim, page, groups, alone, window, sinks, seed=9)
    seen = np.zeros(b.pages * page, bool)
    first_bad = {}
    for i, (own, nq) in enumerate(b.seqs):
        at = b.slots(i)
        seen[at] = True
    rows = kv * page * dim
    for which, buf in enumerate(b.bufs):
        h = buf.view(np.float16).reshape(b.pages, kv, page, dim)
        for s in np.nonzero(~seen)[0]:
            h[s // page, :, s % page] = value
        # the last own token of each sequence with several queries: only its last query sees it
        for i, (own, nq) in enumerate(b.seqs):
            if nq > 1:
                s = b.slots(i)[-1]
                h[s // page, :, s % page] = value
                first_bad[i] = nq - 1
            elif window and len(b.slots(i)) > window:
                s = b.slots(i)[0]   # shared with sequences that may see it
                if all(len(b.slots(j)) - b.seqs[j][1] >= window for j in range(len(b.seqs)) if b.of[j] == b.of[i]):
                    h[s // page, :, s % page] = value
    assert rows
    got = b.run(hip)
    for i, (own, nq) in enumerate(b.seqs):
        stop = first_bad.get(i, nq)
        for c in range(kv):
            want, tol = b.want(i, c)
            g = got[b.off[i]:b.off[i + 1], c * grp * dim:(c + 1) * grp * dim].reshape(want.shape)[:stop]
            assert (np.abs(g - want[:stop]) <= tol[:stop]).all(), (i, c)


def test_attn_sees_non_finite(hip):
    """A row that does see a NaN value is NaN in that element, others are not touched by it."""
    b = Batch(D.F16, 1, 4, 64, 16, [(40, [(20, 1), (30, 1)])], [], seed=1)
    s = b.slots(0)[-1]
    h = b.bufs[1].view(np.float16).reshape(b.pages, 1, 16, 64)
    h[s // 16, 0, s % 16, 5] = np.nan
    got = b.run(hip).reshape(2, 4, 64)
    assert np.isnan(got[0, :, 5]).all() and not np.isnan(np.delete(got[0], 5, 1)).any() and not np.isnan(got[1]).any()


def test_attn_device_lengths_past_the_maxima(hip):
    """Lengths, offsets and pages that are out of range: nothing outside the buffers is looked at, sequences with good ones keep
    their results, query tokens of no sequence and past max_q are not written."""
    b = Batch(D.Q8_0, 1, 4, 64, 16, [(40, [(20, 1), (30, 1), (17, 1)])], [(25, 1), (12, 1)], seed=2)
    b.own[1, 0] = 1 << 30
    b.own[1, 1] = -9
    got = b.run(hip)
    b.check(got, skip=(1,))
    assert np.isfinite(got).all()
    got = b.run(hip, extra=3)
    b.check(got, skip=(1,))
    assert (got[b.n:] == -5.0).all()
    b = Batch(D.Q8_0, 1, 4, 64, 16, [(40, [(20, 3), (30, 1)])], [(25, 2)], seed=2)
    got = b.run(hip, max_q=2)
    b.check(got, skip=(0,))
    assert (got[2] == -5.0).all()


def test_attn_long_offsets(hip):
    """Pages whose byte offsets pass 32 bits, in a cache of 4.8 GB."""
    import torch
    from qxotic_amd.jam import AttnBatch, KvCache
    kv, dim, page, pages = 8, 128, 64, 36700
    c = KvCache(type=D.F16, kv_heads=kv, head_dim=dim, page_tokens=page, n_pages=pages)
    size = hip.kv_cache_bytes(c)
    assert size > 1 << 32
    r = np.random.default_rng(0)
    k, v = torch.zeros(size, dtype=torch.uint8, device="cuda"), torch.zeros(size, dtype=torch.uint8, device="cuda")
    c.k, c.v = k.data_ptr(), v.data_ptr()
    n, use = 150, [36699, 3, 36650]
    x = r.standard_normal((2, n, kv, dim)).astype(np.float16)
    for buf, rows in ((k, x[0]), (v, x[1])):
        h = buf.view(torch.float16).view(pages, kv, page, dim)
        for t in range(n):
            h[use[t // page], :, t % page] = torch.from_numpy(rows[t]).cuda()
    q = r.standard_normal((1, 32 * dim)).astype(np.float32)
    t = [torch.from_numpy(a).cuda() for a in (np.array([0, 1], np.int32), np.array([n], np.int32), np.array([use], np.int32), q)]
    out = torch.zeros((1, 32 * dim), device="cuda")
    torch.cuda.synchronize()
    b = AttnBatch(n_tokens=1, n_seqs=1, max_q=1, max_seq_len=n, q_offsets=t[0].data_ptr(), seq_lens=t[1].data_ptr(),
                  seq_pages=t[2].data_ptr(), ld_seq_pages=3)
    assert hip.attn_shared_prefix(c, b, t[3].data_ptr(), 32 * dim, 32, dim ** -0.5, out.data_ptr(), 32 * dim) == 0, hip.last_error()
    hip.synchronize()
    got = out.cpu().numpy().reshape(32, dim)
    for h in range(kv):
        want, mass, big = D.attention(q.reshape(1, 32, dim)[:, 4 * h:4 * h + 4], x[0][:, h], x[1][:, h], [n - 1], np.float64(np.float32(dim ** -0.5)))
        assert (np.abs(got[4 * h:4 * h + 4] - want[0]) <= (big * (2.0 ** -18 * mass + 2.0 ** -19))[0][:, None]).all()


@pytest.mark.parametrize("name", ["decode_shared", "one_sequence", "prompt", "grouped_32"])
def test_attn_in_a_graph_and_on_another_stream(hip, name):
    """Captured once, replayed with other queries and after larger eager calls of the same context: the eager results' bits."""
    import torch
    from qxotic_amd.jam import HipJAM
    kv, grp, dim, page, groups, alone, window, sinks = CASES[name]
    jam = HipJAM()
    try:
        b = Batch(D.Q8_0, kv, grp, dim, page, groups, alone, window, sinks, seed=5)
        eager = b.run(jam)
        stream = torch.cuda.Stream()
        assert jam.set_stream(stream.cuda_stream) == 0
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            assert b.call() == 0
        big = Batch(D.Q8_0, kv, grp, dim, page, [(400, [(200, 3)] * 6)], [], seed=6)
        for k in range(3):
            big.run(jam)
            scaled = (b.q * np.float32(1 + k)).astype(np.float32)
            b.dev["q"].copy_(torch.from_numpy(scaled))
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
    """What is refused is refused before any work: the pointers here lead nowhere."""
    from qxotic_amd.jam import JAM, AttnBatch, KvCache
    P, E, U = 1 << 20, JAM.EINVAL, JAM.EUNSUPPORTED
    cache = dict(type=JAM.Q8_0, kv_heads=2, head_dim=64, page_tokens=16, n_pages=4, k=P, v=P)
    batch = dict(n_tokens=2, n_seqs=2, n_prefixes=1, max_q=1, max_seq_len=33, max_prefix_len=17, q_offsets=P, seq_lens=P, seq_pages=P,
                 ld_seq_pages=3, prefix_seqs=P, prefix_lens=P, prefix_pages=P, ld_prefix_pages=2)

    def call(c=None, b=None, q=P, ldq=256, heads=4, scale=0.125, out=P, ldo=256, window=0, no=None):
        return hip.attn_shared_prefix(None if no == "c" else KvCache(**{**cache, **(c or {})}),
                                      None if no == "b" else AttnBatch(**{**batch, **(b or {})}), q, ldq, heads, scale, out, ldo, window=window)

    assert call(no="c") == E and call(no="b") == E and call(q=None) == E and call(out=None) == E
    assert call(ldq=255) == E and call(ldo=255) == E and call(heads=3) == E and call(heads=0) == E and call(window=-1) == E
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert call(scale=scale) == E
    for key in ("n_tokens", "n_seqs", "n_prefixes", "max_q", "max_seq_len", "max_prefix_len"):
        assert call(b={key: -1}) == E, key
    for key in ("q_offsets", "seq_lens", "seq_pages", "prefix_seqs", "prefix_lens", "prefix_pages"):
        assert call(b={key: None}) == E, key
    assert call(b={"ld_seq_pages": 2}) == E and call(b={"ld_prefix_pages": 1}) == E
    assert call(c={"head_dim": 32}, ldq=128) == U and call(c={"head_dim": 160}, ldq=1024, ldo=1024) == U
    assert call(c={"type": JAM.BF16}) == U and call(c={"k": P + 4}) == E
    assert call(b={"max_seq_len": 1 << 30, "max_prefix_len": 1 << 30, "ld_seq_pages": 1 << 28, "ld_prefix_pages": 1 << 28}) == U
    assert "attn" in hip.last_error()
    assert call(b={"n_tokens": 0}) == JAM.OK and call(b={"n_seqs": 0}) == JAM.OK and call(b={"max_q": 0}) == JAM.OK
