"""GPU: page tables and slots from lengths, and entries moved between slots, against their definitions (oracle/tree.py): whole numbers and
copied bytes, equal in every place."""
import sys

import numpy as np
import pytest

from oracle import decode as D
from oracle import tree as T

pytestmark = pytest.mark.gpu
NAMES = {D.F16: "F16", D.Q8_0: "Q8_0", D.Q4_0: "Q4_0"}


def say(*a):
    print(*a, file=sys.stderr, flush=True)


class Pool:
    """The device arrays of a call; in place by default."""

    KEYS = ("lens", "targets", "base", "held", "n_free", "free_pages", "seq_pages")

    def __init__(self, lens, targets, held, table, free, page, n_pages, n_tokens, base=None, cap=None, apart=False):
        import torch
        self.torch = torch
        dev = lambda a: torch.from_numpy(np.array(a, np.int32).reshape(np.shape(a))).cuda()   # noqa: E731
        self.page, self.n_pages, self.n_tokens, self.cap = page, n_pages, n_tokens, cap or n_pages
        self.host = dict(lens=list(lens), targets=list(targets), held=list(held), table=[list(r) for r in table], free=list(free),
                         base=list(base) if base is not None else [0] * len(lens))
        stack = np.full(self.cap + 3, -77, np.int32)   # the last three lie behind the list
        stack[:len(free)] = free
        self.d = dict(lens=dev(lens), targets=dev(targets), base=None if base is None else dev(base), held=dev(held), n_free=dev([len(free)]),
                      free_pages=dev(stack), seq_pages=dev(np.array(table, np.int32).reshape(len(lens), len(table[0]) if table else 1)))
        n = len(lens)
        for k, of, size in (("lens_out", "lens", n), ("held_out", "held", n), ("n_free_out", "n_free", 1)):
            self.d[k] = dev([-9] * size) if apart else self.d[of]
        self.d.update(status=dev([-9] * (n + 1)), q_offsets=dev([-9] * (n + 2)), pos=dev([-9] * (n_tokens + 2)), slots=dev([-9] * (n_tokens + 2)))

    def struct(self):
        from qxotic_amd.jam import KvPages
        return KvPages(n_seqs=len(self.host["lens"]), n_tokens=self.n_tokens, page_tokens=self.page, n_pages=self.n_pages, free_cap=self.cap,
                       ld_seq_pages=self.d["seq_pages"].shape[1], **{k: None if t is None else t.data_ptr() for k, t in self.d.items()})

    def run(self, hip):
        self.torch.cuda.synchronize()
        assert hip.kv_resize(self.struct()) == 0, hip.last_error()
        hip.synchronize()
        return self

    def check(self):
        h, n = self.host, len(self.host["lens"])
        out, free = T.resize(self.page, h["lens"], h["targets"], h["base"], h["held"], h["free"], h["table"], self.n_tokens)
        get = lambda k: self.d[k].cpu().numpy()   # noqa: E731
        for k, of in (("lens", "lens_out"), ("held", "held_out"), ("n_free", "n_free_out")):
            assert get(of).tolist() == out[k], k
        assert get("status")[:n].tolist() == out["status"] and get("status")[n] == -9
        assert get("q_offsets")[:n + 1].tolist() == out["q_offsets"] and get("q_offsets")[n + 1] == -9
        for k in ("pos", "slots"):
            assert get(k)[:self.n_tokens].tolist() == out[k] and (get(k)[self.n_tokens:] == -9).all(), k
        assert get("seq_pages").tolist() == out["seq_pages"]
        assert get("free_pages")[:len(free)].tolist() == free and (get("free_pages")[self.cap:] == -77).all()
        return out, free


def make(r, n, page, most, grow, spare=4, slack=0, apart=False, shrink=0.3, base=True):
    lens = r.integers(0, most + 1, n)
    targets = np.where(r.random(n) < shrink, r.integers(0, most + 1, n), lens + r.integers(0, grow + 1, n))
    held = -(-lens // page) + r.integers(0, 2, n)
    ld = -(-(most + grow) // page) + 2
    n_pages = n * ld + spare
    order = list(r.permutation(n_pages))
    table = [[order.pop() for _ in range(h)] + [-5] * (ld - h) for h in held]
    need = np.maximum(-(-targets // page) - held, 0).sum()
    free = order[:int(need) + 5 if slack >= 0 else max(0, int(need) // 2)]
    tokens = int(np.maximum(targets - lens, 0).sum()) + max(slack, 0)
    return Pool(lens, targets, held, table, free, page, n_pages, tokens, r.integers(0, 500, n) if base else None, apart=apart)


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("n,page,most,grow", [(1, 16, 0, 1), (1, 16, 40, 33), (3, 1, 9, 5), (64, 16, 300, 32), (65, 7, 90, 100), (200, 64, 1000, 1),
                                              (1023, 16, 100, 40), (1024, 16, 100, 40), (1025, 32, 64, 70), (2500, 16, 50, 9), (2, 16, 100, 40000), (700, 16, 6000, 30),
                                              (1, 1, 5, 1100000)])
def test_resize(hip, n, page, most, grow, apart):
    say("resize", n, page, most, grow, apart)
    r = np.random.default_rng(n + page)
    for slack in (0, 7):
        p = make(r, n, page, most, grow, slack=slack, apart=apart, base=slack == 0)
        p.run(hip).check()


@pytest.mark.parametrize("n", [1, 40, 1024, 2100])
def test_resize_refusals_on_the_device(hip, n):
    """Too few pages, too few token rows, rows of the table too short: those that fit in front are served, those that shrink too."""
    say("resize refused", n)
    r = np.random.default_rng(n)
    p = make(r, n, 16, 200, 60, slack=-1, apart=True, shrink=0.05).run(hip)   # few pages come back
    out, _ = p.check()
    assert n < 40 or 0 < sum(out["status"]) < n
    p = make(r, n, 16, 200, 60, apart=True)
    p.n_tokens //= 2
    for k in ("pos", "slots"):
        p.d[k] = p.d[k][:p.n_tokens + 2].clone()
        p.d[k].fill_(-9)
    out, _ = p.run(hip).check()
    assert n < 40 or 0 < sum(out["status"]) < n
    p = make(r, n, 16, 200, 60, apart=True, shrink=0.5)
    p.host["targets"][n // 2] = 16 * p.d["seq_pages"].shape[1] + 1
    p.d["targets"][n // 2] = p.host["targets"][n // 2]
    out, _ = p.run(hip).check()
    assert out["status"][n // 2] == 1


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("n", [3, 1500])
def test_resize_refused_with_pages_to_spare(hip, n, apart):
    """A refused sequence that held more pages than its target needs: those are on the list, once, and it holds the rest."""
    r = np.random.default_rng(n)
    lens, targets, held = [30] * n, [33] * n, [int(v) for v in r.integers(2, 7, n)]
    order = list(r.permutation(8 * n))
    table = [[int(order.pop()) for _ in range(h)] + [-5] * (8 - h) for h in held]
    p = Pool(lens, targets, held, table, [], 16, 8 * n, 3 * (n // 2), apart=apart)
    out, free = p.run(hip).check()
    assert sum(out["status"]) > 0
    kept = [row[c] for row, h in zip(out["seq_pages"], out["held"]) for c in range(h)]
    assert len(set(kept + free)) == len(kept) + len(free)   # no page twice


def test_resize_nothing_and_extremes(hip):
    """No sequences, no tokens, lengths below zero and up to the largest integer, counts that the list cannot hold, pages outside the cache."""
    p = Pool([], [], [], [], [3, 1], 16, 4, 2)
    p.run(hip)
    assert p.d["slots"].cpu().tolist() == [-1, -1, -9, -9] and p.d["q_offsets"].cpu().tolist()[0] == 0 and p.d["n_free"].cpu().tolist() == [2]
    p = Pool([5, 9], [5, 3], [1, 1], [[0], [1]], [2], 16, 3, 0).run(hip)
    p.check()
    big = (1 << 31) - 1
    p = Pool([-5, big, 3, big], [-7, big, big, 0], [0, 2, 1, 2], [[-1, -1], [0, 1], [2, -1], [3, 4]], [5, 6], 16, 8, 9, apart=True).run(hip)
    p.check()
    for n_free in (-3, 1 << 30):
        p = Pool([0, 40], [20, 3], [0, 3], [[-1] * 4, [0, 1, 2, -1]], [5, 6], 16, 8, 20, cap=4, apart=True)
        p.d["n_free"].fill_(n_free)
        p.run(hip)
        assert (p.d["free_pages"].cpu()[4:] == -77).all() and 0 <= int(p.d["n_free_out"]) <= 4
    p = Pool([0, 0], [20, 3], [9, -4], [[99, -8, 1, 1]] * 2, [1 << 30, 6], 16, 8, 23, apart=True).run(hip)   # held past the row, bad pages
    slots = p.d["slots"].cpu().numpy()[:23]
    assert (slots[:20] == -1).all() and (slots[20:] < 8 * 16).all()


def test_resize_up_and_down(hip):
    """A step's room taken and given back, in place, replayed: the list, the table and the lengths are what they were."""
    import torch
    from qxotic_amd.jam import HipJAM
    jam = HipJAM()
    try:
        r = np.random.default_rng(3)
        p = make(r, 50, 16, 200, 30, shrink=0.0)
        before = {k: p.d[k].clone() for k in ("lens", "held", "n_free")}
        n_free = int(p.d["n_free"])
        top = p.d["free_pages"][:n_free].clone()
        up = p.struct()
        back = p.d["lens"].clone()
        # down to the lengths before, which need the pages that were held before
        p.d["held"].copy_(torch.tensor([-(-v // 16) for v in p.host["lens"]], dtype=torch.int32))
        before["held"] = p.d["held"].clone()
        down = p.struct()
        down.targets = back.data_ptr()
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        assert jam.set_stream(stream.cuda_stream) == 0
        assert jam.kv_resize(up) == 0 and jam.kv_resize(down) == 0
        jam.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            assert jam.kv_resize(up) == 0 and jam.kv_resize(down) == 0
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            for k, t in before.items():
                assert torch.equal(p.d[k], t), k
            assert torch.equal(p.d["free_pages"][:n_free], top)
    finally:
        jam.close()


def moved(kind, bufs, kv, dim, page, pages, groups):
    """The buffers after the entries of each group, one after another."""
    rows = [{D.F16: 2 * dim, D.Q8_0: dim, D.Q4_0: dim // 2}[kind]] + ([dim // 16] if kind != D.F16 else [])
    out = []
    for buf in bufs:
        buf, at = buf.copy(), 0
        for row in rows:
            plane = buf[at:at + pages * kv * page * row].reshape(pages, kv, page, row)
            at += plane.size
            for g in groups:
                for f, t in g:
                    if 0 <= f < pages * page and 0 <= t < pages * page:
                        plane[t // page, :, t % page] = plane[f // page, :, f % page]
        out.append(buf)
    return out


def move(hip, kind, kv, dim, page, pages, groups, layers, seed=0, tail=()):
    import torch
    from qxotic_amd.jam import KvCache
    r = np.random.default_rng(seed)
    size = pages * page * kv * ({D.F16: 2 * dim, D.Q8_0: dim, D.Q4_0: dim // 2}[kind] + (dim // 16 if kind != D.F16 else 0))
    host = [r.integers(0, 256, size, dtype=np.uint8) for _ in range(2 * layers)]
    devs = [torch.from_numpy(b).cuda() for b in host]
    caches = (KvCache * layers)(*(KvCache(type=kind, kv_heads=kv, head_dim=dim, page_tokens=page, n_pages=pages, k=devs[2 * i].data_ptr(),
                                          v=devs[2 * i + 1].data_ptr()) for i in range(layers)))
    flat = [e for g in groups for e in g] + list(tail)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()   # noqa: E731
    off, src, dst = i32(np.cumsum([0] + [len(g) for g in groups]).tolist()), i32([f for f, _ in flat] or [0]), i32([t for _, t in flat] or [0])
    torch.cuda.synchronize()
    assert hip.kv_move(caches, layers, off.data_ptr(), len(groups), src.data_ptr(), dst.data_ptr(), len(flat)) == 0, hip.last_error()
    hip.synchronize()
    want = moved(kind, host, kv, dim, page, pages, groups)
    for i, (w, d) in enumerate(zip(want, devs)):
        assert np.array_equal(w, d.cpu().numpy()), i


def paths(r, n, nodes, page, spare=2):
    """Groups of a rising path's entries to their sequence's first slots, in a random order of pages."""
    per = -(-nodes // page)
    order, groups = r.permutation(n * per + spare), []
    for i in range(n):
        slot = lambda k: int(order[i * per + k // page] * page + k % page)   # noqa: B023, E731
        keep = np.sort(r.permutation(nodes)[:r.integers(0, nodes + 1)])
        g = [(slot(c), slot(k)) if c != k else (-1, -1) for k, c in enumerate(keep)]
        groups.append(g + [(-1, -1)] * (nodes - len(g)))
    return groups, n * per + spare


@pytest.mark.parametrize("kind", [D.F16, D.Q8_0, D.Q4_0])
@pytest.mark.parametrize("kv,dim,page,n,nodes,layers", [(1, 64, 16, 1, 1, 1), (8, 128, 16, 5, 25, 3), (2, 96, 7, 3, 70, 2), (1, 32, 1, 4, 9, 1),
                                                        (3, 160, 32, 2, 130, 1), (4, 256, 16, 30, 12, 2), (2, 64, 16, 3, 5, 131)])
def test_move_paths(hip, kind, kv, dim, page, n, nodes, layers):
    say("move", NAMES[kind], kv, dim, page, n, nodes, layers)
    r = np.random.default_rng(dim + n)
    groups, pages = paths(r, n, nodes, page)
    move(hip, kind, kv, dim, page, pages, groups, layers, seed=n)


def test_move_in_order(hip):
    """Entries of a group that read what an earlier one wrote, or write the same slot again; slots outside the cache; nothing to do."""
    say("move in order")
    shift = [(i, i + 1) for i in range(40)]
    back = [(i + 1, i) for i in range(50, 70)]
    for kind in (D.F16, D.Q8_0, D.Q4_0):
        move(hip, kind, 2, 64, 16, 8, [shift, back, [(100, 90), (101, 90), (90, 91), (-1, 92), (93, -1), (128, 94), (95, 1 << 30), (96, 97)]], 2)
        move(hip, kind, 2, 64, 16, 8, [[(i, (7 * i + 3) % 128) for i in range(128)]], 1)
        move(hip, kind, 2, 64, 16, 8, [[], [], []], 1, tail=[(1, 2), (3, 4)])   # entries of no group
    move(hip, D.F16, 1, 8, 16, 4, [[(1, 2), (2, 3)]], 1)   # the smallest row
    move(hip, D.Q8_0, 5, 64, 16, 8, [[(i, 64 + i) for i in range(64)]], 1)


def test_move_device_offsets_out_of_range(hip):
    """Offsets below zero, past the entries and falling: nothing outside the arrays is looked at, and no other slot changes."""
    import torch
    from qxotic_amd.jam import KvCache
    a = [torch.randint(0, 256, (4 * 16 * 128,), dtype=torch.uint8, device="cuda") for _ in range(2)]
    c = KvCache(type=D.F16, kv_heads=1, head_dim=64, page_tokens=16, n_pages=4, k=a[0].data_ptr(), v=a[1].data_ptr())
    before = [t.clone() for t in a]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()   # noqa: E731
    off, src, dst = i32([-5, 1 << 30, 3, 2]), i32([5, 6, 7, 8]), i32([9, 9, 9, 9])
    torch.cuda.synchronize()
    assert hip.kv_move(c, 1, off.data_ptr(), 3, src.data_ptr(), dst.data_ptr(), 4) == 0, hip.last_error()
    hip.synchronize()
    for b, t in zip(before, a):
        b.view(4 * 16, 128)[9] = b.view(4 * 16, 128)[8]
        assert torch.equal(b, t)


def test_move_long_offsets(hip):
    """Slots whose byte offsets pass 32 bits."""
    import torch
    from qxotic_amd.jam import KvCache
    kv, dim, page, pages = 8, 128, 64, 36700
    for kind, row in ((D.F16, 256), (D.Q8_0, 128)):
        c = KvCache(type=kind, kv_heads=kv, head_dim=dim, page_tokens=page, n_pages=pages)
        size = hip.kv_cache_bytes(c)
        if kind == D.F16:
            assert size > 1 << 32
        k = torch.zeros(size, dtype=torch.uint8, device="cuda")
        v = torch.zeros(size, dtype=torch.uint8, device="cuda")
        c.k, c.v = k.data_ptr(), v.data_ptr()
        plane = k[:pages * kv * page * row].view(pages, kv, page, row)
        x = torch.randint(0, 256, (kv, row), dtype=torch.uint8, device="cuda")
        plane[pages - 1, :, 3] = x
        i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()   # noqa: E731
        off, src, dst = i32([0, 1]), i32([(pages - 1) * page + 3]), i32([(pages - 2) * page + 63])
        torch.cuda.synchronize()
        assert hip.kv_move(c, 1, off.data_ptr(), 1, src.data_ptr(), dst.data_ptr(), 1) == 0, hip.last_error()
        hip.synchronize()
        assert torch.equal(plane[pages - 2, :, 63], x) and int((plane != 0).any(-1).sum()) <= 2 * kv


def test_refusals(hip):
    """Through the entry points, before any work: the pointers here lead nowhere."""
    from qxotic_amd.jam import JAM, KvCache, KvPages
    P = 1 << 20
    assert hip.kv_resize(None) == JAM.EINVAL and hip.kv_resize(KvPages(n_seqs=1, page_tokens=16)) == JAM.EINVAL and "kv_resize" in hip.last_error()
    c = dict(type=JAM.Q8_0, kv_heads=2, head_dim=64, page_tokens=16, n_pages=4, k=P, v=P)
    two = lambda **kw: (KvCache * 2)(KvCache(**c), KvCache(**{**c, **kw}))   # noqa: E731
    assert hip.kv_move(two(head_dim=96), 2, P, 1, P, P, 1) == JAM.EINVAL and "kv_move" in hip.last_error()
    assert hip.kv_move(two(k=P + 4), 2, P, 1, P, P, 1) == JAM.EINVAL and hip.kv_move(two(v=None), 2, P, 1, P, P, 1) == JAM.EINVAL
    assert hip.kv_move(KvCache(**{**c, "type": JAM.BF16}), 1, P, 1, P, P, 1) == JAM.EUNSUPPORTED
    assert hip.kv_move(two(), 2, None, 1, P, P, 1) == JAM.EINVAL
    assert hip.kv_move(two(), 2, None, 0, P, P, 1) == JAM.OK and hip.kv_move(None, 0, P, 1, P, P, 1) == JAM.OK
