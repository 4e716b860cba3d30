"""GPU: sequences that jamhip_kv_resize refused, through the rest of a step with drafted trees: their drafted tokens have no slots, so nothing
was written for them, nothing of them is accepted, and they stay as they were. Whole numbers and copied bytes, equal in every place."""
import sys

import numpy as np
import pytest

from oracle import decode as D
from oracle import tree as T
from test_gpu_tree import agree, draft, i32

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, file=sys.stderr, flush=True)


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("move", [True, False])
@pytest.mark.parametrize("sizes,longest", [([1], 1), ([1, 1], 4), ([25, 0, 25, 3], 25), ([64] * 9, 64), ([65, 200, 1, 130], 200), ([300, 2, 700], 700),
                                           ([9] * 70, 4), ([5, 5], 0)])
def test_accept_without_slots(hip, sizes, longest, move, apart):
    """Some sequences' tokens have the slot -1: no path, the length as it was, the root again as the next token, no moves."""
    import torch
    from qxotic_amd.jam import Tree, TreePath
    say("accept without slots", sizes[:4], longest, move, apart)
    r = np.random.default_rng(sum(sizes) + longest)
    n, off = len(sizes), np.cumsum([0] + sizes)
    total = int(off[-1]) + 2
    trees = [draft(r, k) for k in sizes]
    tokens, picked = agree(r, trees, share=0.9)
    tokens = [[t + 1000 * i for t in w] for i, w in enumerate(tokens)]   # a sequence's own
    picked = [[t + 1000 * i for t in w] for i, w in enumerate(picked)]
    slots = r.permutation(3 * total)[:total].astype(np.int32)
    gone = [i % 2 == 0 for i in range(n)]
    for i in range(n):
        if gone[i]:
            slots[off[i]:off[i + 1]] = -1
    lens = r.integers(0, 1000, n)
    flat = lambda a: [v for t in a for v in t] + [0] * 2   # noqa: E731
    d = dict(off=i32(off), parents=i32(flat(trees)), tokens=i32(flat(tokens)), picked=i32(flat(picked)), slots=i32(slots), lens=i32(lens),
             lens_out=i32([-9] * n), path=i32([-9] * (n * longest + 1)), accepted=i32([-9] * n), next=i32([-9] * n), src=i32([-9] * total),
             dst=i32([-9] * total))
    p = {k: t.data_ptr() for k, t in d.items()}
    torch.cuda.synchronize()
    path = TreePath(ld_path=longest, path=p["path"], accepted=p["accepted"], next=p["next"], lens=p["lens"],
                    lens_out=p["lens_out" if apart else "lens"], slots=p["slots"])
    if move:
        path.move_from, path.move_to = p["src"], p["dst"]
    tree = Tree(n_tokens=total, n_seqs=n, max_q=max(sizes), q_offsets=p["off"], parents=p["parents"])
    assert hip.tree_accept(tree, p["tokens"], p["picked"], path) == 0, hip.last_error()
    hip.synchronize()
    got = {k: t.cpu().numpy() for k, t in d.items()}
    src, dst = np.full(total, -9), np.full(total, -9)
    for i in range(n):
        a, b = off[i], off[i + 1]
        want, after = T.accept(trees[i], tokens[i], picked[i], slots[a:b], longest)
        assert not (gone[i] and want)
        assert got["path"][i * longest:(i + 1) * longest].tolist() == want + [-1] * (longest - len(want)), i
        assert got["accepted"][i] == len(want) and got["next"][i] == after, i
        assert got["lens_out" if apart else "lens"][i] == lens[i] + len(want), i
        if move:
            src[a:b] = dst[a:b] = -1
            for k, c in enumerate(want):
                if c != k:
                    src[a + k], dst[a + k] = slots[a + c], slots[a + k]
    assert np.array_equal(got["src"], src) and np.array_equal(got["dst"], dst)


@pytest.mark.parametrize("spare,cut,closing", [(1, 0, 0), (2, 0, 9), (3, 5, 30), (0, 14, 9), (64, 30, 60)])
def test_a_captured_step_that_runs_out(hip, spare, cut, closing):
    """A captured step with few pages, or rows for fewer tokens than are drafted, replayed and called eagerly in turn, one conversation ended on the
    way: what was refused keeps its length, its pages and its entries, whatever rows the closing resize has, and no page is held twice."""
    import torch
    from qxotic_amd.jam import HipJAM, KvCache, KvPages, Tree, TreePath
    say("a captured step that runs out", spare, cut, closing)
    jam = HipJAM()
    try:
        r = np.random.default_rng(8 + spare)
        n, nodes, page, ld, kv, dim = 5, 12, 16, 12, 2, 64
        rows = n * nodes - cut
        full = lambda *s: torch.full(s, -9, dtype=torch.int32, device="cuda")   # noqa: E731
        lens0 = r.integers(1, 60, n)
        held0 = -(-lens0 // page)
        pages = int(held0.sum()) + spare
        order = r.permutation(pages)
        table0, used = np.full((n, ld), -5, np.int32), 0
        for i, h in enumerate(held0):
            table0[i, :h] = order[used:used + h]
            used += h
        d = dict(lens=i32(lens0), held=i32(held0), n_free=i32([pages - used]), free=i32(np.concatenate([order[used:], np.full(used, -7)])),
                 table=i32(table0).view(n, ld), grow=i32([nodes] * n), targets=full(n), status=full(n), closed=full(n), off=full(n + 1), off2=full(n + 1),
                 pos=full(rows), slots=full(rows), pos2=full(closing + 1), slots2=full(closing + 1), parents=full(rows), tokens=full(rows),
                 picked=full(rows), path=full(n, nodes), accepted=full(n), next=full(n), before=full(n), after=full(n), src=full(rows), dst=full(rows),
                 masks=torch.zeros((rows, 1), dtype=torch.int64, device="cuda"))
        cache = [torch.randint(0, 256, (pages * page * kv * (dim + 4),), dtype=torch.uint8, device="cuda") for _ in range(2)]
        p = {k: t.data_ptr() for k, t in d.items()}
        c = KvCache(type=D.Q8_0, kv_heads=kv, head_dim=dim, page_tokens=page, n_pages=pages, k=cache[0].data_ptr(), v=cache[1].data_ptr())
        common = dict(n_seqs=n, page_tokens=page, n_pages=pages, free_cap=pages, ld_seq_pages=ld, held=p["held"], n_free=p["n_free"], free_pages=p["free"],
                      seq_pages=p["table"], lens_out=p["lens"], held_out=p["held"], n_free_out=p["n_free"])
        up = KvPages(n_tokens=rows, lens=p["before"], targets=p["targets"], status=p["status"], q_offsets=p["off"], pos=p["pos"], slots=p["slots"], **common)
        down = KvPages(n_tokens=closing, lens=p["lens"], targets=p["after"], status=p["closed"], q_offsets=p["off2"], pos=p["pos2"], slots=p["slots2"], **common)
        tree = Tree(n_tokens=rows, n_seqs=n, max_q=nodes, q_offsets=p["off"], parents=p["parents"])
        path = TreePath(ld_path=nodes, path=p["path"], accepted=p["accepted"], next=p["next"], lens=p["before"], lens_out=p["after"], slots=p["slots"],
                        move_from=p["src"], move_to=p["dst"])
        stream = torch.cuda.Stream()
        assert jam.set_stream(stream.cuda_stream) == 0

        def step():
            with torch.cuda.stream(stream):
                torch.minimum(d["lens"], d["lens"] + d["grow"], out=d["before"])   # an ended conversation's: 0
                d["before"].clamp_(min=0)
                torch.add(d["before"], d["grow"].clamp(min=0), out=d["targets"])
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
        refusals = 0
        for k in range(7):
            grow = [nodes] * n
            if k == 4:
                grow[1] = -(1 << 20)   # ends
            d["grow"].copy_(i32(grow))
            before = [max(min(v, v + g), 0) for v, g in zip(lens, grow)]
            targets = [v + max(g, 0) for v, g in zip(before, grow)]
            trees = [draft(r, t - v) for t, v in zip(targets, before)]
            tokens, picked = agree(r, trees, vocab=3, share=0.9)
            for name, v in (("parents", trees), ("tokens", tokens), ("picked", picked)):
                d[name].copy_(i32(([x for t in v for x in t] + [-1] * rows)[:rows]))
            was = [b.cpu().numpy() for b in cache]
            torch.cuda.synchronize()
            if k % 2:
                step()
            else:
                graph.replay()
            torch.cuda.synchronize()
            a, rest = T.resize(page, before, targets, [0] * n, held, free, table, rows)
            refusals += sum(a["status"])
            moves, after, nexts, counts = [], [], [], []
            for i in range(n):
                b0, b1 = a["q_offsets"][i], a["q_offsets"][i + 1]
                w, x = T.accept(trees[i][:b1 - b0], tokens[i][:b1 - b0], picked[i][:b1 - b0], a["slots"][b0:b1], nodes)
                assert not (a["status"][i] and w)
                moves.append([(a["slots"][b0 + v], a["slots"][b0 + q]) for q, v in enumerate(w) if v != q])
                after.append(before[i] + len(w))
                nexts.append(x)
                counts.append(len(w))
            b, free = T.resize(page, a["lens"], after, [0] * n, a["held"], rest, a["seq_pages"], closing)
            assert b["status"] == [0] * n
            got = {x: t.cpu().numpy() for x, t in d.items()}
            assert got["status"].tolist() == a["status"] and got["closed"].tolist() == b["status"]
            assert got["accepted"].tolist() == counts and got["next"].tolist() == nexts
            assert all(v == q for v, q, s in zip(b["lens"], before, a["status"]) if s)
            lens, held, table = b["lens"], b["held"], b["seq_pages"]
            assert got["lens"].tolist() == lens and got["held"].tolist() == held and got["table"].tolist() == table
            assert got["n_free"][0] == len(free) and got["free"][:len(free)].tolist() == free
            assert got["slots2"].tolist() == [-1] * closing + [-9] and got["pos2"].tolist() == [0] * closing + [-9]   # the closing call has no new tokens
            assert sorted(free + [row[q] for row, h in zip(table, held) for q in range(h)]) == list(range(pages))
            for buf, old in zip(cache, was):   # codes, then scales
                now, at = buf.cpu().numpy(), 0
                for row in (dim, dim // 16):
                    plane = old[at:at + pages * kv * page * row].reshape(pages, kv, page, row)
                    for g in moves:
                        for f, t in g:
                            plane[t // page, :, t % page] = plane[f // page, :, f % page]
                    at += plane.size
                assert np.array_equal(now, old)
        assert refusals > 3
    finally:
        jam.close()
