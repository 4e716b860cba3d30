"""CPU: which keys a drafted token sees (csrc/treemask.h) against the list of them, what the calls around drafted trees refuse
(csrc/treeargs.h), both compiled without HIP, and the layout of the structs of the binding."""
import ctypes
import random
import subprocess
from pathlib import Path

import numpy as np
import pytest

from oracle import tree as T

ROOT = Path(__file__).resolve().parent.parent
SHIM = """
#include "treemask.h"
#include "treeargs.h"
#include "attn_plan.h"
using namespace jamhip;
extern "C" void q_plan(int dim, int kv, int grp, int tokens, int seqs, int prefixes, int max_q, int max_seq, int max_prefix, int tree, int* o) {
    const AttnPlan p = attn_plan(dim, kv, grp, tokens, seqs, prefixes, max_q, max_seq, max_prefix, tree);
    o[0] = p.n, o[1] = p.slots;
    for (int i = 0; i < p.n; i++) {
        const AttnPart& a = p.part[i];
        int* q = o + 2 + 7 * i;
        q[0] = a.mode, q[1] = a.cfg, q[2] = a.tiles, q[3] = a.chunk, q[4] = a.splits, q[5] = a.slot0, q[6] = a.direct;
    }
}
extern "C" int q_rows(int cfg) { return attn_rows(cfg); }
extern "C" int q_keys(int cfg, int dim) { return attn_keys(cfg, dim); }
// o: the range that holds its keys; sees[n], tiles[n]: 64 bits from key i on
extern "C" void q_span(const uint64_t* row, int words, int base, int first, int nq, int window, int skip, int c0, int c1, int n, int* o, int* sees, uint64_t* tiles) {
    const TreeMask m{row, words};
    const TreeSpan s = span_cut(tree_span(m, base, first, nq, window), skip, c0, c1);
    o[0] = span_lo(s), o[1] = span_hi(s);
    for (int i = 0; i < n; i++) sees[i] = span_sees(m, s, i), tiles[i] = span_tile(m, s, i);
}
extern "C" int q_pages(const jamhip_kv_pages* p) { return refuse_pages(p).status; }
extern "C" int q_tree(const jamhip_tree* p) { return refuse_tree(p).status; }
extern "C" int q_masks(const void* m, int words, int max_q) { return refuse_masks(m, words, max_q).status; }
extern "C" int q_path(const jamhip_tree* t, const void* a, const void* b, const jamhip_tree_path* p) { return refuse_path(t, a, b, p).status; }
extern "C" int q_move(const jamhip_kv_cache* c, int n, const void* o, int g, const void* f, const void* t, int e) { return refuse_move(c, n, o, g, f, t, e).status; }
extern "C" int q_size(int i) {
    return i == 0 ? sizeof(jamhip_kv_pages) : i == 1 ? sizeof(jamhip_tree) : i == 2 ? sizeof(jamhip_tree_path) : sizeof(jamhip_kv_cache);
}
"""
OK, E, U, P = 0, 1, 2, 1 << 20


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("tree")
    (d / "t.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{ROOT / 'qxotic_amd' / 'csrc'}", f"-I{ROOT / 'include'}",
                    str(d / "t.cpp"), "-o", str(d / "t.so")], check=True)
    return ctypes.CDLL(str(d / "t.so"))


def test_seen_keys(lib):
    """Ranges, single keys and tiles of 64 against the list of keys; words beside the row are never looked at (they are noise here)."""
    r = random.Random(1)
    for trial in range(3000):
        n_words = r.choice([1, 1, 1, 2, 3])
        base, own = r.choice([0, 0, 5, 70]), r.choice([0, 1, 3, 40, 64, 90, 130])
        nq = r.choice([0, 1, 2, 7, 63, 64, 65, 64 * n_words, 64 * n_words + 9])
        first, window = own - nq, r.choice([0, 0, 0, 1, 2, 5, 64, 100])
        bits = {j for j in range(64 * n_words) if r.random() < r.choice([0.0, 0.1, 0.5, 1.0])}
        row = T.words([bits], n_words)[0]
        noise = np.random.default_rng(trial).integers(0, 1 << 63, n_words + 4, dtype=np.int64).view(np.uint64)
        noise[2:-2] = row
        ctx = base + max(first, 0)
        # drafted token j is the sequence's own first + j: those in front of the own ones have no entry
        have = {j for j in bits if j < min(nq, 64 * n_words) and first + j >= 0}
        want = list(range(ctx)) + [base + first + j for j in sorted(have)]
        want = set(want[-window:] if window else want)
        skip = r.choice([0, 0, base])
        total = base + own - skip
        c0 = r.randint(0, max(0, total)) if r.random() < 0.6 else 0
        c1 = r.randint(c0, max(c0, total)) if r.random() < 0.6 else total
        want = {k - skip for k in want if c0 <= k - skip < c1}
        n = max(total, 1)
        o, sees, tiles = (ctypes.c_int * 2)(), (ctypes.c_int * n)(), (ctypes.c_uint64 * n)()
        lib.q_span(ctypes.c_void_p(noise.ctypes.data + 16), n_words, base, first, nq, window, skip, c0, c1, n, o, sees, tiles)
        assert {i for i in range(n) if sees[i]} == want
        for i in range(n):
            assert tiles[i] == sum(1 << (k - i) for k in want if i <= k < i + 64), (trial, i)
        if want:
            assert o[0] <= min(want) and o[1] > max(want)
        if o[0] < o[1]:
            assert c0 <= o[0] and o[1] <= c1


def plan(lib, *args):
    o = (ctypes.c_int * 16)()
    lib.q_plan(*args, o)
    keys = ("mode", "cfg", "tiles", "chunk", "splits", "slot0", "direct")
    return o[1], [dict(zip(keys, o[2 + 7 * i:9 + 7 * i])) for i in range(o[0])]


def test_tree_plans(lib):
    """How calls of drafted trees are cut: every row and key is in one workgroup's run, by whichever rule; and what the rules choose."""
    r = random.Random(7)
    seen = set()
    for _ in range(3000):
        dim, kv, grp = r.choice([64, 96, 128, 192, 256]), r.choice([1, 2, 8]), r.choice([1, 4, 8, 16])
        seqs, q = r.choice([1, 4, 64, 200]), r.choice([1, 4, 25, 64, 300])
        n = r.choice([0, 0, 1, min(4, seqs)])
        max_seq, prefix = r.choice([1, 128, 129, 745, 4000, 1 << 20]), r.choice([1, 129, 9000]) if n else 0
        slots, parts = plan(lib, dim, kv, grp, seqs * q, seqs, n, q, max_seq, prefix, 1)
        assert [p["mode"] for p in parts] in ([0], [1, 2])
        used = 0
        for p in parts:
            rows, keys = lib.q_rows(p["cfg"]), lib.q_keys(p["cfg"], dim)
            longest = {0: max_seq + prefix, 1: prefix, 2: max_seq}[p["mode"]]
            assert p["chunk"] % keys == 0 and p["chunk"] * p["splits"] >= longest and (p["splits"] == 1 or p["chunk"] * (p["splits"] - 1) < longest)
            assert p["tiles"] >= (seqs * q * grp // rows if p["mode"] == 1 else seqs * -(-q * grp // rows)) and (p["cfg"] != 1 or dim <= 192)
            if p["direct"]:
                assert len(parts) == 1 and slots == 0 and p["splits"] == 1
            else:
                assert p["slot0"] == used
                used += p["splits"]
            seen.add((p["mode"], p["cfg"], p["direct"]))
        assert used == slots
    assert {(0, c, d) for c in (0, 1, 2) for d in (0, 1)} <= seen and {(m, 2, 0) for m in (1, 2)} & seen
    cut = lambda *a: [(p["cfg"], p["splits"]) for p in plan(lib, *a)[1]]   # noqa: E731
    assert cut(128, 8, 4, 25, 1, 0, 25, 745, 0, 1) == [(1, 6)] and cut(128, 8, 4, 25, 1, 0, 25, 745, 0, 0) == [(2, 6)]
    assert cut(128, 8, 4, 25, 1, 0, 25, 512, 0, 1) == [(1, 1)] and cut(256, 8, 4, 25, 1, 0, 25, 745, 0, 1) == [(2, 12)]
    assert cut(128, 8, 4, 256, 8, 0, 32, 2000, 0, 1) == [(2, 4)] and cut(128, 8, 4, 256, 8, 0, 32, 8000, 0, 1) == [(2, 8)]
    assert cut(128, 8, 4, 2048, 64, 0, 32, 4096, 0, 1) == [(2, 1)] and cut(128, 8, 4, 1, 1, 0, 1, 400, 0, 1) == [(0, 1)]


def test_binding_sizes(lib):
    from qxotic_amd.jam import KvCache, KvPages, Tree, TreePath
    assert [ctypes.sizeof(t) for t in (KvPages, Tree, TreePath, KvCache)] == [lib.q_size(i) for i in range(4)]


def test_refused_pages(lib):
    from qxotic_amd.jam import KvPages
    arrays = ("lens", "targets", "base", "held", "n_free", "free_pages", "seq_pages", "lens_out", "held_out", "n_free_out", "status", "q_offsets",
              "pos", "slots")
    good = dict(n_seqs=2, n_tokens=3, page_tokens=16, n_pages=9, free_cap=9, ld_seq_pages=4, **{k: P for k in arrays})
    call = lambda **kw: lib.q_pages(ctypes.byref(KvPages(**{**good, **kw})))   # noqa: E731
    assert lib.q_pages(None) == E and call() == OK and call(base=None) == OK and call(n_tokens=0, pos=None, slots=None) == OK
    assert call(n_seqs=0, **{k: None for k in ("lens", "targets", "held", "lens_out", "held_out", "status", "seq_pages")}) == OK
    for k in arrays:
        assert k == "base" or call(**{k: None}) == E, k
    for k in ("n_seqs", "n_tokens", "page_tokens", "n_pages", "free_cap", "ld_seq_pages"):
        assert call(**{k: -1}) == E, k
    assert call(page_tokens=0) == E and call(n_seqs=(1 << 20) + 1) == U and call(n_pages=1 << 28) == U and call(n_tokens=(1 << 31) - 1) == U


def test_refused_trees(lib):
    from qxotic_amd.jam import KvCache, Tree, TreePath
    tree = lambda **kw: Tree(**{**dict(n_tokens=3, n_seqs=2, max_q=2, q_offsets=P, parents=P), **kw})   # noqa: E731
    call = lambda **kw: lib.q_tree(ctypes.byref(tree(**kw)))   # noqa: E731
    assert lib.q_tree(None) == E and call() == OK and call(q_offsets=None) == E and call(parents=None) == E
    assert call(n_tokens=0, q_offsets=None, parents=None) == OK
    for k in ("n_tokens", "n_seqs", "max_q"):
        assert call(**{k: -1}) == E, k
    assert call(n_seqs=(1 << 20) + 1) == U and call(n_tokens=(1 << 31) - 1) == U
    masks = lambda p, words, q: lib.q_masks(ctypes.c_void_p(p), words, q)   # noqa: E731
    assert masks(P, 1, 64) == OK and masks(P, 2, 65) == OK
    assert masks(None, 1, 1) == E and masks(P + 4, 1, 1) == E and masks(P, 0, 0) == E and masks(P, 1, 65) == E and masks(P, -1, 1) == E
    assert masks(P, 1 << 28, 1) == U
    good = dict(ld_path=4, path=P, accepted=P, next=P, lens=P, lens_out=P, slots=P, move_from=P, move_to=P)
    a, b = ctypes.c_void_p(P), ctypes.c_void_p(P)
    path = lambda a=a, b=b, **kw: lib.q_path(ctypes.byref(tree()), a, b, ctypes.byref(TreePath(**{**good, **kw})))   # noqa: E731
    assert path() == OK and lib.q_path(ctypes.byref(tree()), a, b, None) == E and path(a=None) == E and path(b=None) == E
    for k in ("path", "accepted", "next", "lens", "slots", "move_from", "move_to"):
        assert path(**{k: None}) == E, k
    assert path(ld_path=-1) == E and path(ld_path=0, path=None) == OK
    assert path(lens=None, lens_out=None) == OK and path(move_from=None, move_to=None, slots=None) == OK
    shape = dict(type=8, kv_heads=2, head_dim=64, page_tokens=16, n_pages=4, k=P, v=P)
    caches = lambda *kw: (KvCache * len(kw))(*(KvCache(**{**shape, **k}) for k in kw))   # noqa: E731
    move = lambda c, n, o=a, g=1, f=a, t=a, e=1: lib.q_move(c, n, o, g, f, t, e)   # noqa: E731
    two = caches({}, {"k": 2 * P})
    assert move(two, 2) == OK and move(None, 1) == E and move(two, -1) == E and move(two, 2, g=-1) == E and move(two, 2, e=-1) == E
    assert move(two, 2, o=None) == E and move(two, 2, f=None) == E and move(two, 2, t=None) == E and move(two, 2, o=None, f=None, t=None, e=0) == OK
    for k, v in dict(type=1, kv_heads=1, head_dim=96, page_tokens=8, n_pages=5).items():
        assert move(caches({}, {k: v}), 2) == E, k
    assert move(two, 2, g=(1 << 20) + 1) == U and move(two, 2, e=(1 << 31) - 1) == U


def test_oracle_resize_restores_its_list():
    """The definition itself: what one call takes the next gives back, and the list is as it was."""
    free, table = list(range(20, 9, -1)), [[1, 2, -1, -1], [3, -1, -1, -1], [-1] * 4]
    lens, held = [20, 5, 0], [2, 1, 0]
    up, rest = T.resize(16, lens, [40, 33, 17], [0, 0, 0], held, free, table, 100)
    assert up["status"] == [0, 0, 0] and up["held"] == [3, 3, 2] and len(rest) == len(free) - 5
    down, back = T.resize(16, up["lens"], lens, [0, 0, 0], up["held"], rest, up["seq_pages"], 100)
    assert back == free and down["held"] == held and down["lens"] == lens and down["q_offsets"] == [0, 0, 0, 0]
