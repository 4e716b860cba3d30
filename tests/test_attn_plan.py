"""CPU: how an attention call is cut into workgroups (csrc/attn_plan.h) and the division it addresses pages with (csrc/fastdiv.h),
compiled without HIP."""
import ctypes
import random
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "qxotic_amd" / "csrc"
SHIM = """
#include "attn_plan.h"
#include "fastdiv.h"
using namespace jamhip;
extern "C" void q_attn(int dim, int kv, int grp, int tokens, int seqs, int prefixes, int max_q, int max_seq, int max_prefix, int* o) {
    const AttnPlan p = attn_plan(dim, kv, grp, tokens, seqs, prefixes, max_q, max_seq, max_prefix);
    o[0] = p.n, o[1] = p.slots;
    for (int i = 0; i < p.n; i++) {
        const AttnPart& a = p.part[i];
        int* q = o + 2 + 7 * i;
        q[0] = a.mode, q[1] = a.cfg, q[2] = a.tiles, q[3] = a.chunk, q[4] = a.splits, q[5] = a.slot0, q[6] = a.direct;
    }
}
extern "C" int q_rows(int cfg) { return attn_rows(cfg); }
extern "C" int q_keys(int cfg, int dim) { return attn_keys(cfg, dim); }
extern "C" int q_div(int d, int n) { return FastDiv(d).div(n); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("attn_plan")
    (d / "p.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", str(d / "p.cpp"), "-o", str(d / "p.so")],
                   check=True)
    return ctypes.CDLL(str(d / "p.so"))


def plan(lib, *args):
    o = (ctypes.c_int * 16)()
    lib.q_attn(*args, o)
    keys = ("mode", "cfg", "tiles", "chunk", "splits", "slot0", "direct")
    return o[1], [dict(zip(keys, o[2 + 7 * i:9 + 7 * i])) for i in range(o[0])]


def check(lib, dim, kv, grp, lens, groups, max_seq):
    """lens: query tokens of each sequence; groups: (first, last + 1, prefix length)."""
    tokens, max_q = sum(lens), max(lens)
    slots, parts = plan(lib, dim, kv, grp, tokens, len(lens), len(groups), max_q, max_seq, max((g[2] for g in groups), default=0))
    assert 1 <= len(parts) <= 2 and [p["mode"] for p in parts] in ([0], [1, 2])
    used = 0
    for p in parts:
        rows, keys = lib.q_rows(p["cfg"]), lib.q_keys(p["cfg"], dim)
        longest = {0: max_seq + max((g[2] for g in groups), default=0), 1: max((g[2] for g in groups), default=0), 2: max_seq}[p["mode"]]
        assert p["chunk"] % keys == 0 and p["chunk"] > 0 and p["splits"] >= 1
        assert p["chunk"] * p["splits"] >= longest                         # every key is in a run
        assert p["splits"] == 1 or p["chunk"] * (p["splits"] - 1) < longest   # and no run is past the last
        if p["mode"] == 1:
            need = sum(-(-sum(lens[a:b]) * grp // rows) for a, b, _ in groups)
            assert need <= p["tiles"] <= sum(lens) * grp // rows + len(groups)   # tokens outside the groups are not told apart
        else:
            assert p["tiles"] == len(lens) * -(-max_q * grp // rows)
        assert p["cfg"] != 1 or dim <= 192
        if p["direct"]:
            assert len(parts) == 1 and slots == 0 and p["splits"] == 1
        else:
            assert p["slot0"] == used
            used += p["splits"]
    assert used == slots
    return parts


def test_every_row_and_key_is_covered(lib):
    r = random.Random(1)
    seen = set()
    for _ in range(4000):
        seqs = r.choice([1, 2, 7, 64, 200])
        lens = [r.choice([0, 1, 1, 1, 3, 40, 300]) if r.random() < 0.5 else 1 for _ in range(seqs)]
        lens[0] = max(lens[0], 1)
        n = r.choice([0, 1, 1, min(4, seqs)])
        cuts = sorted(r.randint(0, seqs) for _ in range(n + 1))
        groups = [(a, b, r.choice([0, 1, 129, 5000, 100000])) for a, b in zip(cuts, cuts[1:])]
        for p in check(lib, r.choice([64, 96, 128, 192, 256]), r.choice([1, 2, 8]), r.choice([1, 4, 7, 16, 20]), lens, groups,
                       r.choice([1, 127, 128, 129, 4000, 1 << 20])):
            seen.add((p["mode"], p["cfg"], p["splits"] > 1))
    assert {(m, c) for m, c, _ in seen} == {(m, c) for m in (0, 1, 2) for c in (0, 1, 2)} and (0, 2, True) in seen


def test_choices(lib):
    """A decode step behind a long prefix reads it once for all; one sequence, prompts that fill their tiles and prefixes of a page or two
    are taken sequence by sequence."""
    modes = lambda *a: [(p["mode"], p["cfg"]) for p in plan(lib, *a)[1]]   # noqa: E731
    assert modes(128, 8, 4, 64, 64, 1, 1, 1024, 8192) == [(1, 2), (2, 0)]
    assert modes(128, 8, 4, 32, 32, 4, 1, 300, 24001) == [(1, 1), (2, 0)]
    assert modes(128, 8, 4, 16, 16, 1, 1, 200, 4000) == [(1, 1), (2, 0)] and modes(128, 8, 4, 16, 16, 1, 1, 200, 1500) == [(0, 0)]
    assert modes(128, 8, 4, 512, 64, 1, 8, 100, 16000) == [(1, 2), (2, 1)] and modes(128, 8, 4, 512, 64, 1, 8, 100, 2000) == [(0, 1)]
    assert modes(128, 8, 4, 1, 1, 1, 1, 45, 700) == [(0, 0)]
    assert modes(64, 8, 8, 1792, 8, 1, 256, 256, 4096) == [(0, 2)]
    assert modes(128, 8, 4, 64, 64, 1, 1, 1024, 100) == [(0, 0)]


def test_workgroups_past_32_bits(lib):
    """A call whose workgroups pass 2^31 has no plan; one below keeps every tile. The header's bound is on the safe side."""
    tiles = lambda *a: [p["tiles"] * p["splits"] for p in plan(lib, *a)[1]]   # noqa: E731
    assert tiles(128, 8, 8, 34815, 2048, 0, 32768, 32768, 0) == [2048 * 2048]           # 33.5 million workgroups
    assert tiles(64, 8, 1, 1 << 20, 16383, 0, 1 << 20, 99, 0) == [16383 * 8192]
    for seqs in (1 << 15, 1 << 16, 1 << 19, 1 << 20, (1 << 20) + 1):                    # cut to 32 bits: negative, 0, 0, 0, 8192
        assert plan(lib, 64, 8, 1, 1 << 20, seqs, 0, 1 << 20, 99, 0) == (0, [])
    r = random.Random(3)
    some = 0
    for _ in range(4000):
        dim, kv, grp = r.choice([64, 96, 128, 192, 256]), r.choice([1, 2, 8]), r.choice([1, 4, 7, 16, 20])
        most = ((1 << 31) - 4097) // (kv * grp)
        tokens, seqs = int(most ** r.random()), int(2 ** (24 * r.random()))
        max_q, n = int(tokens ** r.random()), r.choice([0, 1, seqs // 5])
        _, parts = plan(lib, dim, kv, grp, tokens, seqs, n, max_q, r.choice([1, 129, 1 << 20]), r.choice([1, 5000, 100000]) if n else 0)
        for p in parts:
            rows = lib.q_rows(p["cfg"])
            assert p["tiles"] == (tokens * grp // rows + n if p["mode"] == 1 else seqs * -(-max_q * grp // rows))
            assert p["tiles"] * p["splits"] * kv < 1 << 31
        if seqs * (max_q * kv * grp // 128 + kv) < 1 << 30:
            assert parts
        some += not parts
    assert some > 100


def test_fast_division(lib):
    r = random.Random(2)
    for d in [1, 2, 3, 5, 7, 16, 24, 100, 1000, 65535, 65536, 65537, (1 << 30) + 1, (1 << 31) - 1] + [r.randint(1, (1 << 31) - 1) for _ in range(50)]:
        for n in [0, 1, d - 1, d, min(d + 1, (1 << 31) - 1), (1 << 31) - 1, (1 << 31) - 2] + [r.randint(0, (1 << 31) - 1) for _ in range(50)]:
            assert lib.q_div(d, n) == n // d, (d, n)


def test_cache_bytes():
    from qxotic_amd.jam import JAM, HipJAM, KvCache
    shape = dict(kv_heads=2, head_dim=64, page_tokens=16, n_pages=3)
    for kind, row in ((JAM.F16, 128), (JAM.Q8_0, 68), (JAM.Q4_0, 36)):
        assert HipJAM.kv_cache_bytes(KvCache(type=kind, **shape)) == 3 * 16 * 2 * row
    assert HipJAM.kv_cache_bytes(KvCache(type=JAM.Q4_K, **shape)) == -1
    assert HipJAM.kv_cache_bytes(KvCache(type=JAM.Q8_0, **{**shape, "head_dim": 48})) == -1
    assert HipJAM.kv_cache_bytes(KvCache(type=JAM.F16, **{**shape, "head_dim": 48})) == 3 * 16 * 2 * 96
    assert HipJAM.kv_cache_bytes(KvCache(type=JAM.F16, **{**shape, "page_tokens": 0})) == -1
    assert HipJAM.kv_cache_bytes(None) == -1
