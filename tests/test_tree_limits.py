"""CPU: sizes at which the calls around drafted trees would leave 32 bits, and those that they take (csrc/treeargs.h, compiled without HIP)."""
import ctypes
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
SHIM = """
#include "treeargs.h"
using namespace jamhip;
extern "C" int q_path(const jamhip_tree* t, const void* a, const void* b, const jamhip_tree_path* p) { return refuse_path(t, a, b, p).status; }
extern "C" int q_move(const jamhip_kv_cache* c, int n, const void* o, int g, const void* f, const void* t, int e) { return refuse_move(c, n, o, g, f, t, e).status; }
"""
OK, U, P = 0, 2, 1 << 20


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("limits")
    (d / "t.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{ROOT / 'qxotic_amd' / 'csrc'}", f"-I{ROOT / 'include'}",
                    str(d / "t.cpp"), "-o", str(d / "t.so")], check=True)
    return ctypes.CDLL(str(d / "t.so"))


def test_longest_path(lib):
    """A path is written 64 places at a time: their numbers stay below 2^31."""
    from qxotic_amd.jam import Tree, TreePath
    tree = Tree(n_tokens=3, n_seqs=2, max_q=2, q_offsets=P, parents=P)

    def call(longest):
        p = TreePath(ld_path=longest, path=P, accepted=P, next=P)
        return lib.q_path(ctypes.byref(tree), ctypes.c_void_p(P), ctypes.c_void_p(P), ctypes.byref(p))

    most = (1 << 31) - 1 - 4096
    assert call(1) == call(most) == OK and call(most + 1) == call((1 << 31) - 64) == call((1 << 31) - 1) == U


def test_many_groups_of_many_caches(lib):
    """Any number of caches goes with the largest number of groups: they are launched some at a time."""
    from qxotic_amd.jam import KvCache
    shape = dict(type=8, kv_heads=2, head_dim=64, page_tokens=16, n_pages=4, k=P, v=P)
    caches = (KvCache * 2049)(*(KvCache(**shape) for _ in range(2049)))
    a = ctypes.c_void_p(P)
    assert lib.q_move(caches, 2049, a, 1 << 20, a, a, 1) == OK and lib.q_move(caches, 2049, a, (1 << 20) + 1, a, a, 1) == U
