"""CPU: the sorts of the sampling kernel's second launch (csrc/sample_sort.h), run by 256 fibers that stand for a workgroup's threads. Between
two barriers one runs after another, in rising, falling or random order: what holds in every such order needs no thread, and no
wave, to be as far as another."""
import ctypes
import random
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "qxotic_amd" / "csrc"
SHIM = """
#include <ucontext.h>
#include <stdlib.h>
#define JAMHIP_DEV inline
static struct { unsigned x; } threadIdx;
static void __syncthreads();
#include "sample_sort.h"

constexpr int N = jamhip::SM_THREADS, STACK = 1 << 16;
static ucontext_t home, fiber[N];
static char stacks[N][STACK];
static bool ended[N];
static void (*work)();
static void __syncthreads() { const unsigned me = threadIdx.x; swapcontext(&fiber[me], &home); threadIdx.x = me; }
static void body() { work(); ended[threadIdx.x] = true; }

// Every thread up to its next barrier, then again; -1: threads differ in their number of barriers.
static int run(void (*f)(), int order, unsigned seed) {
    srand(seed);
    work = f;
    int place[N];
    for (int i = 0; i < N; i++) {
        getcontext(&fiber[i]);
        fiber[i].uc_stack.ss_sp = stacks[i], fiber[i].uc_stack.ss_size = STACK, fiber[i].uc_link = &home;
        makecontext(&fiber[i], body, 0);
        ended[i] = false, place[i] = order == 1 ? N - 1 - i : i;
    }
    for (;;) {
        if (order == 2)
            for (int i = N - 1; i > 0; i--) {
                const int j = rand() % (i + 1), t = place[i];
                place[i] = place[j], place[j] = t;
            }
        for (int i = 0; i < N; i++) threadIdx.x = place[i], swapcontext(&home, &fiber[place[i]]);
        int n = 0;
        for (int i = 0; i < N; i++) n += ended[i];
        if (n == N) return 0;
        if (n) return -1;
    }
}

static unsigned long long list[4096];
static int count, kept;
static void sort_only() { jamhip::sort_falling(list, count); }
static void sort_and_order() { jamhip::sort_falling(list, count); jamhip::order_by_index(list, kept); }

extern "C" int sort(unsigned long long* a, int n, int m, int order, unsigned seed) {
    for (int i = 0; i < n; i++) list[i] = a[i];
    count = n, kept = m;
    const int r = run(m ? sort_and_order : sort_only, order, seed);
    for (int i = 0; i < (m ? m : n); i++) a[i] = list[i];
    return r;
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("sample_sort")
    (d / "s.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wno-unknown-pragmas", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", str(d / "s.cpp"),
                    "-o", str(d / "s.so")], check=True)
    return ctypes.CDLL(str(d / "s.so"))


def pairs(r, n):
    """Keys, many of them equal, over distinct indices, as the kernel packs them."""
    at = r.sample(range(262144), n)
    return [(r.choice([0xC0000000, 0xC0010000, r.getrandbits(32)]) << 32) | (0xFFFFFFFF ^ i) for i in at]


@pytest.mark.parametrize("order", [0, 1, 2])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 128, 200, 255, 256, 257, 511, 512, 513, 1000, 4095, 4096])
def test_sort(lib, n, order):
    r = random.Random(n)
    v = pairs(r, n)
    a = (ctypes.c_uint64 * n)(*v)
    assert lib.sort(a, n, 0, order, n) == 0
    assert list(a) == sorted(v, reverse=True)


@pytest.mark.parametrize("order", [0, 1, 2])
@pytest.mark.parametrize("n,m", [(1, 1), (64, 64), (80, 65), (65, 64), (200, 128), (200, 199), (256, 256), (300, 70), (300, 257), (2000, 255),
                                 (2000, 1000), (4096, 4096)])
def test_order_by_index(lib, n, m, order):
    """The kept ones in the vocabulary's order, each with its place in the sorted list (where its weight is)."""
    r = random.Random(n + m)
    v = pairs(r, n)
    a = (ctypes.c_uint64 * n)(*v)
    assert lib.sort(a, n, m, order, n) == 0
    top = [0xFFFFFFFF ^ (p & 0xFFFFFFFF) for p in sorted(v, reverse=True)[:m]]
    assert [(0xFFFFFFFF ^ (p >> 32), p & 0xFFFFFFFF) for p in list(a)[:m]] == sorted((i, e) for e, i in enumerate(top))
