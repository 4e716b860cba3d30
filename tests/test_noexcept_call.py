"""CPU: what a call at the C boundary makes of an exception (csrc/noexcept_call.h, compiled without HIP): a status and a text that says what
happened, set in place of an earlier failure's without any memory."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
SHIM = """
#include <cstdio>
#include <cstdlib>
#include <stdexcept>
#include <string>
#include <vector>
#include "noexcept_call.h"
using namespace jamhip;
static bool none = false;   // no memory is to be had
void* operator new(size_t n) {
    void* p = none ? nullptr : malloc(n);
    if (!p) throw std::bad_alloc();
    return p;
}
void operator delete(void* p) noexcept { free(p); }
void operator delete(void* p, size_t) noexcept { free(p); }
static std::string err;
// kind: 0 a status of its own, 1 no memory for the message of a failure, 2 a list too long, 3 another exception
int main(int, char** arg) {
    const int kind = atoi(arg[1]), status = atoi(arg[2]);
    const char* before = arg[3];
    err = before;
    const int st = noexcept_call([&]() -> jamhip_status {
        none = kind > 0;
        if (kind == 1) err = std::string(before) + " and so much more that a string has to be made for it";
        if (kind == 2) { none = false; std::vector<int> v; v.resize(v.max_size()); }
        if (kind == 3) throw 7;
        return (jamhip_status) status;
    }, [](const char* text) { err = text; });
    none = false;
    printf("%d %s", st, err.c_str());
    return 0;
}
"""


@pytest.fixture(scope="module")
def call(tmp_path_factory):
    d = tmp_path_factory.mktemp("noexcept")
    (d / "t.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-Wno-mismatched-new-delete", f"-I{ROOT / 'qxotic_amd' / 'csrc'}", f"-I{ROOT / 'include'}", str(d / "t.cpp"),
                    "-o", str(d / "t")], check=True)

    def run(kind, status, before):
        out = subprocess.run([str(d / "t"), str(kind), str(status), before], check=True, capture_output=True, text=True).stdout
        status, text = out.split(" ", 1)
        return int(status), text

    return run


@pytest.mark.parametrize("before", ["", "x", "attn: window", "the failure of an earlier call, too long for a string's own characters"])
def test_exceptions(call, before):
    from qxotic_amd.jam import JAM
    for status in (JAM.OK, JAM.EUNSUPPORTED, JAM.EBUSY):
        assert call(0, status, before) == (status, before)
    assert call(1, JAM.OK, before) == (JAM.EINVAL, "out of memory")
    assert call(2, JAM.OK, before)[0] == JAM.EINVAL and call(2, JAM.OK, before)[1] in ("out of memory", "internal error")
    assert call(3, JAM.OK, before) == (JAM.EINVAL, "internal error")
