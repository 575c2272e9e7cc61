"""Which rows of a run the convolution may store (csrc/row_mask.hpp, plain C++): none behind the run, whatever the offsets are."""
import ctypes
import os
import random
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include "row_mask.hpp"
using namespace uniql;
static int clamped(int v, int low, int high) { return v < low ? low : (v > high ? high : v); }
// the rows of the run from row0 on that lie in any of the sequences, `lead` rows behind their first one, as the kernel puts them together
extern "C" uint32_t allowed_rows(const int* cu, int count, int total, int row0, int run, int lead) {
    const int rows = total - row0 < run ? total - row0 : run;
    uint32_t allowed = 0;
    for (int s = 0; s < count; ++s) {
        const int first = clamped(cu[s], 0, total), last = clamped(cu[s + 1], first, total);
        allowed = rows_of_either(allowed, rows_between(first + lead - row0, last - row0, rows));
    }
    return allowed;
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    d = tmp_path_factory.mktemp("row_mask")
    (d / "mask.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-shared", "-fPIC", f"-I{os.path.join(ROOT, 'uniql_amd', 'csrc')}", str(d / "mask.cpp"),
                    "-o", str(d / "mask.so")], check=True)
    lib = ctypes.CDLL(str(d / "mask.so"))
    lib.allowed_rows.restype = ctypes.c_uint32
    return lib


def check(lib, cu, total, run, lead):
    array = (ctypes.c_int * len(cu))(*cu)
    clamp = lambda v: max(0, min(v, total))
    for row0 in range(0, total, run):
        want = 0
        for a, b in zip(cu, cu[1:]):
            for row in range(clamp(a) + lead, clamp(b)):
                if row0 <= row < min(row0 + run, total):
                    want |= 1 << (row - row0)
        assert lib.allowed_rows(array, len(cu) - 1, total, row0, run, lead) == want, (cu, total, run, row0)


@pytest.mark.parametrize("lead", [1, 2, 3])
def test_offsets_that_fall_and_rise_again(lib, lead):
    check(lib, [0, 5, 0, 5, 0, 5], 5, 8, lead)
    check(lib, [0, 32, 0, 32], 32, 32, lead)
    check(lib, [-7, 100, -(1 << 31), (1 << 31) - 1, 3, 9], 40, 16, lead)


@pytest.mark.parametrize("run", [8, 16, 32])
def test_any_offsets(lib, run):
    rng = random.Random(run)
    for _ in range(300):
        total = rng.randint(1, 100)
        cu = [rng.randint(-3, total + 3) for _ in range(rng.randint(1, 12))]
        check(lib, cu, total, run, rng.randint(1, 3))
        check(lib, sorted(cu), total, run, rng.randint(1, 3))
