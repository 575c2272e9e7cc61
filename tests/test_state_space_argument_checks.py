"""The C entry points between the projections of a state-space layer refuse what they cannot do before anything is launched, and what
they launch is what they asked scratch memory for (no GPU needed)."""
import ctypes
import os
import shutil
import subprocess
import sys

import pytest

from uniql_amd import _capi
from uniql_amd.build import LIB_PATH

HERE = os.path.dirname(os.path.abspath(__file__))
FAKE = 0x10000


class Sequences(ctypes.Structure):
    _fields_ = [("cu", ctypes.c_void_p), ("starts", ctypes.c_void_p), ("places", ctypes.c_void_p), ("count", ctypes.c_int), ("pool", ctypes.c_int)]


@pytest.fixture(scope="module")
def lib():
    return _capi.load()


def sequences(**kw):
    return ctypes.byref(Sequences(**{**dict(cu=FAKE, starts=None, places=None, count=2, pool=4), **kw}))


BAD_SEQUENCES = [(dict(count=-1), -2), (dict(count=(1 << 24) + 1), -2), (dict(pool=-1), -2), (dict(cu=None, count=3), -2)]


def conv(lib, **kw):
    args = dict(x=FAKE, x_row=64, weight=FAKE, bias=None, state=FAKE, state_out=FAKE, sequences=sequences(), out=FAKE, out_row=64, rows=0,
                channels=64, width=4, activation=1, stream=None)
    return lib.uniql_causal_conv(*{**args, **kw}.values())


def scan(lib, **kw):
    args = dict(x=FAKE, x_row=64, x_head=16, dt=FAKE, dt_row=4, decay=FAKE, b=FAKE, b_row=32, b_group=16, c=FAKE, c_row=32, c_group=16, skip=None,
                dt_bias=None, softplus=1, dt_min=0.0, dt_max=float("inf"), state=FAKE, state_out=FAKE, sequences=sequences(), y=FAKE, y_row=64,
                y_head=16, temp=None, temp_bytes=0, rows=0, heads=4, groups=2, head_dim=16, states=16, stream=None)
    return lib.uniql_state_space_scan(*{**args, **kw}.values())


def norm(lib, **kw):
    args = dict(x=FAKE, x_row=64, z=FAKE, z_row=64, weight=FAKE, out=FAKE, out_row=64, rows=0, channels=64, groups=2, eps=1e-5, stream=None)
    return lib.uniql_gated_group_norm(*{**args, **kw}.values())


def test_nothing_to_do(lib):
    assert conv(lib) == 0 and scan(lib) == 0 and norm(lib) == 0
    assert conv(lib, rows=5, sequences=sequences(count=0)) == 0 and scan(lib, rows=5, sequences=sequences(count=0)) == 0


@pytest.mark.parametrize("kw,code", BAD_SEQUENCES)
def test_sequences(lib, kw, code):
    assert conv(lib, sequences=sequences(**kw)) == code
    assert scan(lib, sequences=sequences(**kw)) == code
    assert conv(lib, sequences=None) == -1 and scan(lib, sequences=None) == -1


def test_conv(lib):
    for kw, code in [(dict(rows=-1), -2), (dict(rows=(1 << 27) + 1), -2), (dict(channels=0), -2), (dict(channels=(1 << 24) + 1), -2),
                     (dict(width=1), -5), (dict(width=5), -5), (dict(rows=3, x=None), -1), (dict(rows=3, weight=None), -1),
                     (dict(rows=3, out=None), -1)]:
        assert conv(lib, **kw) == code, kw


def test_scan(lib):
    for kw, code in [(dict(rows=-1), -2), (dict(rows=(1 << 27) + 1), -2), (dict(heads=0), -2), (dict(heads=(1 << 15) + 1, groups=1), -2),
                     (dict(groups=3), -2), (dict(groups=0), -2), (dict(head_dim=0), -2), (dict(states=0), -2), (dict(head_dim=129), -5),
                     (dict(states=257), -5), (dict(dt_min=1.0, dt_max=0.5), -5), (dict(dt_min=-0.5, dt_max=0.5), -5), (dict(dt_min=float("nan")), -5), (dict(rows=3, x=None), -1),
                     (dict(rows=3, dt=None), -1), (dict(rows=3, decay=None), -1), (dict(rows=3, b=None), -1), (dict(rows=3, c=None), -1),
                     (dict(rows=3, y=None), -1), (dict(rows=3, state=FAKE + 4), -3), (dict(rows=3, state_out=FAKE + 8), -3),
                     (dict(rows=4096, temp_bytes=16), -4), (dict(rows=4096, temp_bytes=1 << 40), -1),
                     (dict(rows=4096, temp=FAKE + 4, temp_bytes=1 << 40), -3)]:
        assert scan(lib, **kw) == code, kw


def test_scan_workspace(lib):
    need = ctypes.c_size_t(7)
    ask = lib.uniql_state_space_scan_workspace
    assert ask(4096, 2, 4, 2, 16, 16, None) == -1
    assert ask(4096, 2, 4, 3, 16, 16, ctypes.byref(need)) == -2
    assert ask(4096, 2, 4, 2, 16, 300, ctypes.byref(need)) == -5
    assert ask(0, 2, 4, 2, 16, 16, ctypes.byref(need)) == 0 and need.value == 0
    assert ask(4096, 2, 4, 2, 16, 16, ctypes.byref(need)) == 0 and need.value > 0


def test_norm(lib):
    for kw, code in [(dict(rows=-1), -2), (dict(channels=0), -2), (dict(groups=0), -2), (dict(groups=3), -2), (dict(eps=-1.0), -5),
                     (dict(eps=float("nan")), -5), (dict(rows=3, x=None), -1), (dict(rows=3, z=None), -1), (dict(rows=3, weight=None), -1),
                     (dict(rows=3, out=None), -1)]:
        assert norm(lib, **kw) == code, kw


LAUNCHES = r"""
import ctypes, itertools, sys
sys.path.insert(0, sys.argv[3])
hip = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(sys.argv[2])
P, I, L, F, Z = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t
lib.uniql_state_space_scan.argtypes = [P, L, L, P, L, P, P, L, L, P, L, L, P, P, I, F, F, P, P, P, P, L, L, P, Z, I, I, I, I, I, P]
lib.uniql_state_space_scan_workspace.argtypes = [I, I, I, I, I, I, ctypes.POINTER(Z)]
class Sequences(ctypes.Structure):
    _fields_ = [("cu", P), ("starts", P), ("places", P), ("count", I), ("pool", I)]
fake = 1 << 20   # an address that nobody reads
def call(rows, count, heads, p, n, temp_bytes, cu=fake, x_row=1 << 16):
    s = Sequences(cu, None, None, count, 4)
    before = hip.fake_launches()
    code = lib.uniql_state_space_scan(fake, x_row, p, fake, heads, fake, fake, n, n, fake, n, n, None, None, 1, 0.0, 1.0, fake, fake, ctypes.byref(s),
                                      fake, heads * p, p, fake, temp_bytes, rows, heads, 1, p, n, None)
    return code, hip.fake_launches() - before
for rows, count, (heads, p, n) in itertools.product((1, 2, 63, 64, 65, 333, 4096, 16384, 100000), (1, 2, 64, 500),
        ((1, 1, 1), (2, 64, 128), (8, 100, 33), (128, 64, 128), (128, 54, 96), (128, 64, 256), (600, 128, 192))):
    need = Z(0)
    assert lib.uniql_state_space_scan_workspace(rows, count, heads, 1, p, n, ctypes.byref(need)) == 0
    code, launches = call(rows, count, heads, p, n, need.value)
    singles = count >= 4 and count * heads < 1 << 20   # single tokens among several sequences have a launch of their own
    assert code == 0 and launches == (2 if need.value else 1) + singles, (rows, count, heads, code, launches)
    if need.value:
        assert call(rows, count, heads, p, n, need.value - 1) == (-4, 0)
    if rows <= 4096:
        assert call(rows, rows, heads, p, n, 0, cu=None) == (0, 1)   # a token each asks for no scratch memory
    assert call(rows, count, heads, p, n, need.value, x_row=(1 << 23) + 2)[0] == 0   # rows far apart do not go straight to LDS
assert hip.fake_refused() == 0 and hip.fake_attributes() == 0
"""


def test_scratch_memory_is_asked_for_where_a_launch_needs_it(tmp_path):
    """two launches where there is scratch memory, one where there is none, one more for single tokens, and no attribute set (calls are recorded into graphs)"""
    if shutil.which("g++") is None or not os.path.exists(LIB_PATH):
        pytest.skip("g++ and the built library are needed")
    recorder = str(tmp_path / "fake_hip.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", os.path.join(HERE, "fake_hip.cpp"), "-o", recorder], check=True)
    run = subprocess.run([sys.executable, "-c", LAUNCHES, recorder, LIB_PATH, os.path.dirname(HERE)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
