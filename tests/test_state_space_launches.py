"""Which kernels the calls of a state-space layer launch, and how much of them (no GPU needed: the launches are recorded)."""
import os
import shutil
import subprocess
import sys

import pytest

from uniql_amd.build import LIB_PATH

HERE = os.path.dirname(os.path.abspath(__file__))

PRELUDE = r"""
import ctypes, sys
sys.path.insert(0, sys.argv[3])
hip = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(sys.argv[2])
from uniql_amd._capi import SIGNATURES
for name in ("uniql_state_space_scan", "uniql_causal_conv", "uniql_gated_group_norm"):
    getattr(lib, name).restype, getattr(lib, name).argtypes = SIGNATURES[name]
hip.recorder_kernel.restype, hip.recorder_workgroups.restype = ctypes.c_void_p, ctypes.c_uint64
class Sequences(ctypes.Structure):
    _fields_ = [("cu", ctypes.c_void_p), ("starts", ctypes.c_void_p), ("places", ctypes.c_void_p), ("count", ctypes.c_int), ("pool", ctypes.c_int)]
fake = 1 << 20   # an address that nobody reads
def scan(rows, count, heads, p, n, x_row, x_head, cu=fake, x=fake, b_row=None):
    s = Sequences(cu, None, None, count, 1 << 30)
    hip.recorder_reset()
    code = lib.uniql_state_space_scan(x, x_row, x_head, fake, heads, fake, fake, b_row or n, n, fake, n, n, None, None, 1, 0.0, 1.0, fake, fake,
                                      ctypes.addressof(s), fake, heads * p, p, fake, 1 << 40, rows, heads, 1, p, n, None)
    return code, hip.recorder_kernel()
"""


def run(source, tmp_path):
    if shutil.which("g++") is None or not os.path.exists(LIB_PATH):
        pytest.skip("g++ and the built library are needed")
    recorder = str(tmp_path / "recorder.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", os.path.join(HERE, "launch_recorder.cpp"), "-o", recorder], check=True)
    done = subprocess.run([sys.executable, "-c", PRELUDE + source, recorder, LIB_PATH, os.path.dirname(HERE)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_odd_widths_pass_through_registers(tmp_path):
    """rows of even strides and odd widths would go straight to LDS from a buffer that ends within a word"""
    run(r"""
for heads, p, n in ((2, 53, 96), (4, 1, 8), (1, 27, 128), (2, 65, 64), (3, 127, 256), (1, 63, 192)):
    pitch = p + 1
    direct = scan(200, 1, heads, p + 1, n, heads * pitch, pitch)
    odd = scan(200, 1, heads, p, n, heads * pitch, pitch)
    through = scan(200, 1, heads, p, n, heads * p | 1, p)
    even_through = scan(200, 1, heads, p + 1, n, heads * pitch + 1, pitch)
    assert all(code == 0 for code, _ in (direct, odd, through, even_through))
    assert odd[1] == through[1] == even_through[1] != direct[1], (p, n)
""", tmp_path)


def test_large_calls_are_several_launches(tmp_path):
    """what the prototypes allow is not refused for its number of workgroups, and no launch has 2^32 threads"""
    run(r"""
def recorded(code, workgroups, several):
    assert code == 0 and hip.recorder_too_large() == 0
    assert hip.recorder_workgroups() == workgroups, (hip.recorder_workgroups(), workgroups)
    assert (hip.recorder_launches() > 1) == several, hip.recorder_launches()
most = (1 << 24) - 1
# single tokens: rows of eight of a head a workgroup where states are no fours
for rows, heads, p, n, blocks in ((8191, 128, 128, 130, 16), (8192, 128, 128, 130, 16), (1 << 24, 1, 1, 1, 1), (40000, 1 << 15, 1, 4, 1), (1 << 24, 5, 100, 128, 2)):
    code, _ = scan(rows, rows, heads, p, n, heads * p, p, cu=None)
    recorded(code, rows * heads * blocks, rows * heads * blocks > most)
def conv(rows, count, channels, cu=fake):
    s = Sequences(cu, None, None, count, 1 << 30)
    hip.recorder_reset()
    return lib.uniql_causal_conv(fake, channels, fake, None, fake, fake, ctypes.addressof(s), fake, channels, rows, channels, 4, 1, None)
recorded(conv(most, most, 8, None), most, False)
recorded(conv(1 << 24, 1 << 24, 8, None), 1 << 24, True)
recorded(conv(1 << 27, 1 << 24, 8), (1 << 24) + (1 << 27) // 32, True)
recorded(conv(1 << 27, 1 << 24, 4096), 2 * ((1 << 24) + (1 << 27) // 32), True)
def norm(rows, channels, groups):
    hip.recorder_reset()
    return lib.uniql_gated_group_norm(fake, channels, fake, channels, fake, fake, channels, rows, channels, groups, 1e-5, None)
recorded(norm(1 << 27, 1024, 1), 1 << 25, True)
recorded(norm(1 << 27, 64, 8), 1 << 28, True)
recorded(norm(1 << 25, 4096, 1), 1 << 25, True)
recorded(norm(1 << 24, 4096, 1), 1 << 24, True)
recorded(norm(most, 4096, 1), most, False)
recorded(norm(3, 64, 8), 6, False)
""", tmp_path)
