"""CPU checks of the token scores' entry points: refusals before any launch."""
import ctypes
import os
import struct

import pytest


@pytest.fixture(scope="module")
def L():
    from delta_kernels import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libgdn2_amd.so not built")
    return _lib.lib()


def view(dtype=0, data=0x1000, strides=(64, 1, 0, 0)):
    return struct.pack("Pii4q", data, dtype, 0, *strides)


def forward(L, rows=4, width=64, x=None, target=0x2000, ts=1, temperature=1.0, top=0, lp=0x3000, tlp=None,
            tt=None, ws=None, n=0):
    return L.gdn2_token_score_forward(rows, width, x or view(), target, ts, None, 0,
                                      ctypes.c_float(temperature), top, lp, 0x4000, tlp, tt, None, ws, n, None)


def backward(L, rows=4, width=64, x=None, stats=0x3000, dls=1, dx=0x4000):
    return L.gdn2_token_score_backward(rows, width, x or view(), 0x2000, 1, None, 0, ctypes.c_float(1.0),
                                       stats, 0x5000, dls, None, 0, dx, None)


def message(L):
    return L.gdn2_last_error().decode()


def test_refusals(L):
    assert forward(L, rows=-1) == 2 and forward(L, width=0) == 2
    assert forward(L, rows=1 << 31) == 2 and forward(L, width=1 << 31) == 2
    assert forward(L, x=view(2)) == 3 and "x:" in message(L)
    assert forward(L, x=view(data=0)) == 1 and forward(L, target=None) == 1
    assert forward(L, x=view(strides=(-64, 1, 0, 0))) == 1 and forward(L, ts=-1) == 1
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-45, 3e38):
        assert forward(L, temperature=t) == 1 and "temperature" in message(L)
    assert forward(L, top=-1) == 2 and forward(L, top=65) == 2 and "top" in message(L)
    assert forward(L, width=8, top=9, tlp=0x5000, tt=0x6000) == 2
    assert forward(L, top=4) == 1 and forward(L, lp=None) == 1
    assert forward(L, rows=0, x=view(data=0), target=None, lp=None) == 0
    assert backward(L, stats=None) == 1 and backward(L, dx=None) == 1 and backward(L, dls=-1) == 1
    assert backward(L, rows=0) == 0


def test_more_rows_than_a_launch_has(L):
    assert forward(L, rows=1 << 24, width=8) == 2 and "rows" in message(L)
    assert backward(L, rows=1 << 24, width=8) == 2 and "rows" in message(L)


def test_workspace(L):
    size = L.gdn2_token_score_workspace_bytes
    assert size(8192, 32768, 8) == 0 and size(8, 32768, 64) == 0 and size(65, 1 << 20, 8) == 0
    need = size(2, 200000, 8)
    assert need > size(2, 200000, 0) > 0
    assert size(-1, 200000, 0) == 0 and size(1, 0, 0) == 0 and size(1, 200000, 65) == 0
    wide = dict(rows=2, width=200000, x=view(strides=(200000, 1, 0, 0)), top=8, tlp=0x5000, tt=0x6000)
    assert forward(L, **wide) == 4 and forward(L, **wide, ws=0x7000, n=need - 1) == 4 and "workspace" in message(L)
    assert forward(L, **wide, ws=0x7008, n=need) == 1
