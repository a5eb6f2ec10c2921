"""CPU checks of the orthogonalised updates' entry points: sizes, and refusals before any launch."""
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


QUINTIC = (3.4445, -4.7750, 2.0315)


def shape(count=2, rows=40, cols=60):
    return struct.pack("3q", count, rows, cols)


def view(dtype=0, data=0x1000, strides=(2400, 60, 1, 0)):
    return struct.pack("Pii4q", data, dtype, 0, *strides)


def run(L, s=None, x=None, out=0x2000, steps=5, k=QUINTIC, eps=1e-7, ws=0x4000, n=1 << 40):
    return L.gdn2_orthogonalize(s or shape(), x or view(), out, steps, None if k is None else struct.pack("3d", *k),
                                ctypes.c_float(eps), ws, n, None)


def update(L, s=None, table=(0x1000, 0x2000, 0x3000) * 2, steps=5, k=QUINTIC, ws=0x4000, n=1 << 40):
    f = ctypes.c_float
    return L.gdn2_muon_update(s or shape(), None if table is None else struct.pack(f"{len(table)}P", *table),
                              f(0.1), f(0.95), 1, f(0), steps, struct.pack("3d", *k), f(1e-7), ws, n, None)


def message(L):
    return L.gdn2_last_error().decode()


@pytest.mark.parametrize("sizes", [(-1, 4, 4), (1, 0, 4), (1, 4, 0), (1 << 31, 4, 4), (1, (1 << 24) + 1, 1),
                                   (1, 1 << 16, 1 << 15)])
def test_bad_shapes(L, sizes):
    assert run(L, shape(*sizes)) == 2 and update(L, shape(*sizes)) == 2
    assert L.gdn2_orthogonalize_workspace_bytes(shape(*sizes)) == 0


def test_refusals(L):
    assert run(L, x=view(2)) == 3 and run(L, x=view(data=0)) == 1 and run(L, out=None) == 1
    assert run(L, x=view(strides=(2400, -60, 1, 0))) == 1
    for steps in (0, -1, 101):
        assert run(L, steps=steps) == 1 and update(L, steps=steps) == 1 and "steps" in message(L)
    for eps in (-1.0, float("nan"), float("inf")):
        assert run(L, eps=eps) == 1 and "epsilon" in message(L)
    for k in ((50.0, 0, 0), (float("inf"), 0, 0), (float("nan"), 0, 0), (1.0, 1.0, 1.0)):
        assert run(L, k=k, steps=20) == 1 and update(L, k=k, steps=20) == 1 and "grow" in message(L)
    assert run(L, k=None) == 1
    need = L.gdn2_orthogonalize_workspace_bytes(shape())
    assert run(L, n=need - 1) == 4 and run(L, ws=None) == 4 and "workspace" in message(L)
    assert run(L, ws=0x4008, n=need) == 1 and update(L, ws=0x4008, n=need) == 1
    assert update(L, table=None) == 1 and update(L, n=need - 1) == 4
    assert update(L, table=(0x1000, 0x2000, 0x3000, 0x1000, None or 0, 0x3000)) == 1 and "tensor 1" in message(L)
    assert run(L, shape(0), x=view(data=0), out=None, ws=None) == 0 and update(L, shape(0), table=None) == 0


@pytest.mark.parametrize("rows,cols", [(1, 1), (512, 512), (512, 2816), (2816, 512), (1, 1 << 24), (1 << 15, 1 << 15)])
def test_sizes(L, rows, cols):
    one, many = (L.gdn2_orthogonalize_workspace_bytes(shape(n, rows, cols)) for n in (1, 1000))
    assert 0 < one <= many <= max(one, (2 << 30) + 100000)
