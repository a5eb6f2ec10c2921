"""CPU checks of the linear-attention block's entry points: sizes, and refusals before any launch."""
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


def shape(B=2, T=200, H=3, K=64, V=64):
    return struct.pack("5q", B, T, H, K, V)


def view(dtype=0, data=0x1000, strides=(64, 64, 64, 1)):
    return struct.pack("Pii4q", data, dtype, 0, *strides)


def message(L):
    return L.gdn2_last_error().decode()


def size(L, query, s, dtype):
    from delta_kernels._lib import Gdn2Shape
    more = (1,) if "checkpoint" in query else ()
    return getattr(L, query)(Gdn2Shape.from_buffer_copy(s), dtype, *more)


def scan(L, s=None, q=None, k=None, v=None, g=None, valid=None, initial=None, out=0x2000, final=0x3000,
         ck=0x4000, n=1 << 40):
    return L.gdn2_linear_scan(s or shape(), q or view(), k or view(), v or view(), g or view(), valid,
                              None, initial, out, final, 1, ck, n, None)


@pytest.mark.parametrize("sizes,text", [
    ((0, 8, 2, 32, 64), "nonempty"), ((2, 0, 2, 32, 64), "nonempty"), ((2, 8, 0, 32, 64), "nonempty"),
    ((2, 8, 2, 0, 64), "widths"), ((2, 8, 2, 32, 129), "widths"), ((1 << 40, 8, 2, 32, 64), "too many"),
    ((1 << 11, 1 << 20, 2, 32, 64), "too many")])
def test_bad_shapes(L, sizes, text):
    assert scan(L, shape(*sizes)) == 2 and text in message(L)
    for query in ("gdn2_linear_checkpoint_bytes", "gdn2_linear_workspace_bytes"):
        assert size(L, query, shape(*sizes), 0) == 0


def test_bad_types(L):
    assert scan(L, q=view(2)) == 3 and "q:" in message(L)
    assert scan(L, q=view(1)) == 3 and "k: dtype must be BF16" in message(L)
    assert scan(L, g=view(1)) == 3 and "g: dtype must be F32" in message(L)
    assert scan(L, valid=view(1)) == 3 and "valid" in message(L)
    assert size(L, "gdn2_linear_checkpoint_bytes", shape(), 2) == 0 and "dtype" in message(L)


def test_bad_pointers_and_strides(L):
    assert scan(L, v=view(data=0)) == 1 and "v: data is null" in message(L)
    assert scan(L, out=None) == 1 and scan(L, final=None) == 1
    assert scan(L, k=view(strides=(64, -64, 64, 1))) == 1 and "negative stride" in message(L)
    assert scan(L, initial=view(strides=(64, 64, 1 << 22, 1))) == 2 and "initial" in message(L)


def test_bad_buffers(L):
    need = size(L, "gdn2_linear_checkpoint_bytes", shape(), 0)
    assert need > 0
    assert scan(L, n=need - 1) == 4 and "checkpoint" in message(L)
    assert scan(L, ck=0x4004, n=need) == 1 and "16-byte aligned" in message(L)
    args = [shape()] + [view()] * 4 + [None] * 3
    tail = [view(), None] + [None] * 6
    assert L.gdn2_linear_backward(*args, 0x4000, need - 1, *tail, 0x5000, 1 << 40, None) == 4
    ws = size(L, "gdn2_linear_workspace_bytes", shape(), 0)
    assert L.gdn2_linear_backward(*args, 0x4000, need, *tail, 0x5000, ws - 1, None) == 4
    assert "workspace" in message(L)


@pytest.mark.parametrize("T", [1, 64, 512, 5000])
@pytest.mark.parametrize("K", [16, 100])
def test_a_forward_alone_needs_less(L, K, T):
    from delta_kernels._lib import Gdn2Shape
    s = Gdn2Shape.from_buffer_copy(shape(T=T, K=K))
    sizes = [L.gdn2_linear_checkpoint_bytes(s, 0, train) for train in (0, 1)]
    assert 0 < sizes[0] <= sizes[1]
    assert K > 64 or sizes[0] < sizes[1]


def test_step_takes_one_token(L):
    assert L.gdn2_linear_step(shape(), *[view()] * 4, None, None, 0x2000, 0x3000, None) == 2
    assert "time == 1" in message(L)
    assert L.gdn2_linear_step(shape(T=1), *[view()] * 4, None, None, None, 0x3000, None) == 1


def test_layer_norm_refusals(L):
    def forward(rows=(1, 1, 4, 8), x=None, weight=0x2000, y=0x3000):
        return L.gdn2_layer_norm_forward(struct.pack("4q", *rows), ctypes.c_float(1e-5), x or view(),
                                         weight, None, y, None, None, None)
    assert forward((1, 1, 4, 0)) == 2 and "width" in message(L)
    assert forward((1, -1, 4, 8)) == 2
    assert forward((1 << 20, 1 << 20, 1, 8)) == 2 and "rows" in message(L)
    assert forward(x=view(2)) == 3
    assert forward(weight=None) == 1 and forward(y=None) == 1
    assert forward((1, 0, 4, 8), y=None) == 0  # nothing to do
    n = L.gdn2_layer_norm_workspace_bytes(4, 8)
    assert n > 0 and L.gdn2_layer_norm_workspace_bytes(-1, 8) == 0
    back = [struct.pack("4q", 1, 1, 4, 8), view(), 0x2000, 0x3000, 0x4000, view(), 0x5000, 0x6000, None]
    assert L.gdn2_layer_norm_backward(*back, 0x7000, n - 1, None) == 4
    assert L.gdn2_layer_norm_backward(*back, 0x7004, n, None) == 1
    back[5] = view(1)
    assert L.gdn2_layer_norm_backward(*back, 0x7000, n, None) == 3


def test_swiglu_q8_refusals(L):
    def forward(rows=4, width=32, dtype=0, h=0x1000):
        return L.gdn2_swiglu_q8_forward(rows, width, dtype, h, 0x2000, 0x3000, 0x4000, None)
    assert forward(width=0) == 2 and forward(rows=-1) == 2
    assert forward(rows=1 << 31, width=1 << 20) == 2 and "too many" in message(L)
    assert forward(dtype=2) == 3 and forward(h=None) == 1
    assert forward(rows=0, h=None) == 0
    assert L.gdn2_swiglu_q8_backward(4, 32, 0, 0x1000, 0x2000, None, 0x3000, None, None) == 1
