"""CPU checks of the gated recurrence's entry points: sizes, and refusals before any launch."""
import os
import struct

import pytest


@pytest.fixture(scope="module")
def L():
    from delta_kernels import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libgdn2_amd.so not built")
    return _lib.lib()


def shape(B=2, T=200, W=96):
    return struct.pack("3q", B, T, W)


def view(dtype=0, data=0x1000, strides=(19200, 96, 1, 0)):
    return struct.pack("Pii4q", data, dtype, 0, *strides)


def message(L):
    return L.gdn2_last_error().decode()


def scan(L, s=None, x=None, g=None, valid=None, initial=None, out=0x2000, final=0x3000, ck=0x4000,
         n=1 << 40):
    return L.gdn2_recurrence_scan(s or shape(), x or view(), g or view(), valid, None, initial, out, final,
                                  1, ck, n, None)


@pytest.mark.parametrize("sizes,text", [
    ((0, 8, 4), "nonempty"), ((2, 0, 4), "nonempty"), ((2, 8, 0), "nonempty"), ((-1, 8, 4), "nonempty"),
    (((1 << 30) + 1, 8, 1), "too many"), ((1, (1 << 30) + 1, 1), "too many"), ((1 << 16, 8, 1 << 15), "too many")])
def test_bad_shapes(L, sizes, text):
    assert scan(L, shape(*sizes)) == 2 and text in message(L)
    assert L.gdn2_recurrence_checkpoint_bytes(shape(*sizes), 0, 1) == 0
    assert L.gdn2_recurrence_workspace_bytes(shape(*sizes), 0) == 0


def test_more_workgroups_than_a_launch_has(L):
    for sizes in ((1 << 27, 1, 1), (1 << 24, 300, 32), (1 << 26, 2, 16)):
        s = shape(*sizes)
        assert scan(L, s) == 2 and "one launch" in message(L)
        assert L.gdn2_recurrence_backward(s, view(), view(), None, None, 0x4000, 1 << 62, view(), None, 0x5000, 0x6000,
                                          None, 0x7000, 1 << 62, None) == 2


def test_bad_types(L):
    assert scan(L, x=view(2)) == 3 and "x:" in message(L)
    assert scan(L, g=view(2)) == 3 and "g:" in message(L)
    assert scan(L, valid=view(1)) == 3 and "valid" in message(L)
    assert scan(L, initial=view(1)) == 3 and "initial" in message(L)
    assert L.gdn2_recurrence_checkpoint_bytes(shape(), 2, 1) == 0 and "dtype" in message(L)


def test_bad_pointers_and_buffers(L):
    assert scan(L, x=view(data=0)) == 1 and "x: data is null" in message(L)
    assert scan(L, out=None) == 1 and scan(L, final=None) == 1
    assert scan(L, g=view(strides=(96, -96, 1, 0))) == 1 and "negative stride" in message(L)
    need = L.gdn2_recurrence_checkpoint_bytes(shape(), 0, 1)
    assert need > 0 and scan(L, n=need - 1) == 4 and "checkpoint" in message(L)
    assert scan(L, ck=None, n=need) == 4
    assert scan(L, ck=0x4004, n=need) == 1 and "16-byte aligned" in message(L)
    ws = L.gdn2_recurrence_workspace_bytes(shape(T=5000), 0)
    need = L.gdn2_recurrence_checkpoint_bytes(shape(T=5000), 0, 1)
    head = [shape(T=5000), view(), view(), None, None]
    tail = [0x5000, 0x6000, None]
    back = L.gdn2_recurrence_backward
    assert back(*head, 0x4000, need - 1, view(), None, *tail, 0x7000, ws, None) == 4
    assert back(*head, 0x4000, need, view(), None, *tail, 0x7000, ws - 1, None) == 4 and "workspace" in message(L)
    assert back(*head, 0x4000, need, view(), None, *tail, 0x7008, ws, None) == 1
    assert back(*head, 0x4000, need, view(1), None, *tail, 0x7000, ws, None) == 3 and "d_output" in message(L)
    assert back(*head, 0x4000, need, None, None, *tail, 0x7000, ws, None) == 1


@pytest.mark.parametrize("T", [1, 31, 33, 256, 257, 100000])
@pytest.mark.parametrize("W", [1, 64, 4096])
def test_sizes(L, T, W):
    for dtype in (0, 1):
        alone, train = (L.gdn2_recurrence_checkpoint_bytes(shape(1, T, W), dtype, n) for n in (0, 1))
        assert 16 <= alone and 4 * W <= train <= alone + 4 * W * (T // 32 + 1)


def test_buffers_that_nothing_needs_may_be_null(L):
    """And are asked for where they are needed: the refusals come before any launch."""
    for T, W in ((5000, 96), (600, 1)):
        s, need = shape(2, T, W), L.gdn2_recurrence_workspace_bytes(shape(2, T, W), 0)
        assert need > 16
        assert L.gdn2_recurrence_scan(s, view(), view(), None, None, None, 0x2000, 0x3000, 0, None, 0, None) == 4
    assert L.gdn2_recurrence_workspace_bytes(shape(1, 600, 1), 0) >= 16
    assert L.gdn2_recurrence_scan(shape(1, 600, 1), view(), view(), None, None, None, 0x2000, 0x3000, 0, None, 0,
                                  None) == 4


def test_step_takes_one_token(L):
    step = L.gdn2_recurrence_step
    assert step(shape(), view(), view(), None, None, 0x2000, 0x3000, None) == 2 and "time == 1" in message(L)
    assert step(shape(T=1), view(), view(), None, None, None, 0x3000, None) == 1
    assert step(shape(T=1), view(), view(), None, None, 0x2000, None, None) == 1
