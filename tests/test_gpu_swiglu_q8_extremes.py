"""8-bit SwiGLU at the ends of what float32 holds: its largest values, and gates whose sigmoid is below the normal
numbers while the result is one.

With e = 2^-24 results are within 16 e of the magnitudes of their terms, times 1 + |gate| for the exponential, and half
a unit of bf16, 2^-8 |result|, where they are bf16; nothing is left over for small ones but half of the smallest
normal number."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import linear_oracle as lo  # noqa: E402
from gpu_util import dev, host  # noqa: E402
from test_gpu_swiglu_q8 import dk  # noqa: E402,F401

pytestmark = pytest.mark.gpu

U, E, TINY = 2.0 ** -8, 2.0 ** -24, 2.0 ** -127


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_the_largest_values(dk, dtype):  # noqa: F811
    top = float(torch.finfo(dtype).max)
    r = np.random.default_rng(0)
    h = torch.tensor(r.normal(size=(4, 128))).to(dtype).double().numpy()
    h[0, 3], h[1, 70], h[2, 32:64], h[3, 40] = top, -top, -top, 127 * 2.0 ** 121
    _, codes, exps = dk.swiglu_q8_forward(dev(h, dtype))
    kept = host(dk.q8_values(codes, exps))
    assert np.isfinite(kept).all()
    block = np.repeat(np.abs(h).reshape(4, 4, 32).max(2), 32, 1)
    assert np.all(np.abs(kept - h) < block / 127)
    rc, re = lo.q8(h)
    assert np.array_equal(codes.cpu().numpy(), rc) and np.array_equal(exps.cpu().numpy(), re)
    da = torch.full((4, 64), 2.0 ** -100, dtype=dtype, device="cuda")
    dh, again = dk.swiglu_q8_backward(codes, exps, da)
    assert torch.isfinite(dh).all()
    want = lo.swiglu_backward(kept, host(da))
    big = np.s_[[1], 6]  # the gate beside the up projection's largest value
    assert np.all(np.abs(host(dh)[big] - want[big]) <= (64 * E + U) * np.abs(want[big]))


@pytest.mark.parametrize("x", [-80.0, -87.0, -88.5, -89.0, -90.0, -91.0, -91.5, -1e-3, 1e-37, 2e-38])
def test_gates_whose_sigmoid_is_not_a_normal_number(dk, x):  # noqa: F811
    x = float(np.float32(x))
    h = np.zeros((1, 64))
    h[:, :32], h[:, 32:] = x, 1.0
    a, codes, exps = dk.swiglu_q8_forward(dev(h))
    size = 1 + abs(x)
    want = lo.swiglu(h)
    assert np.all(np.abs(host(a) - want) <= 16 * E * size * np.abs(want) + TINY)
    kept = lo.q8_values(*lo.q8(h))
    dh, again = dk.swiglu_q8_backward(codes, exps, torch.ones((1, 32), device="cuda"))
    want = lo.swiglu(kept)
    assert np.all(np.abs(host(again) - want) <= 16 * E * size * np.abs(want) + TINY)
    want = lo.swiglu_backward(kept, np.ones((1, 32)))
    s = 1 / (1 + np.exp(-kept[:, :32]))
    terms = np.concatenate([s * (1 + np.abs(kept[:, :32])), s * np.abs(kept[:, :32])], 1)
    assert np.all(np.abs(host(dh) - want) <= 16 * E * size * terms + TINY)


def test_values_of_no_rows(dk):  # noqa: F811
    _, codes, exps = dk.swiglu_q8_forward(torch.empty((0, 64), device="cuda"))
    assert dk.q8_values(codes, exps).shape == (0, 64)
