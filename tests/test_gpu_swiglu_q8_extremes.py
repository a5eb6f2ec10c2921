"""8-bit SwiGLU at the largest values that its types hold.

With e = 2^-24 results are within 64 e of the magnitudes of their terms, and half a unit of bf16, 2^-8 |result|,
where they are bf16."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import linear_oracle as lo  # noqa: E402
from gpu_util import dev, host  # noqa: E402
from test_gpu_swiglu_q8 import dk  # noqa: E402,F401

pytestmark = pytest.mark.gpu

U, E = 2.0 ** -8, 2.0 ** -24


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
