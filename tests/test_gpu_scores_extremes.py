"""Token scores where temperatures, upstream gradients, mask values or sure tokens go to extremes, against the float64
oracle with the bounds of test_gpu_scores."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from gpu_util import dev, host  # noqa: E402
from test_gpu_scores import BOTH, E, F, case, check, dk, rounded, run  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@BOTH
@pytest.mark.parametrize("temperature", [1e-9, 1e-20, 1e-30, 1e-36])
def test_ruled_out_tokens_at_small_temperatures(dk, temperature, dtype):  # noqa: F811
    """Their gradient is 0, however large d_entropy / temperature is."""
    tau = float(np.float32(temperature))
    c = case(31, 6, 300, dtype, tau, masked=True)
    keep = np.isfinite(c["x"])
    c["x"] = rounded(np.where(keep, c["x"] * tau, -np.inf), dtype)
    r, dx = run(dk, c, dtype, 4)
    check(c, dtype, r, dx)
    assert not host(dx)[~keep].any()


@BOTH
def test_ruled_out_tokens_under_large_gradients(dk, dtype):  # noqa: F811
    for size in (1e10, 1e20, 1e35):
        c = case(32, 6, 300, dtype, masked=True)
        c["d"], c["dh"] = (rounded(c[n] * size, F) for n in ("d", "dh"))
        r, dx = run(dk, c, dtype)
        check(c, dtype, r, dx)
        assert not host(dx)[np.isinf(c["x"])].any()


@BOTH
def test_a_sure_token_at_a_small_temperature(dk, dtype):  # noqa: F811
    """The gradients of a row whose probabilities are 0 and 1 are 0, also where those of its scores, divided by the
    temperature, are no float32."""
    x = torch.full((2, 50), -1.0, device="cuda").to(dtype)
    x[:, 7] = 1
    t = torch.tensor([7, 7], device="cuda")
    r, stats = dk.token_log_probs_forward(x, t, 0, None, 1e-36)
    up = torch.full((2,), 1e4, device="cuda")
    assert not dk.token_log_probs_backward(x, t, None, 1e-36, stats, up, up).any()
