"""Token scores where temperatures, upstream gradients, mask values or sure tokens go to extremes, against the float64
oracle with the bounds of test_gpu_scores."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from gpu_util import dev, host  # noqa: E402
from test_gpu_scores import BOTH, E, F, H, case, check, dk, rounded, run  # noqa: E402, F401

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


LOWEST = {dt: float(torch.finfo(dt).min) for dt in (F, H)}


@BOTH
@pytest.mark.parametrize("top", [1, 2, 20, 64])
def test_rows_masked_by_the_lowest_value(dk, top, dtype):  # noqa: F811
    """Equal ones go by their index, also where there are fewer others than alternatives."""
    for width in (70, 500, 5003):
        c = case(33, 8, width, dtype)
        low = LOWEST[dtype]
        c["x"][:6] = low
        c["x"][0, 37] = 5
        c["x"][1, [3, 40, 69]] = (1, 2, 1)
        c["x"][2, width - 30:] = np.arange(30) // 3
        c["x"][4, ::3] = -np.inf
        c["x"][4, 50] = -2
        c["x"][5, ::2] = -np.inf
        c["x"][6, 5:] = -np.inf
        c["x"][6, 40:60] = low
        c["t"][:7] = (37, 40, width - 1, 9, 50, 1, 2)
        c["x"] = rounded(c["x"], dtype)
        check(c, dtype, *run(dk, c, dtype, top))


@BOTH
@pytest.mark.parametrize("top", [2, 20])
def test_rows_in_parts_masked_by_the_lowest_value(dk, top, dtype):  # noqa: F811
    width = 90001
    c = case(34, 5, width, dtype)
    c["x"][:4] = LOWEST[dtype]
    c["x"][0, 60000] = 5
    c["x"][1, 100:102] = (1, 2)
    c["x"][1, 80000:80015] = 1
    c["x"][2, ::2] = -np.inf
    c["x"][3, 37] = 5
    c["t"][:4] = (60000, 101, 1, 37)
    c["x"] = rounded(c["x"], dtype)
    check(c, dtype, *run(dk, c, dtype, top))
