"""Token scores where temperatures, upstream gradients, mask values or sure tokens go to extremes, against the float64
oracle with the bounds of test_gpu_scores."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from gpu_util import dev, host  # noqa: E402
from test_gpu_scores import BOTH, E, F, H, case, check, dk, layouts, rounded, run  # noqa: E402, F401

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


def sure(seed, width, dtype, gap, where):
    """Two rows of a sure token at `where` and others at a distance of gap to gap + 4."""
    r = np.random.default_rng(seed)
    c = case(seed, 2, width, dtype)
    c["x"] = rounded(-gap - 4 * r.random((2, width)), dtype)
    c["t"] = np.array([where, where])
    c["x"][:, where] = 0
    return c


@BOTH
@pytest.mark.parametrize("gap", [8.0, 15.0, 17.0, 19.0, 25.0])
@pytest.mark.parametrize("width", [2, 3, 4, 5, 8, 9, 16, 17, 31, 64, 1000, 10007, 70000])
def test_the_others_of_a_sure_token(dk, width, gap, dtype):  # noqa: F811
    """Log probability and entropy relative to what the others are, e_j = exp(-d_j) each, with E = 2^-24.  An
    exponential is off by (2.3 d + 2.1) E of itself: the distance's, the factor log2 e's and the product's roundings,
    and its own ulp.  A thread's sums of up to 16 floats add 16 E, up to two changes of its maximum and the row's
    (2.3 d + 2.1) E each, of distances that add up to d: (3 d + 32) E of e_j.  The sums in 64 bits stand beside 1,
    and have 2^-53 for each of up to 64 steps.  The entropy's own sum has the same terms, up to 32 roundings in a
    thread and 6 + 16 across the workgroup: (3 d + 80) E of e_j d_j.  A result is rounded once, its sum from two
    parts before."""
    for where in sorted({0, width // 2, width - 1}):
        c = sure(width, width, dtype, gap, where)
        r, dx = run(dk, c, dtype, 1)
        check(c, dtype, r, dx)
        d = np.delete(-c["x"], where, 1)
        e = np.exp(-d)
        others = e.sum(1)
        off = (e * (3 * d + 32)).sum(1) * E + 64 * 2.0 ** -53
        want = -np.log1p(others)
        err = np.abs(host(r.log_probs) - want)
        assert np.all(err <= off + E * np.abs(want)), (where, err / (off + E * np.abs(want)))
        assert torch.equal(r.top_log_probs[:, 0], r.log_probs)
        h = np.log1p(others) + (e * d).sum(1) / (1 + others)
        err = np.abs(host(r.entropy) - h)
        bound = off + (e * d * (3 * d + 80)).sum(1) * E + 2 * E * h
        assert np.all(err <= bound), (where, err / bound)


@BOTH
def test_sure_tokens_in_many_rows_and_other_layouts(dk, dtype):  # noqa: F811
    """The same bits wherever the row stands, whether its columns lie side by side, and beside ruled-out ones."""
    c = sure(41, 3000, dtype, 17.0, 1234)
    two = dev(c["x"], dtype)
    t = torch.full((514,), 1234, device="cuda")
    x = torch.randn(514, 3000, device="cuda").to(dtype)
    x[[0, 513]] = two
    want = dk.token_log_probs(x, t, 2)
    assert torch.all(want.log_probs[[0, 513]] < 0) and torch.all(want.log_probs[[0, 513]] > -1e-3)
    for place in layouts():
        got = dk.token_log_probs(place(x), t, 2)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    check(c, dtype, dk.TokenLogProbs(*(v[[0, 513]] for v in want)))
    x[:, 2000:] = -np.inf
    c["x"][:, 2000:] = -np.inf
    r = dk.token_log_probs(x, t)
    others = np.exp(np.delete(c["x"], 1234, 1)).sum(1)
    # (3 d + 32) E of the others at distances of up to 21, and 64 steps beside 1 in 64 bits
    assert np.all(np.abs(host(r.log_probs[[0, 513]]) + np.log1p(others)) <= others * 97 * E + 64 * 2.0 ** -53)
