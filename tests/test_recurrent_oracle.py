"""The oracle of the recurrent model's operators, against its own differences and plain statements."""
import numpy as np
import pytest

from oracle import recurrent_oracle as ro


def case(seed, B=2, T=9, W=3):
    r = np.random.default_rng(seed)
    valid = (r.random((B, T)) < 0.8).astype(float)
    reset = (r.random((B, T)) < 0.2).astype(float)
    return (r.normal(size=(B, T, W)), -r.exponential(size=(B, T, W)), valid, reset,
            r.normal(size=(B, W)), r.normal(size=(B, T, W)), r.normal(size=(B, W)))


@pytest.mark.parametrize("seed", range(3))
def test_recurrence_gradients_are_the_differences(seed):
    x, g, valid, reset, initial, dy, df = case(seed)

    def loss(x, g, initial):
        y, fin, _ = ro.recurrence(x, g, valid, reset, initial)
        return (y * dy).sum() + (fin * df).sum()

    grads = ro.recurrence_backward(x, g, valid, reset, initial, dy, df)
    args = [x, g, initial]
    step = 1e-6
    for n, d in enumerate(grads):
        for i in np.ndindex(d.shape):
            up, down = [a.copy() for a in args], [a.copy() for a in args]
            up[n][i] += step
            down[n][i] -= step
            # central differences: step^2 of the third derivative, and 1e-16 |loss| / step
            assert abs((loss(*up) - loss(*down)) / (2 * step) - d[i]) < 1e-7


def test_recurrence_is_its_sum():
    x, g, _, _, initial, _, _ = case(7)
    y, fin, _ = ro.recurrence(x, g, None, None, initial)
    total = np.cumsum(g, 1)
    for t in range(x.shape[1]):
        want = np.exp(total[:, t]) * initial
        for s in range(t + 1):
            want = want + np.exp(total[:, t] - total[:, s]) * x[:, s]
        assert np.allclose(y[:, t], want, rtol=1e-12, atol=1e-14)
    assert np.array_equal(fin, y[:, -1])


def test_cuts():
    x, g, _, _, _, dy, _ = case(8)
    x[0, 2, 0] = np.inf
    g[0, 3, 0] = -88.0  # below 2^-126
    y, _, carried = ro.recurrence(x, g)
    assert np.isfinite(y[0, 3:, 0]).all() and carried[0, 3, 0] == 0
    dy[0, 5, 0] = np.nan
    dx, dg, _ = ro.recurrence_backward(x, g, None, None, None, dy)
    assert np.isfinite(dx[0, :3, 0]).all() and dg[0, 3, 0] == 0


@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_score_gradients_are_the_differences(temperature):
    r = np.random.default_rng(3)
    x, t = r.normal(size=(3, 7)), np.array([0, 6, 2])
    x[1, 3] = -np.inf
    d, dh = r.normal(size=3), r.normal(size=3)

    def loss(x):
        _, lp, h = ro.scores(x, t, temperature)
        return (lp * d + h * dh).sum()

    dx = ro.scores_backward(x, t, d, dh, temperature)
    for i in np.ndindex(x.shape):
        if not np.isfinite(x[i]):
            assert dx[i] == 0
            continue
        up, down = x.copy(), x.copy()
        up[i] += 1e-6
        down[i] -= 1e-6
        assert abs((loss(up) - loss(down)) / 2e-6 - dx[i]) < 1e-8


def test_scores_of_two():
    lp, given, h = ro.scores(np.array([[0.0, np.log(3.0)]]), np.array([1]))
    assert np.allclose(np.exp(lp), [[0.25, 0.75]]) and np.allclose(given, np.log(0.75))
    assert np.allclose(h, -0.25 * np.log(0.25) - 0.75 * np.log(0.75))
    assert ro.top(np.array([[1.0, np.nan, 2.0, 2.0, -0.0, 0.0]]), 6).tolist() == [[1, 2, 3, 0, 4, 5]]


@pytest.mark.parametrize("shape", [(4, 9), (9, 4), (5, 5)])
def test_products_change_singular_values_alone(shape):
    r = np.random.default_rng(2)
    u = r.normal(size=shape)
    w, s, vt = np.linalg.svd(u, full_matrices=False)
    a, b, c = ro.COEFFICIENTS
    t = s / (np.sqrt((s ** 2).sum()) + 1e-7)
    for _ in range(5):
        t = t * (a + b * t ** 2 + c * t ** 4)
    got = ro.orthogonalize(u)
    assert np.allclose(got, w @ np.diag(t) @ vt, atol=1e-12)
    assert np.all((t > 0.6) & (t < 1.3))
    near = ro.orthogonalize(u, product=ro.split_product)
    assert 0 < np.abs(near - got).max() < 1e-4
