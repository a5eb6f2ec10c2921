"""The float64 oracle of the linear-attention block against central differences and known values
(CPU)."""
import numpy as np
import pytest

from oracle import linear_oracle as lo


def _case(seed, B=1, T=7, H=2, K=3, V=4):
    r = np.random.default_rng(seed)
    x = dict(q=r.normal(size=(B, T, H, K)), k=r.normal(size=(B, T, H, K)),
             v=r.normal(size=(B, T, H, V)), g=-np.abs(r.normal(size=(B, T, H))),
             initial=r.normal(size=(B, H, K, V)))
    valid, reset = np.ones((B, T)), np.zeros((B, T))
    if T > 4:
        valid[0, 2] = 0
        reset[0, 4] = 1
    return x, valid, reset, r.normal(size=(B, T, H, V)), r.normal(size=(B, H, K, V))


def test_attention_gradient_is_that_of_differences():
    x, valid, reset, do, df = _case(0)

    def loss(y):
        out, fin, _ = lo.attention(y["q"], y["k"], y["v"], y["g"], valid, reset, y["initial"])
        return (out * do).sum() + (fin * df).sum()

    grads = lo.attention_backward(x["q"], x["k"], x["v"], x["g"], valid, reset, x["initial"], do, df)
    for n in x:
        got, h = grads["d" + n], 1e-5
        for i in np.ndindex(x[n].shape):
            lo_, hi = dict(x), dict(x)
            lo_[n], hi[n] = x[n].copy(), x[n].copy()
            lo_[n][i] -= h
            hi[n][i] += h
            assert abs((loss(hi) - loss(lo_)) / (2 * h) - got[i]) < 1e-7, (n, i)


def test_attention_of_one_token_and_of_none():
    x, _, _, _, _ = _case(1, T=1)
    out, fin, _ = lo.attention(x["q"], x["k"], x["v"], x["g"], initial=x["initial"])
    S = np.exp(x["g"][0, 0, 1]) * x["initial"][0, 1] + np.outer(x["k"][0, 0, 1], x["v"][0, 0, 1])
    np.testing.assert_allclose(fin[0, 1], S, rtol=1e-14)
    np.testing.assert_allclose(out[0, 0, 1], x["q"][0, 0, 1] @ S, rtol=1e-14)
    out, fin, _ = lo.attention(x["q"], x["k"], x["v"], x["g"], valid=np.zeros((1, 1)),
                               initial=x["initial"])
    assert np.all(out == 0) and np.array_equal(fin, x["initial"])


def test_layer_norm_gradient_is_that_of_differences():
    r = np.random.default_rng(2)
    x, w, b, dy = (r.normal(size=s) for s in ((3, 5), 5, 5, (3, 5)))
    dx, dw, db = lo.layer_norm_backward(x, w, 1e-3, dy)

    def loss(x, w, b):
        return (lo.layer_norm(x, w, b, 1e-3)[0] * dy).sum()

    for at, got in ((0, dx), (1, dw), (2, db)):
        for i in np.ndindex(got.shape):
            p, m = [[a.copy() for a in (x, w, b)] for _ in range(2)]
            p[at][i] += 1e-5
            m[at][i] -= 1e-5
            assert abs((loss(*p) - loss(*m)) / 2e-5 - got[i]) < 1e-8


def test_swiglu_gradient_is_that_of_differences():
    r = np.random.default_rng(3)
    h, da = r.normal(size=(2, 8)) * 3, r.normal(size=(2, 4))
    got = lo.swiglu_backward(h, da)
    for i in np.ndindex(h.shape):
        p, m = h.copy(), h.copy()
        p[i] += 1e-5
        m[i] -= 1e-5
        d = ((lo.swiglu(p) - lo.swiglu(m)) * da).sum() / 2e-5
        assert abs(d - got[i]) < 1e-8


def test_q8_codes():
    h = np.zeros((1, 2 * 33))
    h[0, :4] = [127, 64.5, 63.5, -0.5]  # 2^0: ties go to the even code
    h[0, 32] = 127.5                    # a block of one column: 2^1, 63.75 -> 64
    h[0, 33] = -1e-40                   # below the smallest scale
    codes, exps = lo.q8(h)
    assert list(codes[0, :4]) == [127, 64, 64, 0] and codes[0, 32] == 64
    assert list(exps[0]) == [127, 128, 1, 1] and codes[0, 33] == 0
    h[0, 1] = np.nan
    codes, exps = lo.q8(h)
    assert exps[0, 0] == 255 and np.isnan(lo.q8_values(codes, exps)[0, :32]).all()
    assert np.isfinite(lo.q8_values(codes, exps)[0, 32:]).all()


@pytest.mark.parametrize("seed", range(3))
def test_q8_error_is_below_its_bound(seed):
    h = np.random.default_rng(seed).normal(size=(5, 2 * 70)) * 10.0 ** seed
    v = lo.q8_values(*lo.q8(h))
    for half in range(2):
        for c in range(0, 70, 32):
            at = np.s_[:, half * 70 + c:half * 70 + min(70, c + 32)]
            assert np.all(np.abs(v[at] - h[at]).max(1) < np.abs(h[at]).max(1) / 127)
