"""SwiGLU that keeps its input in 8 bits, against the float64 oracle: codes and exponents are equal, and
with e = 2^-24 the results are within 16 e of the magnitudes of their terms (an exponential and a
reciprocal of one unit each, and six roundings), and half a unit of bf16 where they are bf16."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import linear_oracle as lo  # noqa: E402
from gpu_util import dev, host  # noqa: E402

pytestmark = pytest.mark.gpu

U, E = 2.0 ** -8, 2.0 ** -24


@pytest.fixture(scope="module")
def dk():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import delta_kernels
    delta_kernels.lib()
    return delta_kernels


def inputs(seed, rows, M, dtype, scale=2.0):
    r = np.random.default_rng(seed)

    def rounded(a):
        return torch.tensor(a, dtype=torch.float32).to(dtype).double().numpy()

    return rounded(r.normal(size=(rows, 2 * M)) * scale), rounded(r.normal(size=(rows, M)))


def near(got, ref, terms, dtype):
    bound = 16 * E * terms + (U * np.abs(ref) if dtype == torch.bfloat16 else 0) + 1e-37
    err = np.abs(host(got) - ref)
    assert np.all(err <= bound), f"{(err / bound).max():.2f} of the bound"


def check(dk, h, da, dtype):
    a, codes, exps = dk.swiglu_q8_forward(dev(h, dtype))
    rc, re = lo.q8(h)
    assert np.array_equal(codes.cpu().numpy(), rc) and np.array_equal(exps.cpu().numpy(), re)
    near(a, lo.swiglu(h), np.abs(lo.swiglu(h)) * (1 + np.abs(h[:, :h.shape[1] // 2])), dtype)
    kept = lo.q8_values(rc, re)
    assert np.array_equal(host(dk.q8_values(codes, exps)), kept)
    dh, again = dk.swiglu_q8_backward(codes, exps, dev(da, dtype))
    gate, up = np.split(kept, 2, 1)
    s = 1 / (1 + np.exp(-gate))
    size = 1 + np.abs(gate)  # exp(-x) is off by about |x| e
    terms = np.concatenate([np.abs(da * up) * s * (1 + np.abs(gate)) * size,
                            np.abs(da * gate) * s * size], 1)
    near(dh, lo.swiglu_backward(kept, da), terms, dtype)
    near(again, lo.swiglu(kept), np.abs(lo.swiglu(kept)) * size, dtype)
    dh2, none = dk.swiglu_q8_backward(codes, exps, dev(da, dtype), False)
    assert none is None and torch.equal(dh, dh2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,M", [(1, 1), (1, 8), (3, 31), (3, 32), (5, 33), (17, 40), (9, 64), (4, 100),
                                    (130, 256), (33, 1001)])
def test_sizes(dk, rows, M, dtype):
    h, da = inputs(M, rows, M, dtype)
    check(dk, h, da, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_magnitudes(dk, dtype):
    """Blocks from nothing to the largest values, and the bounds of an exponent."""
    h, da = inputs(1, 12, 32, dtype)
    h[0] = 0
    h[1] *= 1e-38
    h[2] *= 1e-30
    h[3, 0] = 1e30
    h[4, :32] = 127.0
    h[5, :32] = 127.5
    h[6, 32:] = -254.0
    h[7, 32:] = np.arange(32) - 15.5
    h[8, :32] = -88.0
    h[9, :32] = 100.0
    h[10, 32:] = 3e38
    h = torch.tensor(h, dtype=torch.float32).to(dtype).double().numpy()
    da[10] *= 1e-3
    rc, re = lo.q8(h)
    _, codes, exps = dk.swiglu_q8_forward(dev(h, dtype))
    assert np.array_equal(codes.cpu().numpy(), rc) and np.array_equal(exps.cpu().numpy(), re)
    rows = np.r_[0, 2:10]  # results that float32 holds as normal numbers
    check(dk, h[rows], da[rows], dtype)


def test_a_value_that_is_not_finite_stays_in_its_block(dk):
    h, da = inputs(2, 6, 70, torch.float32)
    clean = dk.swiglu_q8_forward(dev(h))
    cdh = dk.swiglu_q8_backward(clean[1], clean[2], dev(da))[0]
    h[1, 40], h[3, 70 + 3], h[4, 69] = np.nan, np.inf, -np.inf
    a, codes, exps = dk.swiglu_q8_forward(dev(h))
    rc, re = lo.q8(h)
    assert np.array_equal(codes.cpu().numpy(), rc) and np.array_equal(exps.cpu().numpy(), re)
    dh, _ = dk.swiglu_q8_backward(codes, exps, dev(da))
    bad = np.zeros((6, 70), bool)
    bad[1, 32:64] = bad[3, :32] = bad[4, 64:] = True
    bad = np.concatenate([bad, bad], 1)
    assert np.array_equal(host(dh)[~bad], host(cdh)[~bad])
    assert np.isnan(host(dh)[:, :70][bad[:, :70]]).all()
    assert np.isnan(host(a)[1, 40]) and np.isfinite(host(a)[1, 41])


def test_no_rows(dk):
    a, codes, exps = dk.swiglu_q8_forward(torch.empty((0, 64), device="cuda"))
    dh, again = dk.swiglu_q8_backward(codes, exps, torch.empty((0, 32), device="cuda"))
    assert a.shape == again.shape == (0, 32) and dh.shape == (0, 64) and exps.shape == (0, 2)


def test_more_than_32_bits_of_values(dk):
    rows, M = (1 << 17) + 3, 1 << 14  # 2^32 and more values of h
    h = torch.randn((1, 2 * M), device="cuda").to(torch.bfloat16).repeat(rows, 1)
    h[-1] = torch.randn(2 * M, device="cuda").to(torch.bfloat16)
    a, codes, exps = dk.swiglu_q8_forward(h)
    ta, tc, te = dk.swiglu_q8_forward(h[-2:].clone())
    assert torch.equal(a[-2:], ta) and torch.equal(codes[-2:], tc) and torch.equal(exps[-2:], te)
    dh, again = dk.swiglu_q8_backward(codes, exps, a)
    td, tg = dk.swiglu_q8_backward(tc, te, ta)
    assert torch.equal(dh[-2:], td) and torch.equal(again[-2:], tg)


def test_buffers_off_16_bytes(dk):
    h, da = inputs(3, 20, 64, torch.bfloat16)

    def off(x):
        t = torch.empty((x.size + 1,), dtype=torch.bfloat16, device="cuda")[1:].view(x.shape)
        return t.copy_(dev(x, torch.bfloat16))

    a, codes, exps = dk.swiglu_q8_forward(dev(h, torch.bfloat16))
    b = dk.swiglu_q8_forward(off(h))
    assert all(torch.equal(x, y) for x, y in zip((a, codes, exps), b))
    for x, y in zip(dk.swiglu_q8_backward(codes, exps, dev(da, torch.bfloat16)),
                    dk.swiglu_q8_backward(codes, exps, off(da))):
        assert torch.equal(x, y)


def test_autograd_is_the_raw_calls(dk):
    h, da = inputs(4, 24, 48, torch.float32)
    x = dev(h).view(4, 6, 96).requires_grad_(True)
    a = dk.swiglu_q8(x)
    (dx,) = torch.autograd.grad(a, x, dev(da).view(4, 6, 48))
    ra, codes, exps = dk.swiglu_q8_forward(dev(h))
    assert torch.equal(a.view(24, 48), ra)
    assert torch.equal(dx.view(24, 96), dk.swiglu_q8_backward(codes, exps, dev(da))[0])
    # an upstream that is one value for all, and an input that is not contiguous
    (dx,) = torch.autograd.grad(dk.swiglu_q8(x.transpose(0, 1)).sum(), x)
    want = dk.swiglu_q8_backward(codes, exps, torch.ones_like(ra))[0]
    assert torch.equal(dx.reshape(24, 96), want)


def test_gradient_is_near_that_of_differences(dk):
    """The gradient at the kept values, which are off by less than 1/127 of a block's largest: the
    first-order change of the gradient over that distance is the bound."""
    h, da = inputs(5, 8, 64, torch.float32, scale=1.0)
    x = dev(h).requires_grad_(True)
    (dx,) = torch.autograd.grad(dk.swiglu_q8(x), x, dev(da))
    d = np.random.default_rng(1).normal(size=h.shape)
    step = 1e-2
    loss = lambda y: (host(dk.swiglu_q8(dev(y))) * da).sum()  # noqa: E731
    want = (loss(h + step * d) - loss(h - step * d)) / (2 * step)
    kept = lo.q8_values(*lo.q8(h))
    slack = np.abs((lo.swiglu_backward(h, da) - lo.swiglu_backward(kept, da)) * d).sum()
    terms = host(dx) * d
    assert abs(want - terms.sum()) <= slack + 2e-3 * np.abs(terms).sum()


def test_refusals(dk):
    h = torch.zeros((4, 64), device="cuda")
    with pytest.raises(ValueError, match="GPU"):
        dk.swiglu_q8_forward(h.cpu())
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        dk.swiglu_q8_forward(h.half())
    with pytest.raises(ValueError, match="2 M"):
        dk.swiglu_q8_forward(h[:, :63])
    with pytest.raises(ValueError, match="2 M"):
        dk.swiglu_q8(h[:, :63])
    with pytest.raises(ValueError, match="contiguous"):
        dk.swiglu_q8_forward(h[:, ::2])
    a, codes, exps = dk.swiglu_q8_forward(h)
    with pytest.raises(ValueError, match="codes"):
        dk.swiglu_q8_backward(codes[:3], exps, a)
    with pytest.raises(ValueError, match="exponents"):
        dk.swiglu_q8_backward(codes, exps[:, :1], a)
    with pytest.raises(ValueError, match="da must"):
        dk.swiglu_q8_backward(codes, exps, a[:, ::2][:, :, None])
