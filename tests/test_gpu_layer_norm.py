"""Layer norm against the float64 oracle.

Bounds, fixed before the first run, with e = 2^-24: a sum in the kernels' order has at most 64 roundings
on the way (32 columns of a thread, six lane steps, 16 waves, and the sums' own), so
  y      64 e (|w| r max|x| + |b|): the mean is off by a fraction of max|x|, and so is x - mean
  dx     64 e r (|c| + mean|c| + (|xh| + 1 + r max|x|) mean|c xh| + r max|x| (|c| + mean|c|))
  dw     (64 + rows / 256) e sum |dy| (|xh| + r max|x|),  db the same of |dy|
and half a unit of bf16, 2^-8 |result|, where the result is bf16."""
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


def check(x, w, b, dy, eps, dtype, y, dx, dw, db):
    x, dy = x.reshape(-1, x.shape[-1]), dy.reshape(-1, x.shape[-1])
    ry, mean, inv = lo.layer_norm(x, w, b, eps)
    rdx, rdw, rdb = lo.layer_norm_backward(x, w, eps, dy)
    top = (np.abs(x).max(1) * inv)[:, None]
    xh = np.abs((x - mean[:, None]) * inv[:, None])
    c = np.abs(dy * w)
    mc, mcx = c.mean(1, keepdims=True), (c * xh).mean(1, keepdims=True)
    half = U if dtype == torch.bfloat16 else 0
    bounds = dict(
        y=(y, ry, 64 * E * (np.abs(w) * top + (0 if b is None else np.abs(b))) + half * np.abs(ry)),
        dx=(dx, rdx, 64 * E * inv[:, None] * (c + mc + (xh + 1 + top) * mcx + top * (c + mc))
            + half * np.abs(rdx)))
    n = 64 + len(x) / 256
    bounds["dw"] = (dw, rdw, n * E * (np.abs(dy) * (xh + top)).sum(0))
    if b is not None:
        bounds["db"] = (db, rdb, n * E * np.abs(dy).sum(0))
    for name, (got, ref, bound) in bounds.items():
        got = host(got).reshape(ref.shape)
        err = np.abs(got - ref)
        assert np.all(np.isfinite(got)), name
        assert np.all(err <= bound + 1e-37), f"{name}: {(err / (bound + 1e-37)).max():.2f} of the bound"


def inputs(seed, shape, dtype, offset=0.0):
    r = np.random.default_rng(seed)

    def rounded(a):
        return torch.tensor(a, dtype=torch.float32).to(dtype).double().numpy()

    W = shape[-1]
    f32 = lambda a: a.astype(np.float32).astype(np.float64)  # noqa: E731
    return (rounded(r.normal(size=shape) * 2 + offset), f32(1 + 0.3 * r.normal(size=W)),
            f32(r.normal(size=W)), rounded(r.normal(size=shape)))


def run(dk, x, w, b, dy, eps, dtype):
    tx, tw = dev(x, dtype).requires_grad_(True), dev(w).requires_grad_(True)
    tb = None if b is None else dev(b).requires_grad_(True)
    y = dk.layer_norm(tx, tw, tb, eps)
    grads = torch.autograd.grad(y, [t for t in (tx, tw, tb) if t is not None], dev(dy, dtype))
    return (y,) + tuple(grads) + (() if b is not None else (None,))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("W", [1, 2, 7, 8, 63, 64, 65, 120, 128, 136, 256, 257, 500, 512, 513, 1000, 1024,
                               1025, 2048, 2049, 5003, 8192, 8200, 32768, 32769, 40000])
def test_widths(dk, W, dtype):
    rows = 5 if W > 4000 else 37
    x, w, b, dy = inputs(W, (rows, W), dtype)
    eps = 1e-5
    check(x, w, b, dy, eps, dtype, *run(dk, x, w, b, dy, eps, dtype))


@pytest.mark.parametrize("rows", [1, 2, 3, 31, 33, 511, 513, 4099])
@pytest.mark.parametrize("W", [64, 100, 512])
def test_rows(dk, rows, W):
    """Rows short of a workgroup's, and more than the workgroups of the backward take in one turn."""
    x, w, b, dy = inputs(rows, (rows, W), torch.bfloat16)
    check(x, w, b, dy, 1e-5, torch.bfloat16, *run(dk, x, w, b, dy, 1e-5, torch.bfloat16))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,W", [(200, 8193), (130, 10000), (70, 40001), (33000, 33), (33000, 40)])
def test_rows_beyond_the_partial_sums(dk, rows, W, dtype):
    """More rows than rows of partial sums: wide ones, odd widths and others."""
    x, w, b, dy = inputs(rows, (rows, W), dtype)
    check(x, w, b, dy, 1e-5, dtype, *run(dk, x, w, b, dy, 1e-5, dtype))


@pytest.mark.parametrize("W", [40, 9000, 33000])
def test_gradients_that_nobody_wants(dk, W):
    x, w, b, dy = inputs(3, (70, W), torch.float32)
    x, w, b, dy = dev(x), dev(w), dev(b), dev(dy)
    _, mean, inv = dk.layer_norm_forward(x, w, b)
    dx, dw, db = dk.layer_norm_backward(x, w, mean, inv, dy)
    assert torch.equal(dk.layer_norm_backward(x, w, mean, inv, dy, want_bias=False, want_weight=False)[0], dx)
    only = dk.layer_norm_backward(x, w, mean, inv, dy, want_x=False)
    assert only[0] is None and torch.equal(only[1], dw) and torch.equal(only[2], db)


def test_no_rows(dk):
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.empty((0, 64), dtype=dtype, device="cuda", requires_grad=True)
        w, b = (torch.ones(64, device="cuda", requires_grad=True) for _ in range(2))
        y = dk.layer_norm(x, w, b)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
        assert y.shape == dx.shape == (0, 64) and not dw.any() and not db.any()


def test_without_a_bias(dk):
    x, w, _, dy = inputs(1, (50, 200), torch.float32)
    check(x, w, None, dy, 1e-5, torch.float32, *run(dk, x, w, None, dy, 1e-5, torch.float32))


@pytest.mark.parametrize("W", [64, 1000, 5003])
def test_rows_far_from_zero(dk, W):
    """A mean of 1000 standard deviations: a difference of squares would have nothing left."""
    x, w, b, dy = inputs(2, (20, W), torch.float32, offset=2000.0)
    check(x, w, b, dy, 1e-5, torch.float32, *run(dk, x, w, b, dy, 1e-5, torch.float32))


def test_constant_rows(dk):
    x = np.full((4, 96), 3.25)
    _, w, b, dy = inputs(3, (4, 96), torch.float32)
    y, dx, dw, db = run(dk, x, w, b, dy, 1e-5, torch.float32)
    assert np.array_equal(host(y), np.broadcast_to(b, (4, 96))) and not host(dw).any()
    check(x, w, b, dy, 1e-5, torch.float32, y, dx, dw, db)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("W", [64, 72, 33])
def test_strides(dk, W, dtype):
    """Head outputs read where they lie, a broadcast upstream, every other column."""
    x, w, b, dy = inputs(4, (2, 5, 3, W), dtype)
    big = torch.full((2, 3, 5, 2 * W), float("nan"), dtype=dtype, device="cuda")
    tx = big[..., :W].transpose(1, 2)
    tx.copy_(dev(x, dtype))
    ty = big[..., W:].transpose(1, 2)
    ty.copy_(dev(dy, dtype))
    y, mean, inv = dk.layer_norm_forward(tx, dev(w), dev(b), 1e-5)
    check(x, w, b, dy, 1e-5, dtype, y, *dk.layer_norm_backward(tx, dev(w), mean, inv, ty))
    one = dev(dy[:1, :1, :1], dtype).expand(2, 5, 3, W)
    check(x, w, b, np.broadcast_to(dy[:1, :1, :1], x.shape), 1e-5, dtype, y,
          *dk.layer_norm_backward(tx, dev(w), mean, inv, one))
    odd = torch.empty((2, 5, 3, 2 * W), dtype=dtype, device="cuda")[..., ::2]
    odd.copy_(dev(x, dtype))
    y, mean, inv = dk.layer_norm_forward(odd, dev(w), dev(b), 1e-5)
    check(x, w, b, dy, 1e-5, dtype, y, *dk.layer_norm_backward(odd, dev(w), mean, inv, dev(dy, dtype)))
    deep = odd.unsqueeze(0)  # five axes: flattened
    assert torch.equal(dk.layer_norm(deep, dev(w), dev(b), 1e-5)[0], y)


def test_a_value_that_is_not_finite_stays_in_its_row(dk):
    x, w, b, dy = inputs(5, (70, 64), torch.float32)
    clean = run(dk, x, w, b, dy, 1e-5, torch.float32)
    x[33, 5] = np.inf
    got = run(dk, x, w, b, dy, 1e-5, torch.float32)
    rows = np.arange(70) != 33
    for i in (0, 1):
        assert np.array_equal(host(got[i])[rows], host(clean[i])[rows])
        assert np.isnan(host(got[i])[33]).any()
    assert np.array_equal(host(got[3]), host(clean[3]))


def test_gradient_is_that_of_differences(dk):
    x, w, b, dy = inputs(6, (9, 70), torch.float32)
    _, dx, dw, db = run(dk, x, w, b, dy, 1e-2, torch.float32)
    r = np.random.default_rng(1)

    def loss(x, w, b):
        return (host(dk.layer_norm(dev(x), dev(w), dev(b), 1e-2)) * dy).sum()

    for at, got in ((0, dx), (1, dw), (2, db)):
        p, m = [x, w, b], [x, w, b]
        d, h = r.normal(size=p[at].shape), 1e-2
        p[at], m[at] = p[at] + h * d, m[at] - h * d
        terms = host(got) * d
        assert abs((loss(*p) - loss(*m)) / (2 * h) - terms.sum()) <= 2e-3 * np.abs(terms).sum()


def test_more_than_32_bits_of_values(dk):
    x = torch.randn((1, 4096), device="cuda").to(torch.bfloat16).repeat(1 << 20, 1)  # 2^32 values
    x[-1] = torch.randn(4096, device="cuda").to(torch.bfloat16)
    w, b = torch.rand(4096, device="cuda"), torch.rand(4096, device="cuda")
    y, mean, inv = dk.layer_norm_forward(x, w, b)
    tail, m, i = dk.layer_norm_forward(x[-2:].clone(), w, b)
    assert torch.equal(y[-2:], tail) and torch.equal(mean[-2:], m) and torch.equal(inv[-2:], i)
    dx, _, _ = dk.layer_norm_backward(x, w, mean, inv, y)
    dt, _, _ = dk.layer_norm_backward(x[-2:].clone(), w, m, i, tail)
    assert torch.equal(dx[-2:], dt)


def test_runs_are_equal_bit_for_bit(dk):
    x, w, b, dy = inputs(7, (3000, 512), torch.bfloat16)
    for a, c in zip(run(dk, x, w, b, dy, 1e-5, torch.bfloat16), run(dk, x, w, b, dy, 1e-5, torch.bfloat16)):
        assert torch.equal(a, c)


def test_refusals(dk):
    x, w = torch.zeros((4, 8), device="cuda"), torch.ones(8, device="cuda")
    with pytest.raises(ValueError, match="GPU"):
        dk.layer_norm(x.cpu(), w.cpu())
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        dk.layer_norm(x.half(), w)
    with pytest.raises(ValueError, match="weight"):
        dk.layer_norm(x, w[:7])
    with pytest.raises(ValueError, match="weight"):
        dk.layer_norm(x, w.bfloat16())
    with pytest.raises(ValueError, match="bias"):
        dk.layer_norm(x, w, w[:7])
    with pytest.raises(ValueError, match="W >= 1"):
        dk.layer_norm(x[:, :0], w[:0])
    with pytest.raises(ValueError, match="live on"):
        dk.layer_norm(x, w.cpu())
    y, mean, inv = dk.layer_norm_forward(x, w)
    with pytest.raises(ValueError, match="dy"):
        dk.layer_norm_backward(x, w, mean, inv, x[:3])
    with pytest.raises(ValueError, match="mean"):
        dk.layer_norm_backward(x, w, mean[:3], inv, x)
