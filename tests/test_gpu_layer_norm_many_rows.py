"""Layer norm's parameter gradients over many rows, at and off 16-byte addresses: those read by elements are added
up in more parts.

With e = 2^-24 a sum in the kernels' order has (64 + rows / 256) roundings at most, and x - mean is off by 64 e of the
row's largest value: (128 + rows / 256) e of the sum of magnitudes."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_layer_norm import dk, E  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("W", [20, 24, 1028])
@pytest.mark.parametrize("off", [0, 1])
def test_many_rows(dk, off, W, dtype):  # noqa: F811
    rows = 33000
    r = torch.Generator(device="cuda").manual_seed(W)
    x, dy = (torch.randn((rows * W + off,), generator=r, device="cuda").to(dtype)[off:].view(rows, W)
             for _ in range(2))
    w = torch.randn((W,), generator=r, device="cuda")
    _, mean, inv = dk.layer_norm_forward(x, w)
    _, dw, db = dk.layer_norm_backward(x, w, mean, inv, dy)
    _, again, _ = dk.layer_norm_backward(x, w, mean, inv, dy)
    assert torch.equal(dw, again)
    xd, dyd = x.double(), dy.double()
    var, m = torch.var_mean(xd, -1, correction=0, keepdim=True)
    xh = (xd - m) / (var + 1e-5).sqrt()
    top = (xd.abs().amax(-1, keepdim=True) / (var + 1e-5).sqrt())
    n = 128 + rows / 256
    assert ((dw.double() - (dyd * xh).sum(0)).abs() <= n * E * (dyd.abs() * (xh.abs() + top)).sum(0)).all()
    assert ((db.double() - dyd.sum(0)).abs() <= n * E * dyd.abs().sum(0)).all()
