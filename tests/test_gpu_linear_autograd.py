"""Derivatives that the linear-attention block's operators do not have are refused, not dropped."""
import pytest

torch = pytest.importorskip("torch")
fwAD = pytest.importorskip("torch.autograd.forward_ad")

from test_gpu_linear import dk  # noqa: E402,F401

pytestmark = pytest.mark.gpu


def inputs(K=16, V=8, T=6):
    r = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn((2, T, 3, n), generator=r, device="cuda") for n in (K, K, V))
    return q, k, v, -torch.rand((2, T, 3), generator=r, device="cuda")


def operators(dk):  # noqa: F811
    """Name, call of one tensor, that tensor."""
    q, k, v, g = inputs()
    w = torch.ones((16,), device="cuda")
    return (("linear_attention", lambda x: dk.linear_attention(x, k, v, g)[0], q),
            ("its decay", lambda x: dk.linear_attention(q, k, v, x)[0], g),
            ("layer_norm", lambda x: dk.layer_norm(x, w), q),
            ("its weight", lambda x: dk.layer_norm(q, x), w),
            ("swiglu_q8", dk.swiglu_q8, q))


def test_forward_mode_is_refused(dk):  # noqa: F811
    for name, call, x in operators(dk):
        with fwAD.dual_level():
            with pytest.raises((RuntimeError, NotImplementedError)):
                call(fwAD.make_dual(x, torch.ones_like(x)))
                pytest.fail(name)
            call(x)  # without a tangent it runs


def penalty(y, x):
    """A loss that has the gradient of another one in it."""
    (d,) = torch.autograd.grad((y ** 2).sum(), x, create_graph=True)
    return y.sum() + (d ** 2).sum()


def test_second_derivatives_are_refused(dk):  # noqa: F811
    for name, call, x in operators(dk):
        x = x.clone().requires_grad_(True)
        loss = penalty(call(x), x)
        with pytest.raises(RuntimeError, match="twice"):
            loss.backward()
            pytest.fail(name)


def test_second_derivatives_of_the_mlp_are_refused(dk):  # noqa: F811
    from delta_mixers.linear import LinearLMConfig, Q8SwiGLU
    mlp = Q8SwiGLU(LinearLMConfig(d_model=16, mlp_width=32), device="cuda")
    x = torch.randn((4, 16), device="cuda", requires_grad=True)
    loss = penalty(mlp(x), x)
    with pytest.raises(RuntimeError, match="twice"):
        loss.backward()
