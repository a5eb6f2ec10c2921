"""Derivatives that the linear-attention block's operators do not have are refused, not dropped, and a state that
a step changes in place is known to have changed."""
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


def test_a_step_on_a_state_that_a_backward_needs(dk):  # noqa: F811
    q, k, v, g = inputs(K=100)
    state = torch.randn((2, 3, 100, 8), device="cuda")
    q.requires_grad_(True)
    out, _ = dk.linear_attention(q, k, v, g, None, None, state)
    with torch.no_grad():
        dk.linear_attention_step(state, q[:, :1], k[:, :1], v[:, :1], g[:, :1])
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()


@pytest.mark.parametrize("which", ["state", "q", "k", "v", "g"])
def test_a_step_has_no_gradient(dk, which):  # noqa: F811
    q, k, v, g = (x[:, :1].clone() for x in inputs())
    x = dict(state=torch.zeros((2, 3, 16, 8), device="cuda"), q=q, k=k, v=v, g=g)
    x[which].requires_grad_(True)
    with pytest.raises(ValueError, match="no gradient"):
        dk.linear_attention_step(**x)
    with torch.no_grad():
        dk.linear_attention_step(**x)


def test_a_step_in_inference_mode(dk):  # noqa: F811
    with torch.inference_mode():
        q, k, v, g = (x[:, :1].clone() for x in inputs())
        a, b = torch.zeros((2, 2, 3, 16, 8), device="cuda").unbind()
        out = dk.linear_attention_step(a, q, k, v, g)
        seq, fin = dk.linear_attention(q, k, v, g, None, None, b)
    assert torch.allclose(out, seq, rtol=1e-5, atol=1e-6) and torch.allclose(a, fin, rtol=1e-5, atol=1e-6)


def test_a_step_in_forward_mode(dk):  # noqa: F811
    q, k, v, g = (x[:, :1].clone() for x in inputs())
    state = torch.zeros((2, 3, 16, 8), device="cuda")
    with fwAD.dual_level():
        dk.linear_attention_step(state, q, k, v, g)  # without a tangent it runs
        with pytest.raises(ValueError, match="no gradient"):
            dk.linear_attention_step(state, fwAD.make_dual(q, torch.ones_like(q)), k, v, g)
