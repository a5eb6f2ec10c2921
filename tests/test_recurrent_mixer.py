"""The recurrent mixer's gates at their ends (CPU: plain torch operations)."""
import pytest

torch = pytest.importorskip("torch")


def mixer(width=6):
    from delta_mixers.recurrent import RecurrentLMConfig, RecurrentMixer
    m = RecurrentMixer(RecurrentLMConfig(vocab=8, d_model=3, layers=1, width=width, mlp_width=8))
    with torch.no_grad():
        m.in_proj.zero_()
        m.in_proj[:width, 1] = torch.linspace(-1, 1, width)  # u from the second column
        m.in_proj[width:2 * width, 0] = 1.0  # r is the first column
    return m


@pytest.mark.parametrize("closed", ["gate", "rate"])
def test_gates_that_are_closed(closed):
    """A log decay of 0 (the state stays, nothing comes in): the gradients of a float64 mixer with a gate that is
    open by what float32 cannot hold are 0 there, and so are those of the closed gate."""
    m = mixer()
    r = torch.tensor([-110.0, 110.0, 0.3, -2.0])
    if closed == "rate":
        with torch.no_grad():
            m.decay[2] = -120.0
    x = torch.stack([r, torch.tensor([1.0, 0.5, -1.0, 2.0]), torch.zeros(4)], -1)[None].requires_grad_(True)
    u, g, _ = m._split(x)
    assert not u[0, 0].any() and not g[0, 0].any() and u[0, 1:, 0].all()
    params = [x, m.in_proj, m.decay]
    got = torch.autograd.grad(u.sum() + (g * torch.arange(1.0, 7)).sum(), params)
    wide = [p.detach().double().requires_grad_(True) for p in params]
    wx, w, decay = wide
    uu, rr, _ = (wx @ w.t()).chunk(3, -1)
    gg = -2 * torch.sigmoid(rr) * torch.nn.functional.softplus(decay)
    want = torch.autograd.grad((torch.sqrt(-torch.expm1(2 * gg)) * uu).sum()
                               + (gg * torch.arange(1.0, 7).double()).sum(), wide)
    for a, b in zip(got, want):
        # a dozen float32 operations, of gradients up to b's largest; sqrt(exp(-110)) is 1e-24
        assert torch.isfinite(a).all() and (a - b).abs().max() <= 2.0 ** -20 * b.abs().max()


def test_values_are_those_without_care():
    m = mixer(40)
    x = torch.randn(3, 50, 3)
    u, g, _ = m._split(x)
    uu = (x @ m.in_proj.t())[..., :40]
    assert torch.equal(u, torch.sqrt(-torch.expm1(2 * g)) * uu)
