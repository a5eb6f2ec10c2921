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


def models(device=None):
    from delta_mixers.linear import LinearLM, LinearLMConfig
    from delta_mixers.model import GdnLM, GdnLMConfig
    from delta_mixers.recurrent import RecurrentLM, RecurrentLMConfig
    return [RecurrentLM(RecurrentLMConfig(vocab=64, d_model=64, layers=2, width=40, mlp_width=64), device),
            LinearLM(LinearLMConfig(vocab=64, d_model=64, layers=2, heads=2, key_dim=16, value_dim=16, mlp_width=64),
                     device),
            GdnLM(GdnLMConfig(vocab=64, d_model=128, layers=2, heads=2, mlp_width=64), device)]


@pytest.mark.parametrize("which", range(3))
def test_what_muon_takes_of_the_models(which):
    from delta_mixers.recurrent import make_optimizers
    model = models()[which]
    names = {id(p): n for n, p in model.named_parameters()}
    muon, adamw = ({names[id(p)] for g in o.param_groups for p in g["params"]} for o in make_optimizers(model))
    assert muon == {f"blocks.{i}.{n}" for i in range(2) for n in ("mixer.in_proj", "mixer.out", "mlp.w13", "mlp.w2")}
    assert adamw == set(names.values()) - muon


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(3))
def test_both_optimizers_train_each_model(which):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from delta_mixers.recurrent import make_optimizers, train_step
    torch.manual_seed(0)
    model = models("cuda")[which]
    opts = make_optimizers(model)
    tokens = torch.randint(0, 64, (4, 65), device="cuda")
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    for _ in range(2):
        assert torch.isfinite(train_step(model, opts, lambda m: m.loss(tokens)))
    for n, p in model.named_parameters():
        assert torch.isfinite(p).all() and not torch.equal(p, before[n]), n


def test_the_same_values_without_gradients():
    m = mixer()
    x = torch.tensor([-110.0, -3.0, 110.0, 0.0, 1.0, 0.2]).view(1, 6, 1) * torch.ones(3)
    with torch.no_grad():
        alone = m._split(x)
    assert all(torch.equal(a, b) for a, b in zip(alone, m._split(x)))
