"""The linear-attention language model: its operators together, in training and token by token."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lm():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import delta_mixers.linear as lm
    lm.dk.lib()
    return lm


def small(lm, dtype, layers=2, width=96):
    torch.manual_seed(0)
    cfg = lm.LinearLMConfig(vocab=64, d_model=64, layers=layers, heads=4, key_dim=16, value_dim=24,
                            mlp_width=width, compute_dtype=dtype)
    return lm.LinearLM(cfg, device="cuda")


def plain(model, tokens):
    """The model's logits in float64 plain torch."""
    cfg = model.cfg
    H, K, V = cfg.heads, cfg.key_dim, cfg.value_dim
    P = {n: p.double() for n, p in model.named_parameters()}

    def norm(x, n, bias=True):
        c = x - x.mean(-1, keepdim=True)
        y = c / (c.square().mean(-1, keepdim=True) + cfg.norm_epsilon).sqrt() * P[n + ".weight"]
        return y + P[n + ".bias"] if bias else y

    x = P["embed"][tokens]
    B, T = tokens.shape
    t = torch.arange(T, device=tokens.device)
    for i in range(cfg.layers):
        b = f"blocks.{i}."
        q, k, v, gate = (norm(x, b + "norm1") @ P[b + "mixer.in_proj"].t()).split(
            (H * K, H * K, H * V, H * V), -1)
        q, k, v = (y.view(B, T, H, -1).transpose(1, 2) for y in (q * K ** -0.5, k, v))
        g = -torch.nn.functional.softplus(P[b + "mixer.decay"])
        w = torch.exp(g[:, None, None] * (t[:, None] - t[None, :]).clamp(min=0))
        w = w * (t[:, None] >= t[None, :])
        o = norm(((q @ k.transpose(-1, -2) * w) @ v).transpose(1, 2), b + "mixer.norm", False)
        y = o.reshape(B, T, H * V) * torch.nn.functional.silu(gate)
        x = x + y @ P[b + "mixer.out"].t()
        h1, h3 = (norm(x, b + "norm2") @ P[b + "mlp.w13"].t()).chunk(2, -1)
        x = x + (torch.nn.functional.silu(h1) * h3) @ P[b + "mlp.w2"].t()
    return norm(x, "norm") @ P["embed"].t()


def test_logits_are_the_plain_model_s(lm):
    model = small(lm, torch.float32)
    tokens = torch.randint(0, 64, (3, 77), device="cuda")
    ref = plain(model, tokens)
    got = model(tokens).double()
    # two blocks of float32 operators and GEMMs
    assert (got - ref).norm() <= 1e-4 * ref.norm()


def test_gradients_are_the_plain_model_s(lm):
    """But for the MLP's hidden activation in 8 bits: its gradients are off by what 1/127 of a block's
    largest value makes, a few percent at most; those that it does not touch are exact."""
    model = small(lm, torch.float32, layers=1)
    tokens = torch.randint(0, 64, (3, 50), device="cuda")
    up = torch.randn(3, 50, 64, device="cuda")
    (model(tokens) * up).sum().backward()
    got = {n: p.grad.clone().double() for n, p in model.named_parameters()}
    model.zero_grad()
    (plain(model, tokens) * up.double()).sum().backward()
    for n, p in model.named_parameters():
        ref = p.grad.double()
        exact = n in ("norm.weight", "norm.bias")
        tol = 1e-4 if exact else 3e-2
        assert (got[n] - ref).norm() <= tol * ref.norm(), n


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 3e-2)])
def test_tokens_one_by_one_give_the_whole_sequence_s_logits(lm, dtype, tol):
    model = small(lm, dtype)
    tokens = torch.randint(0, 64, (5, 90), device="cuda")
    with torch.no_grad():
        whole = model(tokens).double()
    logits, states = model.prefill(tokens[:, :64])
    assert (logits.double() - whole[:, 63]).norm() <= tol * whole[:, 63].norm()
    logits, states = model.prefill(tokens[:, 64:80], states)  # the prompt's continuation
    assert (logits.double() - whole[:, 79]).norm() <= tol * whole[:, 79].norm()
    for t in range(80, 90):
        logits = model.step(tokens[:, t], states)
        assert (logits.double() - whole[:, t]).norm() <= tol * whole[:, t].norm(), t


def test_documents_and_padding(lm):
    """Packed documents with resets, and padding at the end, give each document's own logits."""
    model = small(lm, torch.float32)
    a, b = (torch.randint(0, 64, (1, n), device="cuda") for n in (40, 70))
    reset = torch.zeros((1, 130), device="cuda")
    reset[0, 40] = 1
    valid = torch.ones((1, 130), device="cuda")
    valid[0, 110:] = 0
    packed = torch.cat([a, b, torch.zeros((1, 20), dtype=torch.long, device="cuda")], 1)
    with torch.no_grad():
        got = model(packed, valid, reset)
        assert torch.allclose(got[:, :40], model(a), rtol=1e-3, atol=1e-3)
        assert torch.allclose(got[:, 40:110], model(b), rtol=1e-3, atol=1e-3)


def test_training_steps_lower_the_loss(lm):
    model = small(lm, torch.bfloat16)
    opt = lm.dk.FusedAdamW(model.parameters(), lr=3e-3)
    tokens = torch.randint(0, 64, (8, 65), device="cuda")
    losses = []
    for _ in range(40):
        opt.zero_grad(set_to_none=True)
        loss = model.loss(tokens)
        loss.backward()
        opt.step()
        losses.append(loss.item())
    assert losses[-1] < 0.7 * losses[0], losses


def test_the_mlp_keeps_8_bits(lm):
    """Bytes that the feed-forward holds between the passes: x, codes and exponents, and no copy of the
    hidden activation."""
    M, rows = 1408, 2048
    mlp = lm.Q8SwiGLU(lm.LinearLMConfig(d_model=256, mlp_width=M), device="cuda")
    x = torch.randn(1, rows, 256, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
        mlp(x)
    weights = sum(t.numel() * t.element_size() for t in saved if t.shape[0] in (2 * M, 256))
    held = sum(t.numel() * t.element_size() for t in saved) - weights
    assert held == rows * (2 * 256 + 2 * M + 2 * M // 32)
