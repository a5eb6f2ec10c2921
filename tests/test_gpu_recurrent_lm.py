"""The recurrent language model: its operators together, in training, in scoring and token by token."""
import pytest

torch = pytest.importorskip("torch")
import torch.utils.checkpoint  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lm():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import delta_mixers.recurrent as lm
    lm.dk.lib()
    return lm


def small(lm, dtype, layers=2):
    torch.manual_seed(0)
    cfg = lm.RecurrentLMConfig(vocab=64, d_model=64, layers=layers, width=72, mlp_width=96, compute_dtype=dtype)
    return lm.RecurrentLM(cfg, device="cuda")


def plain(model, tokens):
    """The model's logits in float64 plain torch."""
    cfg = model.cfg
    P = {n: p.double() for n, p in model.named_parameters()}

    def norm(x, n):
        c = x - x.mean(-1, keepdim=True)
        return c / (c.square().mean(-1, keepdim=True) + cfg.norm_epsilon).sqrt() * P[n + ".weight"] + P[n + ".bias"]

    x = P["embed"][tokens]
    for i in range(cfg.layers):
        b = f"blocks.{i}."
        u, r, gate = (norm(x, b + "norm1") @ P[b + "mixer.in_proj"].t()).chunk(3, -1)
        g = -2 * torch.sigmoid(r) * torch.nn.functional.softplus(P[b + "mixer.decay"])
        h, hs = torch.zeros_like(u[:, 0]), []
        for t in range(tokens.shape[1]):
            h = g[:, t].exp() * h + (1 - (2 * g[:, t]).exp()).sqrt() * u[:, t]
            hs.append(h)
        x = x + (torch.stack(hs, 1) * torch.nn.functional.silu(gate)) @ P[b + "mixer.out"].t()
        h1, h3 = (norm(x, b + "norm2") @ P[b + "mlp.w13"].t()).chunk(2, -1)
        x = x + (torch.nn.functional.silu(h1) * h3) @ P[b + "mlp.w2"].t()
    return norm(x, "norm") @ P["embed"].t()


def test_logits_are_the_plain_model_s(lm):
    model = small(lm, torch.float32)
    tokens = torch.randint(0, 64, (3, 77), device="cuda")
    ref = plain(model, tokens)
    # two blocks of float32 operators and GEMMs
    assert (model(tokens).double() - ref).norm() <= 1e-4 * ref.norm()


def test_gradients_of_a_policy_loss_are_the_plain_model_s(lm):
    """But for the MLP's hidden activation in 8 bits: its gradients are off by what 1/127 of a block's largest
    value makes, a few percent at most; those that it does not touch are exact."""
    model = small(lm, torch.float32, layers=1)
    tokens = torch.randint(0, 64, (3, 50), device="cuda")
    valid = (torch.rand(3, 50, device="cuda") < 0.8).float()
    adv = torch.randn(3, 49, device="cuda")
    loss = model.policy_loss(tokens, adv, valid, 0.1)
    loss.backward()
    got = {n: p.grad.clone().double() for n, p in model.named_parameters()}
    model.zero_grad()
    lp = torch.log_softmax(plain(model, tokens[:, :-1]), -1)
    on = valid[:, 1:].double()
    given = lp.gather(-1, tokens[:, 1:, None])[..., 0]
    ref = -((adv * given * on).sum() - 0.1 * ((lp.exp() * lp).sum(-1) * on).sum()) / on.sum()
    assert abs(float(loss) - float(ref)) <= 1e-5 * (1 + abs(float(ref)))
    ref.backward()
    for n, p in model.named_parameters():
        want = p.grad.double()
        tol = 1e-4 if n in ("norm.weight", "norm.bias") else 3e-2
        assert (got[n] - want).norm() <= tol * want.norm(), n


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


def test_scores_are_the_cross_entropy_s(lm):
    from delta_mixers.linear import LinearLM, LinearLMConfig
    from delta_mixers.model import GdnLM, GdnLMConfig
    tokens = torch.randint(0, 64, (3, 65), device="cuda")
    torch.manual_seed(1)
    models = [small(lm, torch.float32),
              LinearLM(LinearLMConfig(vocab=64, d_model=64, layers=1, heads=2, key_dim=16, value_dim=16, mlp_width=64,
                                      compute_dtype=torch.float32), device="cuda"),
              GdnLM(GdnLMConfig(vocab=64, d_model=128, layers=1, heads=2, mlp_width=64), device="cuda")]
    for model in models:
        with torch.no_grad():
            r, loss = model.score(tokens, top=64), model.loss(tokens)
        assert r.log_probs.shape == (3, 64) and r.top_tokens.shape == (3, 64, 64)
        # bfloat16 logits are the same ones on both sides; the loss is a float32 mean
        assert abs(float(-r.log_probs.double().mean() - loss)) <= 1e-2 * float(loss)
        p = r.top_log_probs.double().exp()
        assert torch.allclose(p.sum(-1), torch.ones_like(p[..., 0]), atol=1e-5)
        assert torch.allclose(-(p * r.top_log_probs).sum(-1), r.entropy.double(), atol=1e-5)
        valid = torch.ones((3, 65), device="cuda")
        valid[1, 30:] = 0
        with torch.no_grad():
            part = model.score(tokens, valid, 2)
        assert torch.equal(part.log_probs[0], r.log_probs[0]) and not part.log_probs[1, 29:].any()
        assert torch.equal(part.top_tokens[2], r.top_tokens[2, :, :2])


def test_a_training_step_of_all_operators(lm):
    """Scan, scores, their gradients and both optimizers in one step: every parameter moves, the matrices by
    their orthogonalised momentum, and the model stays finite."""
    from oracle import recurrent_oracle as ro
    model = small(lm, torch.float32)
    opts = lm.make_optimizers(model, lr=0.01, weight_decay=0.0)
    muon = {id(p) for g in opts[0].param_groups for p in g["params"]}
    names = {n for n, p in model.named_parameters() if id(p) in muon}
    assert names == {f"blocks.{i}.{n}" for i in range(2) for n in ("mixer.in_proj", "mixer.out", "mlp.w13", "mlp.w2")}
    tokens = torch.randint(0, 64, (4, 40), device="cuda")
    adv = torch.randn(4, 39, device="cuda")
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    loss = lm.train_step(model, opts, lambda m: m.policy_loss(tokens, adv, None, 0.01))
    assert torch.isfinite(loss)
    for n, p in model.named_parameters():
        assert torch.isfinite(p).all() and not torch.equal(p, before[n]), n
        if n in names:
            g = p.grad.double().cpu().numpy()
            want, _ = ro.muon(before[n].double().cpu().numpy(), g, 0 * g, 0.01)
            assert abs(p.detach().double().cpu().numpy() - want).max() <= 1e-5, n  # 0.01 of results to 1e-4
    for _ in range(3):
        assert torch.isfinite(lm.train_step(model, opts, lambda m: m.loss(tokens)))


def test_the_example_runs(lm, capsys):
    lm.main(steps=3)
    assert "the prompt" in capsys.readouterr().out


def test_in_inference_mode(lm):
    dk = lm.dk
    with torch.inference_mode():
        x, g = torch.randn(2, 3, 9, 40, device="cuda").unbind()
        g = -g.abs()
        y, fin = dk.gated_recurrence(x, g)
        state = torch.zeros(3, 40, device="cuda")
        one = torch.cat([dk.gated_recurrence_step(state, x[:, t:t + 1], g[:, t:t + 1]) for t in range(9)], 1)
        assert torch.allclose(one, y, rtol=1e-5, atol=1e-6) and torch.allclose(state, fin, rtol=1e-5, atol=1e-6)
        s = dk.token_log_probs(y, torch.zeros(3, 9, device="cuda", dtype=torch.int64), 2)
        assert torch.allclose(s.log_probs, torch.log_softmax(y, -1)[..., 0], rtol=1e-5, atol=1e-5)
        p, m = torch.zeros(2, 20, 30, device="cuda").unbind()
        u = torch.randn(20, 30, device="cuda")
        dk.muon_update(p, u, m, 1.0, nesterov=False)
        assert torch.equal(m, u) and torch.equal(p, -dk.orthogonalize(u))


def test_saved_tensors_moved_and_blocks_made_again(lm):
    """The same gradients where autograd keeps what is saved elsewhere, or runs the forward again."""
    dk = lm.dk
    torch.manual_seed(2)
    x, g = torch.randn(2, 3, 600, 40, device="cuda").unbind()
    x, g = x.requires_grad_(True), (-g.abs()).detach().requires_grad_(True)
    tokens = torch.randint(0, 40, (3, 600), device="cuda")

    def loss(x, g):
        y, fin = dk.gated_recurrence(x, g)
        r = dk.token_log_probs(y, tokens)
        return r.log_probs.sum() + 0.3 * r.entropy.sum() + fin.sum()

    want = torch.autograd.grad(loss(x, g), (x, g))
    with torch.autograd.graph.save_on_cpu():
        moved = loss(x, g)
    again = torch.utils.checkpoint.checkpoint(loss, x, g, use_reentrant=False)
    for other in (moved, again):
        for a, b in zip(want, torch.autograd.grad(other, (x, g))):
            assert torch.equal(a, b)
