"""The recurrent language model at the ends of what it is called with."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_recurrent_lm import lm, small  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_a_training_step_with_gates_that_are_closed(lm, dtype):  # noqa: F811
    model = small(lm, dtype)
    with torch.no_grad():
        for b in model.blocks:
            b.mixer.in_proj[72:144] *= 1000  # r of both signs, far past where its sigmoid is 0
            b.mixer.decay[3] = -120.0
    tokens = torch.randint(0, 64, (4, 40), device="cuda")
    opts = lm.make_optimizers(model)
    x = model.blocks[0].norm1(model.embed[tokens]).to(dtype)
    assert (model.blocks[0].mixer._split(x)[1][..., 4:] == 0).any()
    for _ in range(2):
        assert torch.isfinite(lm.train_step(model, opts, lambda m: m.loss(tokens)))
        for n, p in model.named_parameters():
            assert torch.isfinite(p.grad).all() and torch.isfinite(p).all(), n


def linear(lm):  # noqa: F811
    from delta_mixers.linear import LinearLM, LinearLMConfig
    torch.manual_seed(1)
    return LinearLM(LinearLMConfig(vocab=64, d_model=64, layers=2, heads=2, key_dim=16, value_dim=16, mlp_width=64,
                                   compute_dtype=torch.float32), device="cuda")


def batch(boolean):
    """Documents a, b, c: two packed in a row that is padded at its end, one in a row padded before and after."""
    a, b, c = (torch.randint(0, 64, (1, n), device="cuda") for n in (31, 50, 64))
    tokens = torch.randint(0, 64, (2, 90), device="cuda")
    present, reset = torch.zeros(2, 2, 90, device="cuda").unbind()
    tokens[0, :31], tokens[0, 31:81], tokens[1, 13:77] = a[0], b[0], c[0]
    present[0, :81], present[1, 13:77], reset[0, 31], reset[0, 0] = 1, 1, 1, 1
    places = ((a, 0, 0), (b, 0, 31), (c, 1, 13))
    return tokens, places, (present.bool(), reset.bool()) if boolean else (present, reset)


@pytest.mark.parametrize("kind", ["recurrent", "linear"])
def test_padded_and_packed_documents_score_like_each_alone(lm, kind):  # noqa: F811
    model = small(lm, torch.float32) if kind == "recurrent" else linear(lm)
    tokens, places, (present, reset) = batch(kind == "linear")
    with torch.no_grad():
        got = model.score(tokens, None, 3, 0.8, present, reset)
        rest = torch.ones(2, 89, dtype=torch.bool, device="cuda")
        for doc, row, at in places:
            want, here = model.score(doc, None, 3, 0.8), slice(at, at + doc.shape[1] - 1)
            for name in ("log_probs", "entropy", "top_log_probs"):
                assert torch.allclose(getattr(got, name)[row, here], getattr(want, name)[0], rtol=1e-3, atol=1e-3)
            rest[row, here] = False
        for v in got:
            assert not v[rest].any()
        valid = (torch.rand(2, 90, device="cuda") < 0.5).float()
        some = model.score(tokens, valid, 0, 0.8, present, reset).log_probs
        assert torch.equal(some, got.log_probs * valid[:, 1:])
        only = model.score(tokens, None, 0, 0.8, None, reset).log_probs
        assert torch.equal(only[0, :80], got.log_probs[0, :80]) and only[1].all()


def test_a_policy_loss_of_padded_and_packed_documents(lm):  # noqa: F811
    """Is that of the documents alone, with its gradients: but for the MLP's hidden activation in 8 bits, a few
    percent, as in test_gpu_recurrent_lm."""
    model = small(lm, torch.float32, layers=1)
    tokens, places, (present, reset) = batch(False)
    adv = torch.randn(2, 89, device="cuda")
    loss = model.policy_loss(tokens, adv, None, 0.1, present, reset)
    loss.backward()
    got = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad()
    total, n = 0.0, 0
    for doc, row, at in places:
        k = doc.shape[1] - 1
        total, n = total + k * model.policy_loss(doc, adv[row:row + 1, at:at + k], None, 0.1), n + k
    (total / n).backward()
    assert abs(float(loss) - float(total / n)) <= 1e-4 * (1 + abs(float(loss)))
    for name, p in model.named_parameters():
        tol = 1e-4 if name in ("norm.weight", "norm.bias") else 3e-2
        assert (got[name] - p.grad).norm() <= tol * p.grad.norm(), name
