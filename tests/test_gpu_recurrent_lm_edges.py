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
