"""Short linear-attention calls take the form of long ones: a few tokens have the same bits as with padding
behind them."""
import pytest

torch = pytest.importorskip("torch")

from gpu_util import dev  # noqa: E402
from test_gpu_linear import dk, problem  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T", [1, 2, 4, 5])
@pytest.mark.parametrize("K,V", [(64, 64), (24, 100)])
def test_padding_behind_changes_nothing(dk, K, V, T, dtype):  # noqa: F811
    p = problem(T, 2, 9, 3, K, V, dtype, initial=True, final=True)
    valid = torch.zeros((2, 9), device="cuda")
    valid[:, :T] = 1
    initial, df = dev(p["initial"]), dev(p["df"])

    def call(n, valid):
        q, k, v, do = (dev(p[m][:, :n], dtype) for m in ("q", "k", "v", "do"))
        g = dev(p["g"][:, :n])
        out, fin, ck = dk.linear_attention_forward(q, k, v, g, valid, None, initial)
        return (out, fin) + dk.linear_attention_backward(q, k, v, g, valid, None, initial, ck, do, df)

    names = ("out", "final", "dq", "dk", "dv", "dg", "dinitial")
    for name, a, b in zip(names, call(T, None), call(9, valid)):
        assert torch.equal(a, b if a.dim() == 4 and a.shape[1] == 3 else b[:, :T]), name
