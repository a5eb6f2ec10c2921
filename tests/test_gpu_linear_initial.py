"""Initial states whose rows or columns lie far apart."""
import pytest

torch = pytest.importorskip("torch")

from gpu_util import dev  # noqa: E402
from test_gpu_linear import dk, problem  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("stride", [(1 << 22, 1), (1, 1 << 22), (5, 1 << 23)])
@pytest.mark.parametrize("K,V", [(2, 3), (1, 70)])
def test_far_rows_and_columns(dk, K, V, stride):  # noqa: F811
    p = problem(1, 1, 20, 1, K, V, torch.float32, initial=True)
    q, k, v, do = (dev(p[n]) for n in ("q", "k", "v", "do"))
    g, dense = dev(p["g"]), dev(p["initial"])
    far = torch.zeros((sum(s * n for s, n in zip(stride, (K, V))),), device="cuda") \
        .as_strided((1, 1, K, V), (0, 0) + stride)
    far.copy_(dense)
    a, b = (dk.linear_attention_forward(q, k, v, g, None, None, s) for s in (far, dense))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    da, db = (dk.linear_attention_backward(q, k, v, g, None, None, s, x[2], do)
              for s, x in ((far, a), (dense, b)))
    for x, y in zip(da, db):
        assert torch.equal(x, y)
