"""The gradient of one decay a head, summed over very many tokens.

The bound: the sum's own rounding, and 32 e of the sum of magnitudes for the order of its terms (64 lanes, 16 waves
and eight more doublings), e = 2^-24."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_linear import dk, E  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,T,H", [(1 << 19, 1, 1), (3, 4001, 5), (1 << 10, 70, 20)])
def test_the_sum_of_many_equal_ones(dk, B, T, H):  # noqa: F811
    """Every sequence is the same, so that roundings of a running sum all fall the same way."""
    r = torch.Generator(device="cuda").manual_seed(B)

    def one(*size):
        x = torch.randn((1,) + size, generator=r, device="cuda")
        return x.expand((B,) + size)

    q, k, v, do = one(T, H, 2), one(T, H, 2), one(T, H, 2), one(T, H, 2)
    initial = one(H, 2, 2)
    g = -torch.rand((H,), generator=r, device="cuda")
    ck = dk.linear_attention_forward(q, k, v, g, None, None, initial)[2]
    heads = dk.linear_attention_backward(q, k, v, g, None, None, initial, ck, do)[3]
    each = dk.linear_attention_backward(q, k, v, g.expand(B, T, H), None, None, initial, ck, do)[3]
    want = each.double().sum((0, 1))
    size = each.double().abs().sum((0, 1))
    assert ((heads.double() - want).abs() <= 32 * E * size).all(), \
        float(((heads.double() - want).abs() / (E * size)).max())
