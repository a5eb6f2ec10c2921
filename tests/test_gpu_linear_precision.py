"""bf16 linear attention against float32 arithmetic whose result alone is rounded.

Bounds, fixed before the first run.  With u = 2^-8 (a rounding to bf16), e = 2^-24 and A the same result with
every input replaced by its magnitude: the result's own rounding u |result|, and for the operands, of which
each term of a sum meets one that is not exact, two bf16 terms of it, 2^-16 A, with float32 sums of 128 e A = 2^-17 A:
together 2^-15 A."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from gpu_util import dev, host  # noqa: E402
from test_gpu_linear import dk, oracle, problem, run, sizes  # noqa: E402,F401

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
BF16 = torch.bfloat16
WIDTHS = [(16, 24), (64, 64), (33, 40), (70, 9), (64, 128), (128, 128)]


def rounded_once(got, p):
    ref, A = oracle(p), sizes(p)
    for n in ("out", "dq", "dk", "dv"):
        bound = U * np.abs(ref[n]) + 2.0 ** -15 * A[n] + 1e-30
        err = np.abs(got[n] - ref[n])
        assert np.all(err <= bound), f"{n}: {float((err / bound).max()):.2f} of the bound"


@pytest.mark.parametrize("K,V", WIDTHS)
def test_only_the_result_is_rounded(dk, K, V):  # noqa: F811
    p = problem(K + V, 1, 150, 2, K, V, BF16, masks=True, initial=True, final=True)
    rounded_once(run(dk, p, BF16), p)


@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 6, 7, 8, 16, 65])
@pytest.mark.parametrize("K,V", [(64, 64), (128, 16)])
def test_in_short_sequences_too(dk, K, V, T):  # noqa: F811
    p = problem(T, 3, T, 2, K, V, BF16, initial=True, final=True)
    rounded_once(run(dk, p, BF16), p)


@pytest.mark.parametrize("K,V", [(12, 9), (70, 9), (16, 100)])
def test_in_segments(dk, K, V):  # noqa: F811
    p = problem(5, 1, 1100, 1, K, V, BF16, masks=True, initial=True, final=True, slow=True)
    rounded_once(run(dk, p, BF16), p)


@pytest.mark.parametrize("T", [3, 200, 1100])
@pytest.mark.parametrize("K,V", [(16, 16), (66, 16), (32, 80), (128, 128)])
def test_gradients_do_not_depend_on_those_that_are_wanted(dk, K, V, T):  # noqa: F811
    """The same bits, whichever of them are computed: those of a frozen decay among them."""
    p = problem(14, 1, T, 2, K, V, BF16, masks=T > 3, initial=True, final=True)
    x = [dev(p[n], BF16) for n in ("q", "k", "v")]
    x += [dev(p[n]) for n in ("g", "valid", "reset", "initial")]
    ck = dk.linear_attention_forward(*x)[2]
    up = dev(p["do"], BF16), dev(p["df"])
    all_of_them = dk.linear_attention_backward(*x, ck, *up)
    for wanted in ((True, True, True, False, True), (True, False, False, False, False),
                   (False, True, False, False, False), (False, False, True, False, False),
                   (False, False, False, True, False)):
        some = dk.linear_attention_backward(*x, ck, *up, wanted)
        for w, a, b in zip(wanted, all_of_them, some):
            assert torch.equal(a, b) if w else b is None, wanted
    assert np.isfinite(host(all_of_them[3])).all()
