"""The gate's gradient at every token, next to others of very different size.

dg_t is a sum over the pairs of tokens (and states) that span t.  The bound is what spans t alone: with e = 2^-24 and
A_t the same sum of magnitudes, 512 e A_t: 128 e for the states on either side, the rest for the decays and sums
in between."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_linear import dk, oracle, problem, run, sizes, E  # noqa: E402,F401

pytestmark = pytest.mark.gpu

DTYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
WIDTHS = pytest.mark.parametrize("K,V", [(64, 64), (16, 72), (96, 24), (128, 128)])


def check(dk, p, dtype):  # noqa: F811
    got, ref, A = run(dk, p, dtype)["dg"], oracle(p)["dg"], sizes(p)["dg"]
    bound = 512 * E * A + 1e-30
    err = np.abs(got - ref)
    worst = np.argmax(err / bound)
    assert np.all(err <= bound), f"{float((err / bound).max()):.3g} of the bound at {worst}"


@DTYPES
@WIDTHS
def test_a_large_state_that_fades(dk, K, V, dtype):  # noqa: F811
    p = problem(1, 1, 500, 1, K, V, dtype, initial=True, final=True)
    p["initial"] *= 1e4
    p["g"][:] = -0.5
    check(dk, p, dtype)


@DTYPES
@WIDTHS
@pytest.mark.parametrize("T", [500, 1500])
@pytest.mark.parametrize("after", [True, False])
def test_a_strong_decay_between_regions(dk, after, T, K, V, dtype):  # noqa: F811
    """exp(-30), which is no cut, between tokens of size 1 and tokens of size 100."""
    p = problem(2, 2, T, 1, K, V, dtype, slow=True)
    at = T - 100 if after else 100
    p["g"][:, at] = -30.0
    large = np.s_[:, at:] if after else np.s_[:, :at]
    for n in ("v", "do"):
        p[n] = p[n].copy()
        p[n][large] = torch.tensor(p[n][large] * 100).to(dtype).double().numpy()
    check(dk, p, dtype)
