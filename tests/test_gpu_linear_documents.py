"""What is not finite in linear attention stays in its document, across the segments of a long sequence too,
and decays that overflow do no harm to a state that is zero.

Bounds as in test_gpu_linear, with u = 2^-8, e = 2^-24 and A the same result of magnitudes: 2.1 u A for bf16
results, 128 e A for float32 ones, and for dg 256 e max A over the sequence."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from gpu_util import host  # noqa: E402
from test_gpu_linear import compare, dk, oracle, problem, run, sizes, E, U  # noqa: E402,F401

pytestmark = pytest.mark.gpu

DTYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


def packed(seed, dtype, starts, T, V=16):
    p = problem(seed, 1, T, 1, 16, V, dtype, initial=True, final=True)
    p["reset"] = np.zeros((1, T))
    p["reset"][0, list(starts)] = 1
    return p


def same_elsewhere(got, p, dtype, inside):
    """got is the oracle's result of the clean problem p outside the document `inside`."""
    ref, A = oracle(p), sizes(p)
    T = p["q"].shape[1]
    out = np.ones(T, bool)
    out[inside] = False
    for n in ("out", "dq", "dk", "dv", "dg"):
        bound = 256 * E * A[n].max() if n == "dg" else \
            (2.1 * U if dtype == torch.bfloat16 else 128 * E) * A[n][:, out] + 1e-30
        err = np.abs(got[n] - ref[n])[:, out]
        assert np.all(err <= bound), f"{n}: first at {np.argwhere(~(err <= bound))[0]}"
    for n in ("fin", "dinitial"):
        assert np.all(np.abs(got[n] - ref[n]) <= 128 * E * A[n] + 1e-30), n


@DTYPES
@pytest.mark.parametrize("V", [16, 80])
@pytest.mark.parametrize("bad", [np.nan, np.inf, 200.0], ids=["nan", "inf", "overflow"])
@pytest.mark.parametrize("forwards", [True, False], ids=["forward", "backward"])
def test_a_gate_in_a_carried_segment(dk, forwards, bad, V, dtype):  # noqa: F811
    """A gate that is not finite, or grows past float32, in one chunk of a segment of two, and a reset in the
    other: the document behind the reset (forwards), and that before it (backwards), see nothing of it."""
    C = 64 if dtype == torch.bfloat16 else 32
    # segments are two chunks: 4 and 5 are one
    starts = (3 * C + 5, 5 * C + 20, 8 * C + 5) if forwards else (4 * C + 20, 6 * C + 30, 8 * C + 5)
    p = packed(1, dtype, starts, 33 * C - 7, V)
    dirty = dict(p, g=p["g"].copy())
    at = 4 * C + 30 if forwards else 5 * C + 20
    dirty["g"][0, at, 0] = bad
    if bad == 200.0:
        dirty["g"][0, at - 1, 0] = bad  # states of the document, too, pass what float32 holds
    got = run(dk, dirty, dtype)
    first = max(s for s in starts if s <= at)
    last = min(s for s in starts if s > at)
    same_elsewhere(got, p, dtype, np.s_[first:last])


@DTYPES
@pytest.mark.parametrize("V", [16, 80])
@pytest.mark.parametrize("T", [200, 1500])
@pytest.mark.parametrize("cut", [False, True])
def test_growth_of_nothing(dk, cut, T, V, dtype):  # noqa: F811
    """Gates that multiply to more than float32 holds, over tokens where neither a state nor its adjoint is
    there yet: each factor is finite, and zero stays zero."""
    lo_, hi = T // 2 - 60, T // 2 + 60
    p = problem(2, 1, T, 1, 16, V, dtype)
    p["g"][0, lo_:hi, 0] = 2.0
    p["k"][0, :hi] = 0
    p["do"][0, lo_:] = 0
    if cut:
        p["reset"] = np.zeros((1, T))
        p["reset"][0, hi + 3] = 1
    compare(run(dk, p, dtype), p, dtype)


@DTYPES
@pytest.mark.parametrize("V", [16, 80])
def test_pairs_that_overflow_unseen(dk, V, dtype):  # noqa: F811
    """Large values whose product no token sees, since the one comes later than the other or lies in another
    document: it is infinite, and reaches nothing."""
    p = packed(3, dtype, (0, 20, 50), 64, V)
    big = 2.0 ** 70
    for a, b in (("q", "k"), ("do", "v")):
        x = {n: p[n].copy() for n in (a, b)}
        x[a][0, 22], x[b][0, 40] = big * np.sign(p[a][0, 22]), big * np.sign(p[b][0, 40])  # later
        x[a][0, 52], x[b][0, 10] = big * np.sign(p[a][0, 52]), big * np.sign(p[b][0, 10])  # another document
        d = dict(p, **x)
        compare(run(dk, d, dtype), d, dtype)


@DTYPES
@pytest.mark.parametrize("V", [16, 80])
def test_products_with_states_that_overflow_unseen(dk, V, dtype):  # noqa: F811
    """The state before a chunk, or its adjoint behind it, against large values behind, or before, a reset in it."""
    p = packed(4, dtype, (100,), 200, V)
    p["initial"] = p["df"] = None
    p["g"][:] = -0.01
    big = 2.0 ** 70
    for a, b in (("k", "q"), ("v", "do")):  # 10 is in the state before 64, 120 sees none of it
        x = {n: p[n].copy() for n in (a, b)}
        x[a][0, 10], x[b][0, 120] = big * np.sign(p[a][0, 10]), big * np.sign(p[b][0, 120])
        d = dict(p, **x)
        compare(run(dk, d, dtype), d, dtype)
    for a, b in (("q", "k"), ("do", "v")):  # 150 is in the adjoint behind 128, 70 sees none of it
        x = {n: p[n].copy() for n in (a, b)}
        x[a][0, 150], x[b][0, 70] = big * np.sign(p[a][0, 150]), big * np.sign(p[b][0, 70])
        d = dict(p, **x)
        compare(run(dk, d, dtype), d, dtype)


@pytest.mark.parametrize("g,want", [(100.0, "zero"), (300.0, "zero"), (np.inf, "nan"), (np.nan, "nan")])
def test_a_step_that_grows(dk, g, want):  # noqa: F811
    """The step takes gates as the sequence does: a state of zero stays so under a finite gate, one that is there
    grows as far as float32 goes."""
    q = torch.ones((1, 1, 1, 4), device="cuda")
    k = torch.zeros_like(q)
    gate = torch.full((1, 1, 1), g, device="cuda")
    state = torch.zeros((1, 1, 4, 4), device="cuda")
    state[0, 0, 0, 0] = 1e-38
    out = host(dk.linear_attention_step(state, q, k, q, gate))
    seq, fin = dk.linear_attention(q, k, q, gate, None, None, torch.zeros_like(state))
    if want == "nan":
        assert np.isnan(out).all() and torch.isnan(seq).all() and torch.isnan(fin).all()
        return
    assert np.all(out[..., 1:] == 0) and torch.all(seq == 0) and torch.all(fin == 0)
    grown = 1e-38 * np.exp(min(g, 700.0))
    assert out[0, 0, 0, 0] == np.inf if grown > 3.4e38 else abs(out[0, 0, 0, 0] - grown) <= 1e-4 * grown


@DTYPES
@pytest.mark.parametrize("V", [16, 80])
def test_a_gate_inside_one_chunk(dk, V, dtype):  # noqa: F811
    """A document inside one chunk, with a gate that is NaN: the gradients of its gates are, and no others."""
    p = packed(6, dtype, (5, 25), 32, V)
    p["g"] = p["g"].copy()
    clean = dict(p, g=p["g"].copy())
    p["g"][0, 15, 0] = np.nan
    got = run(dk, p, dtype)
    same_elsewhere(got, clean, dtype, np.s_[5:25])
    assert np.isnan(got["dg"][0, 6:25]).all()
    assert np.isnan(got["out"][0, 15:25]).all()
