"""Linear attention with a decay for each head, and its step, against the float64 oracle.

Bounds, fixed before the first run.  With u = 2^-8 (bf16: eight significant bits) and e = 2^-24 (float32), A the same result
with every input replaced by its magnitude (all terms added up):
  bf16 results  the pairs' weights or the state are rounded once, and the result: 2.1 u A
  float32 results (also of bf16 inputs: those products are exact)  128 e A: sums of up to 64 terms in
                a chunk and a few tens of chunks, and decays off by a few units
  dg            additions and subtractions of sums over a segment: 256 e max A over the sequence"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import linear_oracle as lo  # noqa: E402
from gpu_util import dev, host  # noqa: E402

pytestmark = pytest.mark.gpu

U, E = 2.0 ** -8, 2.0 ** -24


@pytest.fixture(scope="module")
def dk():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import delta_kernels
    delta_kernels.lib()
    return delta_kernels


def problem(seed, B, T, H, K, V, dtype, masks=False, head_decay=False, initial=False, final=False,
            slow=False):
    r = np.random.default_rng(seed)

    def rounded(x):
        return torch.tensor(x, dtype=torch.float32).to(dtype).double().numpy()

    p = dict(q=rounded(r.normal(size=(B, T, H, K))), k=rounded(r.normal(size=(B, T, H, K)) / 4),
             v=rounded(r.normal(size=(B, T, H, V))), do=rounded(r.normal(size=(B, T, H, V))))
    g = -np.exp(r.normal(size=(H,) if head_decay else (B, T, H)) * 1.5 - (6 if slow else 2))
    p["g"] = g.astype(np.float32).astype(np.float64)
    p["valid"] = p["reset"] = p["initial"] = p["df"] = None
    if masks:
        p["valid"] = (r.random((B, T)) > 0.2).astype(np.float64)
        p["valid"][0, T - T // 3:] = 0
        if B > 1:
            p["valid"][1] = 0  # a sequence of padding alone
        p["reset"] = (r.random((B, T)) < 0.05).astype(np.float64)
    if initial:
        p["initial"] = r.normal(size=(B, H, K, V)).astype(np.float32).astype(np.float64)
    if final:
        p["df"] = r.normal(size=(B, H, K, V)).astype(np.float32).astype(np.float64)
    return p


def oracle(p):
    B, T, H, _ = p["q"].shape
    g = np.broadcast_to(p["g"], (B, T, H))
    out, fin, _ = lo.attention(p["q"], p["k"], p["v"], g, p["valid"], p["reset"], p["initial"])
    grads = lo.attention_backward(p["q"], p["k"], p["v"], g, p["valid"], p["reset"], p["initial"],
                                  p["do"], p["df"])
    return dict(out=out, fin=fin, **grads)


def sizes(p):
    """The same with magnitudes: what the bounds scale with."""
    return oracle({n: np.abs(x) if n in ("q", "k", "v", "do", "initial", "df") and x is not None
                   else x for n, x in p.items()})


def run(dk, p, dtype, x=None):
    x = x or {n: dev(p[n], dtype) for n in ("q", "k", "v")}
    leaves = {n: x[n].requires_grad_(True) for n in x}
    g = dev(p["g"]).requires_grad_(True)
    init = dev(p["initial"])
    if init is not None:
        init.requires_grad_(True)
    out, fin = dk.linear_attention(x["q"], x["k"], x["v"], g, dev(p["valid"]), dev(p["reset"]),
                                   init)
    outs, ups = [out], [dev(p["do"], dtype)]
    if p["df"] is not None:
        outs.append(fin)
        ups.append(dev(p["df"]))
    ins = [leaves["q"], leaves["k"], leaves["v"], g] + ([] if init is None else [init])
    grads = torch.autograd.grad(outs, ins, ups)
    res = dict(out=out, fin=fin, **dict(zip(("dq", "dk", "dv", "dg", "dinitial"), grads)))
    return {n: host(t) for n, t in res.items()}


def compare(got, p, dtype, names=None):
    ref, A = oracle(p), sizes(p)
    if p["g"].ndim == 1:
        for r in (ref, A):
            r["dg"] = r["dg"].sum((0, 1))
    for n in names or got:
        a = A[n]
        if n == "dg":
            bound = 256 * E * (a.max((0, 1), keepdims=True) if a.ndim == 3 else a)
        elif dtype == torch.bfloat16 and n not in ("fin", "dinitial"):
            bound = 2.1 * U * a
        else:
            bound = 128 * E * a
        assert got[n].shape == ref[n].shape, n
        err = np.abs(got[n] - ref[n])
        assert np.all(np.isfinite(got[n])), n
        worst = float((err / (bound + 1e-30)).max())
        assert np.all(err <= bound + 1e-30), f"{n}: {worst:.3f} of the bound"
    if p["valid"] is not None:
        pad = p["valid"] == 0
        for n in ("out", "dq", "dk", "dv"):
            assert np.all(got[n][pad] == 0), n


LENGTHS = [1, 2, 31, 32, 33, 63, 64, 65, 127, 129, 200]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T", LENGTHS)
def test_lengths(dk, T, dtype):
    p = problem(T, 2, T, 2, 16, 24, dtype, masks=T > 2, initial=T % 2 == 1, final=T % 3 == 0)
    compare(run(dk, p, dtype), p, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("K,V", [(1, 1), (8, 5), (33, 40), (64, 64), (65, 64), (64, 128), (128, 64),
                                 (127, 128), (128, 128)])
def test_widths(dk, K, V, dtype):
    p = problem(K + V, 1, 150, 2, K, V, dtype, masks=True, initial=True, final=True)
    compare(run(dk, p, dtype), p, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("head_decay", [False, True])
@pytest.mark.parametrize("masks", [False, True])
@pytest.mark.parametrize("K,V", [(12, 9), (70, 9)])
def test_segments_of_long_sequences(dk, K, V, masks, head_decay, dtype):
    """One sequence is cut into many segments; memories longer than a segment."""
    p = problem(5, 1, 1100, 1, K, V, dtype, masks=masks, head_decay=head_decay, initial=True,
                final=True, slow=True)
    compare(run(dk, p, dtype), p, dtype)


def test_many_sequences_in_one_segment(dk):
    p = problem(6, 40, 70, 16, 4, 4, torch.float32, masks=True)
    compare(run(dk, p, torch.float32), p, torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("V", [8, 72])
def test_gates_at_their_limits(dk, V, dtype):
    """Decays of 0 (-inf, and far below what exp holds), of 1, growth, and a reset at every token."""
    p = problem(7, 1, 140, 2, 8, V, dtype, masks=True, initial=True, final=True)
    g = p["g"]
    g[0, 10, 0], g[0, 70, 1], g[0, 100, 0] = -np.inf, -500.0, -104.0
    g[0, 20:60, 1] = 0.0
    g[0, 61:66, 0] = 0.25
    compare(run(dk, p, dtype), p, dtype)
    p["reset"][:] = 1
    got = run(dk, p, dtype)
    compare(got, p, dtype)
    assert np.all(got["dg"] == 0)


def test_strong_and_weak_decays_side_by_side(dk):
    """Sums of the gates that float32 could not hold next to each other: -100 and -1e-4."""
    p = problem(8, 1, 96, 1, 4, 4, torch.float32)
    p["g"][0, :, 0] = np.where(np.arange(96) % 3 == 0, -100.0, -1e-4).astype(np.float32)
    compare(run(dk, p, torch.float32), p, torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_strides(dk, dtype):
    """Heads before time, every other channel, rows off 16 bytes, and one k and v for all heads: the
    gradient of a broadcast input is the sum over what it was broadcast to."""
    p = problem(9, 2, 90, 4, 24, 16, dtype, masks=True)
    p["v"][:] = p["v"][:, :, :1]
    p["k"][:] = p["k"][:, :, :1]
    t = {n: dev(p[n], dtype) for n in ("q", "k", "v")}
    q = torch.empty((2, 4, 90, 48), dtype=dtype, device="cuda")[..., ::2].transpose(1, 2)
    q.copy_(t["q"])
    kb = torch.empty((2 * 90 * 24 + 1,), dtype=dtype, device="cuda")[1:].view(2, 90, 1, 24)
    kb.copy_(t["k"][:, :, :1])
    vb = t["v"][:, :, :1].contiguous()
    kb.requires_grad_(True)
    vb.requires_grad_(True)
    q.requires_grad_(True)
    g = dev(p["g"]).requires_grad_(True)
    out, _ = dk.linear_attention(q, kb.expand(2, 90, 4, 24), vb.expand(2, 90, 4, 16), g,
                                 dev(p["valid"]), dev(p["reset"]))
    do = dev(p["do"], dtype).transpose(2, 3).contiguous().transpose(2, 3)
    dq, dkb, dvb, dg = torch.autograd.grad(out, (q, kb, vb, g), do)
    ref, A = oracle(p), sizes(p)
    tol = 2.1 * U if dtype == torch.bfloat16 else 128 * E
    assert np.all(np.abs(host(out) - ref["out"]) <= tol * A["out"])
    assert np.all(np.abs(host(dq) - ref["dq"]) <= tol * A["dq"])
    assert np.all(np.abs(host(dg) - ref["dg"]) <= 256 * E * A["dg"].max())
    # the heads' gradients are rounded to bf16, then added and rounded again
    for got, n in ((dkb, "dk"), (dvb, "dv")):
        a = A[n].sum(2, keepdims=True)
        assert np.all(np.abs(host(got) - ref[n].sum(2, keepdims=True)) <= 2 * tol * a)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_padding_may_hold_anything(dk, dtype):
    p = problem(10, 2, 130, 2, 64, 64, dtype, masks=True, initial=True, final=True)
    clean = run(dk, p, dtype)
    pad = p["valid"] == 0
    for n, x in (("q", np.nan), ("k", np.inf), ("v", -np.inf), ("do", np.nan), ("g", np.nan)):
        p[n] = p[n].copy()
        p[n][pad] = x
    dirty = run(dk, p, dtype)
    for n in clean:
        assert np.array_equal(clean[n], dirty[n]), n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("name", ["q", "k", "v", "g", "do"])
@pytest.mark.parametrize("V", [16, 80])
def test_a_value_that_is_not_finite_stays_with_those_that_see_it(dk, V, name, dtype):
    """A NaN at one token of one document reaches that document's later outputs (and the gradients of
    what they depend on), but no earlier token's output, no other document and no other sequence."""
    p = problem(11, 2, 200, 2, 16, V, dtype, masks=False)
    p["reset"] = np.zeros((2, 200))
    p["reset"][0, [40, 150]] = 1
    p["valid"] = np.ones((2, 200))
    clean, A = run(dk, p, dtype), sizes(p)
    tol = {n: 2 * (2.1 * U if dtype == torch.bfloat16 else 128 * E) * A[n]
           for n in ("out", "dq", "dk", "dv")}
    tol["dg"] = np.full_like(A["dg"], 2 * 256 * E * A["dg"].max())

    def same(n, where):  # its chunk is taken token by token: other roundings
        assert np.all(np.abs(got[n] - clean[n])[where] <= tol[n][where]), n

    at = 90
    p[name] = p[name].copy()
    p[name][0, at, 0] = np.nan
    got = run(dk, p, dtype)
    inside = np.zeros((2, 200, 2), bool)
    inside[0, 40:150, 0] = True
    for n in ("out", "dq", "dk", "dv", "dg"):
        far = ~inside
        same(n, far)
    before = np.s_[0, 40:at, 0]
    after = np.s_[0, at + 1:150, 0]
    if name == "do":
        assert np.array_equal(got["out"], clean["out"])
        for n in ("dk", "dv"):  # tokens that come later give nothing to it
            same(n, after)
        same("dq", after)
        same("dq", before)
    else:
        same("out", before)
        assert np.isnan(got["out"][0, at, 0]).all()
    if name == "q":
        same("out", after)
    if name in ("k", "v", "g"):
        assert np.isnan(got["out"][after]).any(-1).all()


def test_rows_more_than_32_bits_apart(dk):
    """Tokens 65536 elements apart, so that the last ones lie beyond 2^32 elements: the same results as
    from a copy."""
    T, far = 66000, 1 << 16
    buf = torch.empty((T * far,), dtype=torch.bfloat16, device="cuda")
    x = [buf[64 * i:].as_strided((1, T, 1, 32), (0, far, 64, 1)) for i in range(3)]
    for t in x:
        t.copy_(torch.randn(t.shape, device="cuda"))
    dense = [t.contiguous() for t in x]
    g = -torch.rand((1, T, 1), device="cuda")
    a = dk.linear_attention_forward(*x, g)
    b = dk.linear_attention_forward(*dense, g)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    da = dk.linear_attention_backward(*x, g, None, None, None, a[2], x[1])
    db = dk.linear_attention_backward(*dense, g, None, None, None, b[2], dense[1])
    for i, (p, q) in enumerate(zip(da[:4], db[:4])):
        assert torch.equal(p, q), i


def test_more_sequences_than_a_grid_axis_holds(dk):
    """65600 heads in two segments each: the same as a few of them alone."""
    B, T, H = 4100, 17 * 32, 16
    q = torch.randn((1, T, 1, 4), device="cuda").expand(B, T, H, 4)
    g = torch.linspace(-0.5, -0.01, H, device="cuda")
    out, fin, _ = dk.linear_attention_forward(q, q, q, g)
    few, few_fin, _ = dk.linear_attention_forward(q[:1], q[:1], q[:1], g)
    for b in (0, 1, 4095, 4096, 4099):
        assert torch.allclose(fin[b], few_fin[0], rtol=1e-5, atol=1e-5), b
        assert torch.allclose(out[b], few[0], rtol=1e-5, atol=1e-4), b


def test_runs_are_equal_bit_for_bit(dk):
    p = problem(12, 2, 700, 2, 64, 64, torch.bfloat16, initial=True, final=True)
    a, b = run(dk, p, torch.bfloat16), run(dk, p, torch.bfloat16)
    for n in a:
        assert np.array_equal(a[n], b[n]), n


def test_gradient_is_that_of_differences(dk):
    p = problem(13, 1, 140, 2, 16, 12, torch.float32, masks=True, initial=True, final=True)
    got = run(dk, p, torch.float32)
    r = np.random.default_rng(0)

    def loss(y):
        out, fin = dk.linear_attention(dev(y["q"]), dev(y["k"]), dev(y["v"]), dev(y["g"]),
                                       dev(y["valid"]), dev(y["reset"]), dev(y["initial"]))
        return (host(out) * y["do"]).sum() + (host(fin) * y["df"]).sum()

    for n in ("q", "k", "v", "g", "initial"):
        d = r.normal(size=p[n].shape)
        h = 1e-2
        hi, lo_ = dict(p), dict(p)
        hi[n], lo_[n] = p[n] + h * d, p[n] - h * d
        want = (loss(hi) - loss(lo_)) / (2 * h)
        have = (got["d" + n] * d).sum()
        # linear but for g (third order in h d); the difference of float32 results over 2 h
        scale = np.abs(got["d" + n] * d).sum()
        assert abs(want - have) <= 2e-3 * scale, n


@pytest.mark.parametrize("K", [16, 66])
@pytest.mark.parametrize("T", [40, 400, 1100])
def test_a_forward_that_no_backward_follows(dk, T, K):
    """The same output and state, from a checkpoint that a backward refuses where it holds too little."""
    from delta_kernels._lib import Gdn2Error
    p = problem(16, 1, T, 2, K, 16, torch.bfloat16, masks=True, initial=True)
    x = [dev(p[n], torch.bfloat16) for n in ("q", "k", "v")]
    x += [dev(p[n]) for n in ("g", "valid", "reset", "initial")]
    out, fin, ck = dk.linear_attention_forward(*x)
    o2, f2, scratch = dk.linear_attention_forward(*x, train=False)
    assert torch.equal(out, o2) and torch.equal(fin, f2)
    assert scratch.numel() <= ck.numel()
    if scratch.numel() < ck.numel():
        with pytest.raises(Gdn2Error, match="checkpoint"):
            dk.linear_attention_backward(*x, scratch, out)


@pytest.mark.parametrize("K", [16, 66])
def test_gradients_that_nobody_wants(dk, K):
    p = problem(14, 1, 100, 2, K, 16, torch.float32, initial=True)
    ref = run(dk, p, torch.float32)
    x = {n: dev(p[n]) for n in ("q", "k", "v", "g", "initial")}
    names = dict(q="dq", k="dk", v="dv", g="dg", initial="dinitial")
    for n in names:
        y = dict(x, **{n: x[n].clone().requires_grad_(True)})
        out, _ = dk.linear_attention(y["q"], y["k"], y["v"], y["g"], None, None, y["initial"])
        (got,) = torch.autograd.grad(out, y[n], dev(p["do"]))
        assert np.array_equal(host(got), ref[names[n]]), n
    # a loss of the final state alone
    y = {n: t.clone().requires_grad_(True) for n, t in x.items()}
    _, fin = dk.linear_attention(y["q"], y["k"], y["v"], y["g"], None, None, y["initial"])
    df = np.random.default_rng(1).normal(size=fin.shape)
    grads = torch.autograd.grad(fin, [y[n] for n in ("q", "k", "v", "g", "initial")], dev(df))
    q = dict(p, do=np.zeros_like(p["do"]), df=df.astype(np.float32).astype(np.float64))
    compare({names[n]: host(t) for n, t in zip(("q", "k", "v", "g", "initial"), grads)}, q,
            torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("K,V", [(64, 64), (1, 1), (33, 40), (128, 128), (16, 127)])
@pytest.mark.parametrize("B,H", [(1, 1), (3, 5)])
def test_steps_continue_a_prompt(dk, B, H, K, V, dtype):
    """A prompt and then single tokens: the results of the whole sequence.  The step itself has no
    rounding but the result's: u |out| in bf16."""
    T, n = 40, 5
    p = problem(15, B, T + n, H, K, V, dtype, masks=True, initial=True)
    ref, A = oracle(p), sizes(p)
    x = {m: dev(p[m], dtype) for m in ("q", "k", "v")}
    g, valid, reset = dev(p["g"]), dev(p["valid"]), dev(p["reset"])
    _, state = dk.linear_attention(x["q"][:, :T], x["k"][:, :T], x["v"][:, :T], g[:, :T],
                                   valid[:, :T], reset[:, :T], dev(p["initial"]))
    for t in range(T, T + n):
        at = np.s_[:, t:t + 1]
        out = dk.linear_attention_step(state, x["q"][at], x["k"][at], x["v"][at], g[at], valid[at],
                                       reset[at])
        bound = 128 * E * A["out"][at]
        if dtype == torch.bfloat16:
            bound = bound + U * np.abs(ref["out"][at])
        assert np.all(np.abs(host(out) - ref["out"][at]) <= bound + 1e-30)
    assert np.all(np.abs(host(state) - ref["fin"]) <= 128 * E * A["fin"])


def test_step_with_one_decay_a_head_and_without_masks(dk):
    p = problem(16, 2, 1, 3, 8, 12, torch.float32, head_decay=True, initial=True)
    state = dev(p["initial"])
    out = dk.linear_attention_step(state, *[dev(p[n]) for n in ("q", "k", "v", "g")])
    ref, A = oracle(p), sizes(p)
    assert np.all(np.abs(host(out) - ref["out"]) <= 128 * E * A["out"])
    # a reset empties a state that holds anything
    state = torch.full_like(state, float("nan"))
    dk.linear_attention_step(state, *[dev(p[n]) for n in ("q", "k", "v", "g")], None,
                             torch.ones((2, 1), device="cuda"))
    want = np.einsum("bhk,bhv->bhkv", p["k"][:, 0], p["v"][:, 0])
    assert np.all(np.abs(host(state) - want) <= 2 * E * np.abs(want))


def test_on_a_stream_of_its_own(dk):
    p = problem(17, 2, 300, 2, 32, 32, torch.bfloat16, initial=True, final=True)
    ref = run(dk, p, torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(dk, p, torch.bfloat16)
    for n in ref:
        assert np.array_equal(ref[n], got[n]), n


def test_in_a_graph(dk):
    """Captured once and replayed with other inputs."""
    p = problem(18, 1, 300, 2, 64, 64, torch.bfloat16)
    x = {n: dev(p[n], torch.bfloat16) for n in ("q", "k", "v", "do")}
    g = dev(p["g"])

    def both():
        out, fin, ck = dk.linear_attention_forward(x["q"], x["k"], x["v"], g)
        return (out, fin) + dk.linear_attention_backward(x["q"], x["k"], x["v"], g, None, None, None,
                                                         ck, x["do"])[:4]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        both()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for turn in range(3):
        for t in x.values():
            t.copy_(torch.randn_like(t))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, both()):
            assert torch.equal(a, b), turn


def test_refusals(dk):
    q = torch.zeros((2, 8, 3, 16), device="cuda")
    g = torch.zeros((2, 8, 3), device="cuda")
    m = torch.ones((2, 8), device="cuda")
    f = dk.linear_attention
    with pytest.raises(ValueError, match="GPU"):
        f(q.cpu(), q.cpu(), q.cpu(), g.cpu())
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        f(q.half(), q.half(), q.half(), g)
    with pytest.raises(TypeError, match="one dtype"):
        f(q, q.bfloat16(), q, g)
    with pytest.raises(ValueError, match="share"):
        f(q, q[:, :7], q, g)
    with pytest.raises(ValueError, match="g must"):
        f(q, q, q, g[:, :, :2])
    with pytest.raises(ValueError, match="valid"):
        f(q, q, q, g, m[:, :7])
    with pytest.raises(ValueError, match="nondifferentiable"):
        f(q, q, q, g, m.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="initial"):
        f(q, q, q, g, None, None, torch.zeros((2, 3, 16, 15), device="cuda"))
    with pytest.raises(ValueError, match="live on"):
        f(q, q, q, g.cpu())
    from delta_kernels._lib import Gdn2Error
    with pytest.raises(Gdn2Error, match="nonempty"):
        f(q[:, :0], q[:, :0], q[:, :0], g[:, :0])
    wide = torch.zeros((1, 2, 1, 129), device="cuda")
    with pytest.raises(Gdn2Error, match="widths"):
        f(wide, wide, wide, torch.zeros((1,), device="cuda"))
    state = torch.zeros((2, 3, 16, 16), device="cuda")
    with pytest.raises(Gdn2Error, match="time == 1"):
        dk.linear_attention_step(state, q, q, q, g)
    with pytest.raises(ValueError, match="state"):
        dk.linear_attention_step(state.transpose(2, 3), q[:, :1], q[:, :1], q[:, :1], g[:, :1])
    with pytest.raises(ValueError, match="state"):
        dk.linear_attention_step(state[:1], q[:, :1], q[:, :1], q[:, :1], g[:, :1])
    out, fin, ck = dk.linear_attention_forward(q, q, q, g)
    with pytest.raises(Gdn2Error, match="checkpoint"):
        dk.linear_attention_backward(q, q, q, g, None, None, None, ck[:0], q)
    with pytest.raises(ValueError, match="d_output"):
        dk.linear_attention_backward(q, q, q, g, None, None, None, ck, q[:, :7])
