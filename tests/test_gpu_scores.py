"""Log probabilities, entropy and alternatives against the float64 oracle.

Bounds, fixed before the first run, with e = 2^-24, z = x / temperature, d_j = max z - z_j, D = sum p d and
D2 = sum p d^2 of a row.  An exponential is off by (2 d + 4) e (its argument's two roundings, and itself), a
sum of 32 in a thread by 32 e, the joins by 4 e each in 64 bits but for their factors:
  log s       (64 + 4 D) e
  log_probs   that, 4 d_t e for the given value's distance and e |log_probs| for the result
  entropy     that of log s, and (c + 64) e D + 4 e D2 of its own sum over a thread's c columns
  dx_j        p_j times the relative error of p_j, (64 + 4 D + 4 d_j + 2 |log p_j|) e, of everything that
              p_j multiplies, and |dh| times the errors of log p_j and the entropy; 4 e |dlp| at the target
and half a step of bf16, 2^-8 |dx|, where the gradient is bf16."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import recurrent_oracle as ro  # noqa: E402
from gpu_util import dev, host  # noqa: E402

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
F, H = torch.float32, torch.bfloat16
BOTH = pytest.mark.parametrize("dtype", [F, H], ids=["f32", "bf16"])


@pytest.fixture(scope="module")
def dk():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import delta_kernels
    delta_kernels.lib()
    return delta_kernels


def rounded(a, dtype):
    return torch.tensor(a, dtype=F).to(dtype).double().numpy()


def case(seed, rows, width, dtype, temperature=1.0, masked=False):
    r = np.random.default_rng(seed)
    x = r.normal(size=(rows, width)) * 2 + 8 * (r.random((rows, width)) < 2 / width)
    t = r.integers(0, width, rows)
    if masked:
        keep = x[np.arange(rows), t]
        x[r.random((rows, width)) < 0.5] = -np.inf
        x[np.arange(rows), t] = keep
    return dict(x=rounded(x, dtype), t=t, d=rounded(r.normal(size=rows), F),
                dh=rounded(r.normal(size=rows), F), temperature=temperature, valid=None)


def threads(rows, width, dtype):
    """Columns of a thread, at most: the smallest workgroups have 64."""
    n = 256 if rows >= 512 else 1024
    return -(-width // 64) if width <= 1024 else max(8, -(-width // n) + 32)


def check(c, dtype, r, dx=None):
    x, t, tau, valid = c["x"], c["t"], c["temperature"], c["valid"]
    on = np.ones(len(t), bool) if valid is None else valid != 0
    lp, given, h = ro.scores(x, t, tau)
    with np.errstate(invalid="ignore"):
        z = x / tau
        d = z.max(1, keepdims=True) - z
    p = np.exp(lp)
    d0, lp0 = np.where(p > 0, d, 0), np.where(p > 0, lp, 0)
    D, D2 = (p * d0).sum(1), (p * d0 ** 2).sum(1)
    logs = (64 + 4 * D) * E
    dt = d[np.arange(len(t)), t]
    bounds = dict(log_probs=logs + 4 * E * dt + E * np.abs(given),
                  entropy=logs + E * (threads(*x.shape, dtype) + 64) * D + 4 * E * D2)
    for name, ref in (("log_probs", given), ("entropy", h)):
        got = host(getattr(r, name)).reshape(-1)
        err = np.abs(got - ref)[on]
        assert np.all(got[~on] == 0)
        assert np.all(err <= bounds[name][on]), f"{name}: {(err / bounds[name][on]).max():.2f} of the bound"
    if r.top_tokens is not None:
        k = r.top_tokens.shape[-1]
        want = ro.top(x, k)
        got = r.top_tokens.cpu().numpy().reshape(-1, k)
        assert np.array_equal(got[on], want[on]) and not got[~on].any()
        wlp = np.take_along_axis(lp, want, 1)
        glp = host(r.top_log_probs).reshape(-1, k)
        inf = np.isinf(wlp)
        assert np.array_equal(glp[on][inf[on]], wlp[on][inf[on]]) and not glp[~on].any()
        bound = logs[:, None] + 4 * E * np.take_along_axis(np.where(inf.any(), d0, d), want, 1) + E * np.abs(wlp)
        keep = on[:, None] & ~inf
        assert np.all(np.abs(glp[keep] - wlp[keep]) <= bound[keep])
    if dx is not None:
        ref = ro.scores_backward(x, t, c["d"], c["dh"], tau)
        dl, dh = np.abs(c["d"])[:, None], np.abs(c["dh"])[:, None]
        rel = (64 + 4 * D[:, None] + 4 * d0 + 2 * np.abs(lp0)) * E
        bound = p * ((dl + dh * (np.abs(lp0) + h[:, None])) * (rel + 4 * E)
                     + dh * (rel + bounds["entropy"][:, None]))
        bound[np.arange(len(t)), t] += 4 * E * dl[:, 0]
        bound = bound / tau + 2.0 ** -120
        if dtype == H:
            bound = bound + 2.0 ** -8 * np.abs(ref)
        got = host(dx).reshape(ref.shape)
        err = np.abs(got - ref)[on]
        assert not got[~on].any()
        assert np.all(err <= bound[on]), f"dx: {(err / bound[on]).max():.2f} of the bound"


def run(dk, c, dtype, top=0, place=lambda t: t):
    x = place(dev(c["x"], dtype)).requires_grad_(True)
    t, valid = dev(c["t"], torch.int64), dev(c["valid"])
    r = dk.token_log_probs(x, t, top, valid, c["temperature"])
    (dx,) = torch.autograd.grad([r.log_probs, r.entropy], [x], [dev(c["d"]), dev(c["dh"])])
    assert dx.dtype == dtype and r.log_probs.dtype == F
    with torch.no_grad():
        alone = dk.token_log_probs(x, t, top, valid, c["temperature"])
    assert all(a is b or torch.equal(a, b) for a, b in zip(r, alone))
    return r, dx


@BOTH
@pytest.mark.parametrize("width", [1, 2, 3, 4, 7, 8, 9, 31, 33, 64, 100, 127, 513, 1000, 2049, 5003, 10007, 32768,
                                   50001])
def test_widths(dk, width, dtype):
    top = min(20, width)
    for seed, (masked, temperature) in enumerate(((False, 1.0), (True, 0.7))):
        c = case(width + seed, 5, width, dtype, temperature, masked)
        check(c, dtype, *run(dk, c, dtype, top))


@BOTH
@pytest.mark.parametrize("rows", [1, 2, 511, 512, 700])
def test_rows(dk, rows, dtype):
    c = case(rows, rows, 900, dtype)
    check(c, dtype, *run(dk, c, dtype, 3))


def test_a_wide_row(dk):
    c = case(1, 1, 262147, H)
    check(c, H, *run(dk, c, H, 64))


@BOTH
@pytest.mark.parametrize("rows,width", [(1, 65536), (1, 65537), (3, 100003), (11, 131072), (64, 70000), (2, 200000),
                                        (65, 70000)])
def test_rows_in_parts(dk, rows, width, dtype):
    """Few rows that are wide: parts, whose sums and alternatives are joined; 65 rows are not split."""
    c = case(width, rows, width, dtype, 0.8, masked=rows == 3)
    c["valid"] = np.ones(rows)
    c["valid"][1:rows:3] = 0
    r = np.random.default_rng(rows)
    c["x"][0] = rounded(r.integers(-2, 3, width).astype(float), dtype)  # thousands at the bound
    check(c, dtype, *run(dk, c, dtype, 20))
    if rows < 3:
        check(c, dtype, *run(dk, c, dtype, 64))
        check(c, dtype, *run(dk, c, dtype, 0))


@BOTH
def test_rows_in_parts_at_the_edges(dk, dtype):
    """Parts without a finite value, values that are not finite, and alternatives that all lie in one part."""
    width = 90001
    c = case(3, 6, width, dtype)
    nan, inf = np.nan, np.inf
    c["x"][0, 100:] = -inf
    c["x"][0, 200] = 1.0
    c["t"][0] = 5
    c["x"][1] = -inf
    c["x"][2, 70000], c["x"][2, 5] = nan, inf
    c["x"][3, 80000:80030] = np.linspace(20, 30, 30)
    c["x"][3] = rounded(c["x"][3], dtype)
    c["x"][4, ::2] = -0.0
    c["x"][4, 1::2] = 0.0
    x = dev(c["x"], dtype).requires_grad_(True)
    r = dk.token_log_probs(x, dev(c["t"], torch.int64), 25)
    (dx,) = torch.autograd.grad([r.log_probs, r.entropy], [x], [dev(c["d"]), dev(c["dh"])])
    assert np.array_equal(r.top_tokens.cpu().numpy(), ro.top(c["x"], 25))
    for row in (1, 2):
        assert r.log_probs[row].isnan() and r.entropy[row].isnan() and dx[row].isnan().all()
    for row in (0, 3, 4, 5):
        keep = slice(row, row + 1)
        sub = dict(c, x=c["x"][keep], t=c["t"][keep], d=c["d"][keep], dh=c["dh"][keep])
        check(sub, dtype, dk.TokenLogProbs(*(t[keep] for t in r)), dx[keep])


@BOTH
@pytest.mark.parametrize("top", [1, 2, 31, 32, 63, 64])
def test_alternatives(dk, top, dtype):
    for width in (64, 65, 3000):
        c = case(top, 7, width, dtype)
        check(c, dtype, *run(dk, c, dtype, top))


@BOTH
def test_equal_values_go_by_their_index(dk, dtype):
    r = np.random.default_rng(5)
    for width in (70, 4000, 40000):
        c = case(6, 6, width, dtype)
        c["x"] = r.integers(-3, 3, (6, width)).astype(float)  # thousands at the bound
        c["x"][1] = 0  # all equal
        c["x"][2, ::2] = -0.0
        c["x"][2, 1::2] = 0.0
        c["x"][3] = -5
        c["x"][3, 11:71:3] = 1  # a few above, the rest equal
        c["x"][4] = -np.arange(width) // 4
        c["x"] = rounded(c["x"], dtype)
        check(c, dtype, *run(dk, c, dtype, 20))


@BOTH
def test_few_values_that_are_finite(dk, dtype):
    c = case(7, 4, 500, dtype)
    for row, left in enumerate((1, 5, 20, 21)):
        out = np.ones(500, bool)
        out[37:37 + left] = False
        c["x"][row, out] = -np.inf
        c["t"][row] = 37
    check(c, dtype, *run(dk, c, dtype, 20))


@BOTH
def test_one_sure_token(dk, dtype):
    """The others together are 1e-6 of the distribution: the log probability is that, and no 0."""
    c = case(8, 2, 4096, dtype)
    c["x"] = rounded(np.full((2, 4096), -22.125), dtype)
    c["x"][0, 77] = c["x"][1, 4095] = 0
    c["t"] = np.array([77, 4095])
    r, dx = run(dk, c, dtype)
    check(c, dtype, r, dx)
    want = -4095 * np.exp(-22.125)
    # the others of a row are off by (2 * 22 + 64) e of themselves; 32 of them share a sum with the 1
    # (off by 32 e at most each, and no more than they are)
    bound = np.abs(want) * 108 * E + 32 * np.exp(-22.125)
    assert np.all(np.abs(host(r.log_probs) - want) <= bound)


@BOTH
def test_padded_rows_are_not_read(dk, dtype):
    c = case(9, 40, 333, dtype)
    c["valid"] = (np.random.default_rng(1).random(40) < 0.5).astype(float)
    c["valid"][:2] = (0, 1)
    c["t"][c["valid"] == 0] = -1
    good = c["x"].copy()
    c["x"][c["valid"] == 0] = np.nan
    r, dx = run(dk, c, dtype, 4)
    c["x"], c["t"] = good, np.where(c["valid"] == 0, 0, c["t"])
    check(c, dtype, r, dx)


@BOTH
def test_values_that_are_not_finite(dk, dtype):
    c = case(10, 6, 700, dtype)
    nan, inf = np.nan, np.inf
    c["x"][0, 5], c["x"][1, 6], c["x"][1, 600] = nan, inf, inf
    c["x"][2] = -inf
    c["x"][3, :3] = (inf, nan, nan)
    c["x"][4, 9] = -inf
    c["t"][4] = 9
    x = dev(c["x"], dtype).requires_grad_(True)
    r = dk.token_log_probs(x, dev(c["t"], torch.int64), 5)
    (dx,) = torch.autograd.grad([r.log_probs, r.entropy], [x], [dev(c["d"]), dev(c["dh"])])
    for row in range(4):
        assert r.log_probs[row].isnan() and r.entropy[row].isnan() and dx[row].isnan().all()
    assert r.log_probs[4] == -inf and torch.isfinite(r.entropy[4]) and torch.isfinite(dx[4]).all()
    assert np.array_equal(r.top_tokens.cpu().numpy(), ro.top(c["x"], 5))
    keep = slice(5, 6)
    sub = dict(c, x=c["x"][keep], t=c["t"][keep], d=c["d"][keep], dh=c["dh"][keep])
    check(sub, dtype, dk.TokenLogProbs(*(t[keep] for t in r)), dx[keep])


@BOTH
def test_values_far_apart(dk, dtype):
    c = case(11, 3, 300, dtype)
    big = rounded(np.array([3e38]), dtype)[0]
    c["x"][0, 0], c["x"][0, 1], c["t"][0] = big, -big, 1  # their distance is no float32
    c["x"][1, 0], c["t"][1] = 1e4, 0
    c["x"][2] -= 1e4
    c["x"] = rounded(c["x"], dtype)
    x = dev(c["x"], dtype).requires_grad_(True)
    r = dk.token_log_probs(x, dev(c["t"], torch.int64), 2)
    (dx,) = torch.autograd.grad([r.log_probs, r.entropy], [x], [dev(c["d"]), dev(c["dh"])])
    assert r.log_probs[0] == -float("inf") and r.entropy[0] == 0 and r.top_tokens[0, 0] == 0
    assert torch.isfinite(dx).all()
    sub = dict(c, x=c["x"][1:], t=c["t"][1:], d=c["d"][1:], dh=c["dh"][1:])
    check(sub, dtype, dk.TokenLogProbs(*(t[1:] for t in r)), dx[1:])


@BOTH
def test_targets_out_of_range(dk, dtype):
    c = case(12, 4, 50, dtype)
    t = c["t"].copy()
    t[:3] = (-1, 50, 1 << 40)
    x = dev(c["x"], dtype).requires_grad_(True)
    r = dk.token_log_probs(x, dev(t, torch.int64))
    assert r.log_probs[:3].isnan().all() and torch.isfinite(r.entropy).all()
    d = dev(c["d"])
    d[2] = 0  # left out of the loss
    (dx,) = torch.autograd.grad([r.log_probs, r.entropy], [x], [d, dev(c["dh"])])
    assert dx[:2].isnan().all() and torch.isfinite(dx[2:]).all()


@BOTH
@pytest.mark.parametrize("temperature", [1e-3, 0.3, 5.0, 1e6])
def test_temperatures(dk, temperature, dtype):
    c = case(13, 4, 600, dtype, temperature)
    check(c, dtype, *run(dk, c, dtype, 8))


def layouts():
    def padded(t):
        wide = torch.full((t.shape[0], t.shape[1] + 5), float("nan"), dtype=t.dtype, device=t.device)
        wide[:, 3:-2] = t
        return wide[:, 3:-2]

    def columns_first(t):
        return t.t().contiguous().t()

    def every_second(t):
        wide = torch.full((t.shape[0], 2 * t.shape[1]), float("nan"), dtype=t.dtype, device=t.device)
        wide[:, ::2] = t
        return wide[:, ::2]

    return [padded, columns_first, every_second]


@BOTH
@pytest.mark.parametrize("place", layouts(), ids=lambda f: f.__name__)
def test_layouts(dk, place, dtype):
    for width in (37, 1024, 5001):
        c = case(14, 6, width, dtype)
        x = place(dev(c["x"], dtype))
        t = dev(c["t"], torch.int64).repeat_interleave(3)[::3]
        c["valid"] = np.array([1.0, 0, 1, 1, 1, 0])
        valid = dev(c["valid"]).repeat_interleave(2)[::2]
        r, stats = dk.token_log_probs_forward(x, t, 5, valid)
        up = [dev(c[n]).repeat_interleave(2)[::2] for n in ("d", "dh")]
        dx = dk.token_log_probs_backward(x, t, valid, 1.0, stats, *up)
        check(c, dtype, r, dx)


def test_axes_and_broadcasts(dk):
    c = case(15, 12, 100, F)
    x = dev(c["x"]).view(3, 4, 100)
    t = dev(c["t"], torch.int64).view(3, 4)
    r = dk.token_log_probs(x.transpose(0, 1), t.t(), 2)
    assert r.log_probs.shape == (4, 3) and r.top_tokens.shape == (4, 3, 2)
    flat = dk.token_log_probs(dev(c["x"]), dev(c["t"], torch.int64), 2)
    assert torch.equal(r.log_probs.t().reshape(-1), flat.log_probs)
    one = dk.token_log_probs(x[0, 0], t[0, 0])
    assert one.log_probs.shape == () and torch.equal(one.log_probs, flat.log_probs[0])
    # one row of logits for many tokens: its gradient is their sum
    row = x[0, 0].clone().requires_grad_(True)
    lp = dk.token_log_probs(row.expand(12, 100), dev(c["t"], torch.int64)).log_probs
    (d,) = torch.autograd.grad(lp.sum(), row)
    x12 = np.broadcast_to(c["x"][0], (12, 100))
    ref = ro.scores_backward(x12, c["t"], np.ones(12), np.zeros(12))
    assert np.all(np.abs(host(d) - ref.sum(0)) <= 200 * E * np.abs(ref).sum(0))


def test_gradients_of_one_output(dk):
    c = case(16, 5, 60, F)
    x = dev(c["x"]).requires_grad_(True)
    t = dev(c["t"], torch.int64)
    r = dk.token_log_probs(x, t, 3)
    assert not r.top_log_probs.requires_grad
    (dx,) = torch.autograd.grad(r.log_probs, x, dev(c["d"]), retain_graph=True)
    check(dict(c, dh=np.zeros(5)), F, r, dx)
    (dx,) = torch.autograd.grad(r.entropy.sum(), x)  # an expanded upstream
    check(dict(c, d=np.zeros(5), dh=np.ones(5)), F, r, dx)


def test_no_rows(dk):
    x = torch.zeros((0, 7), device="cuda", requires_grad=True)
    r = dk.token_log_probs(x, torch.zeros((0,), dtype=torch.int64, device="cuda"), 2)
    assert r.log_probs.shape == (0,) and r.top_tokens.shape == (0, 2)
    (d,) = torch.autograd.grad(r.log_probs.sum(), x)
    assert d.shape == (0, 7)


def test_offsets_beyond_32_bits(dk):
    far = (1 << 31) + 8
    big = torch.empty((far + 600,), dtype=H, device="cuda")
    c = case(17, 2, 500, H)
    x = big.as_strided((2, 500), (far, 1))
    x.copy_(dev(c["x"], H))
    t = dev(c["t"], torch.int64)
    r, stats = dk.token_log_probs_forward(x, t, 4)
    check(c, H, r, dk.token_log_probs_backward(x, t, None, 1.0, stats, dev(c["d"]), dev(c["dh"])))
    del big, x
    rows, width = 70000, 32768  # rows * width > 2^31
    x = torch.zeros((rows, width), dtype=H, device="cuda")
    c = case(18, 3, width, H)
    x[-3:] = dev(c["x"], H)
    t = torch.zeros((rows,), dtype=torch.int64, device="cuda")
    t[-3:] = dev(c["t"], torch.int64)
    r, stats = dk.token_log_probs_forward(x, t)
    up = torch.zeros((2, rows), device="cuda")
    up[0, -3:], up[1, -3:] = dev(c["d"]), dev(c["dh"])
    dx = dk.token_log_probs_backward(x, t, None, 1.0, stats, up[0], up[1])
    check(c, H, dk.TokenLogProbs(r.log_probs[-3:], r.entropy[-3:], None, None), dx[-3:])
    assert not dx[:-3].any()


@pytest.mark.parametrize("rows,width,dtype", [(3000, 50001, H), (1400, 50003, F)])
def test_a_gradient_larger_than_the_caches(dk, rows, width, dtype):
    """The same bits as of its rows a hundred at a time."""
    torch.manual_seed(5)
    x = torch.randn(rows, width, device="cuda", dtype=dtype)
    tokens = torch.randint(0, width, (rows,), device="cuda")
    dl, dh = torch.randn(2, rows, device="cuda")
    _, stats = dk.token_log_probs_forward(x, tokens)
    dx = dk.token_log_probs_backward(x, tokens, None, 0.8, stats, dl, dh)
    for i in range(0, rows, 100):
        r = slice(i, i + 100)
        part = dk.token_log_probs_backward(x[r], tokens[r], None, 0.8, stats[r].contiguous(), dl[r], dh[r])
        assert torch.equal(dx[r], part)


def test_same_bits_each_time_and_on_other_streams(dk):
    c = case(19, 9, 5001, H)
    c["x"][1] = 0
    x, t, d, dh = dev(c["x"], H), dev(c["t"], torch.int64), dev(c["d"]), dev(c["dh"])

    def both():
        r, stats = dk.token_log_probs_forward(x, t, 20)
        return tuple(r) + (dk.token_log_probs_backward(x, t, None, 1.0, stats, d, dh),)

    first = both()
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams:
        with torch.cuda.stream(s):
            results.append(both())
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(first, r))


def test_captured_and_replayed(dk):
    c = [case(s, 7, 3001, H) for s in (20, 21, 22)]
    static = [dev(c[0]["x"], H), dev(c[0]["t"], torch.int64), dev(c[0]["d"]), dev(c[0]["dh"])]

    def both():
        r, stats = dk.token_log_probs_forward(static[0], static[1], 6)
        return r, dk.token_log_probs_backward(static[0], static[1], None, 1.0, stats, *static[2:])

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r, dx = both()
    for n in (1, 2, 0, 1):
        for s, name in zip(static, ("x", "t", "d", "dh")):
            s.copy_(dev(c[n][name], s.dtype))
        graph.replay()
        torch.cuda.synchronize()
        check(c[n], H, dk.TokenLogProbs(*(a.clone() for a in r)), dx.clone())
        other, dother = both()
        assert all(torch.equal(a, b) for a, b in zip(tuple(r) + (dx,), tuple(other) + (dother,)))


def test_refusals(dk):
    x = torch.zeros((2, 5), device="cuda")
    t = torch.zeros((2,), dtype=torch.int64, device="cuda")
    for args, error in (((x.cpu(), t), "GPU"), ((x, t.cpu()), "tokens must live"), ((x, t[:1]), "tokens must have"),
                        ((x, t, 6), "top"), ((x, t, -1), "top"), ((x, t, 0, t.float()[:1]), "valid must have"),
                        ((x, t, 0, None, 0.0), "temperature"), ((x, t, 0, None, float("nan")), "temperature"),
                        ((x[:, :0], t), "width")):
        with pytest.raises(ValueError, match=error):
            dk.token_log_probs(*args)
    with pytest.raises(ValueError, match="top"):
        dk.token_log_probs(torch.zeros((2, 100), device="cuda"), t, 65)
    with pytest.raises(TypeError):
        dk.token_log_probs(x.half(), t)
    with pytest.raises(TypeError):
        dk.token_log_probs(x, t.int())
    with pytest.raises(ValueError, match="nondifferentiable"):
        dk.token_log_probs(x, t, 0, torch.ones((2,), device="cuda", requires_grad=True))
    with pytest.raises(dk._lib.Gdn2Error, match="temperature"):
        dk.token_log_probs(x, t, 0, None, 1e-44)
    _, stats = dk.token_log_probs_forward(x, t)
    with pytest.raises(ValueError, match="stats"):
        dk.token_log_probs_backward(x, t, None, 1.0, stats[:1])
    with pytest.raises(ValueError, match="d_entropy"):
        dk.token_log_probs_backward(x, t, None, 1.0, stats, None, stats)
    dx = dk.token_log_probs_backward(x, t, None, 1.0, stats)
    assert not dx.any()


def test_other_derivatives_are_refused(dk):
    fwAD = pytest.importorskip("torch.autograd.forward_ad")
    x = torch.randn((2, 5), device="cuda")
    t = torch.zeros((2,), dtype=torch.int64, device="cuda")
    with fwAD.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            dk.token_log_probs(fwAD.make_dual(x, x), t)
        dk.token_log_probs(x, t)
    x.requires_grad_(True)
    (d,) = torch.autograd.grad(dk.token_log_probs(x * x, t).log_probs.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        (d ** 2).sum().backward()
