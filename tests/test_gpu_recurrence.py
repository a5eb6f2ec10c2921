"""Gated linear recurrence against the float64 oracle.

Bounds, fixed before the first run, with e = 2^-24.  A term of a state is a value times a decay.  On its
way it meets at most 16 roundings in a lane's run, 24 in a wave, 48 across waves and 8 for each block of 32
to 256 tokens (or segment) that it passes, and its decay is off by 88 e, the rounding of an exponent that
reaches 126 at most: N = 200 + 8 T / 32 roundings of the term at worst.  Summed over the terms
  y, final, dx, d_initial   N e (the same recurrence of the magnitudes)
  dg                        2 N e (magnitude of what is carried) (magnitude of the adjoint)
and half a step of bf16, 2^-8 |result|, where the result is bf16."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import recurrent_oracle as ro  # noqa: E402
from gpu_util import dev, host  # noqa: E402

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
F, H = torch.float32, torch.bfloat16
TYPES = [(F, F), (H, H), (H, F), (F, H)]
NAMES = ["f32", "bf16", "bf16-f32", "f32-bf16"]


@pytest.fixture(scope="module")
def dk():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import delta_kernels
    delta_kernels.lib()
    return delta_kernels


def rounded(a, dtype):
    return torch.tensor(a, dtype=F).to(dtype).double().numpy()


def inputs(seed, B, T, W, types, masks=False, initial=False):
    r = np.random.default_rng(seed)
    c = dict(x=rounded(r.normal(size=(B, T, W)), types[0]),
             g=rounded(-np.exp(r.uniform(-6, 1, size=W)) * r.random((B, T, W)), types[1]),
             valid=None, reset=None, initial=None,
             dy=rounded(r.normal(size=(B, T, W)), types[0]), df=rounded(r.normal(size=(B, W)), F))
    if masks:
        c["valid"] = (r.random((B, T)) < 0.8).astype(float)
        c["reset"] = (r.random((B, T)) < 0.05).astype(float)
    if initial:
        c["initial"] = rounded(r.normal(size=(B, W)), F)
    return c


def check(c, types, y, fin, dx=None, dg=None, di=None):
    x, g, valid, reset, initial = (c[n] for n in ("x", "g", "valid", "reset", "initial"))
    n = (200 + x.shape[1] / 4) * E
    mag = None if initial is None else np.abs(initial)
    ry, rf, _ = ro.recurrence(x, g, valid, reset, initial)
    my, mf, mc = ro.recurrence(np.abs(x), g, valid, reset, mag)
    half = [2.0 ** -8 if t == H else 0 for t in types]
    bounds = dict(y=(y, ry, n * my + half[0] * np.abs(ry)), final=(fin, rf, n * mf))
    if dx is not None:
        rdx, rdg, rdi = ro.recurrence_backward(x, g, valid, reset, initial, c["dy"], c["df"])
        mdx, _, mdi = ro.recurrence_backward(np.abs(x), g, valid, reset, mag, np.abs(c["dy"]),
                                             np.abs(c["df"]))
        bounds.update(dx=(dx, rdx, n * mdx + half[0] * np.abs(rdx)),
                      dg=(dg, rdg, 2 * n * mc * mdx + half[1] * np.abs(rdg)))
        if di is not None:
            bounds["d_initial"] = (di, rdi, n * mdi)
    for name, (got, ref, bound) in bounds.items():
        got = host(got)
        assert got.shape == ref.shape, name
        assert np.all(np.isfinite(got)), name
        err, bound = np.abs(got - ref), bound + 2.0 ** -120
        assert np.all(err <= bound), f"{name}: {(err / bound).max():.2f} of the bound"


def run(dk, c, types, place=lambda t: t):
    x, g = (place(dev(c[n], t)).requires_grad_(True) for n, t in (("x", types[0]), ("g", types[1])))
    initial = None if c["initial"] is None else dev(c["initial"]).requires_grad_(True)
    y, fin = dk.gated_recurrence(x, g, dev(c["valid"]), dev(c["reset"]), initial)
    assert y.dtype == types[0] and fin.dtype == F
    wrt = [x, g] + ([] if initial is None else [initial])
    grads = torch.autograd.grad([y, fin], wrt, [place(dev(c["dy"], types[0])), dev(c["df"])])
    assert grads[0].dtype == types[0] and grads[1].dtype == types[1]
    return (y, fin) + grads


@pytest.mark.parametrize("types", TYPES, ids=NAMES)
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 31, 32, 33, 63, 64, 65, 127, 129, 255, 256, 257, 511, 513, 1000])
def test_lengths(dk, T, types):
    c = inputs(T, 2, T, 72, types, initial=True)
    check(c, types, *run(dk, c, types))


@pytest.mark.parametrize("types", TYPES, ids=NAMES)
@pytest.mark.parametrize("W", [1, 2, 3, 7, 8, 9, 31, 32, 33, 63, 64, 65, 100, 128, 200, 513])
def test_widths(dk, W, types):
    c = inputs(W, 3, 70, W, types, masks=True, initial=True)
    check(c, types, *run(dk, c, types))


@pytest.mark.parametrize("types", TYPES, ids=NAMES)
@pytest.mark.parametrize("B,T,W", [(1, 5000, 3), (1, 3000, 64), (2, 2049, 40), (5, 700, 130)])
def test_segments(dk, B, T, W, types):
    for masks in (False, True):
        c = inputs(T, B, T, W, types, masks=masks, initial=masks)
        check(c, types, *run(dk, c, types))


@pytest.mark.parametrize("types", TYPES, ids=NAMES)
@pytest.mark.parametrize("B,T,W", [(20, 600, 520), (33, 257, 510), (130, 300, 270), (600, 70, 40), (1100, 130, 5)])
def test_workgroups_that_share_units(dk, B, T, W, types):
    """Enough sequences and channels for workgroups of 4 and of 2 waves, over several blocks."""
    c = inputs(T, B, T, W, types, masks=T != 300, initial=T != 600)
    check(c, types, *run(dk, c, types))


@pytest.mark.parametrize("B,T,W", [(1, 1, 1), (1, 30, 1), (1, 300, 1), (1, 520, 1), (1, 600, 1), (1, 1100, 1),
                                   (2, 600, 1), (1, 600, 2), (1, 20, 40), (300, 600, 33)])
def test_smallest_buffers(dk, B, T, W):
    for types in TYPES:
        c = inputs(B + T, B, T, W, types, initial=True)
        args = dev(c["x"], types[0]), dev(c["g"], types[1]), None, None, dev(c["initial"])
        y, fin, _ = dk.gated_recurrence_forward(*args, train=False)
        check(c, types, y, fin)
        check(c, types, *run(dk, c, types))


@pytest.mark.parametrize("types", TYPES, ids=NAMES)
def test_many_channels(dk, types):
    c = inputs(3, 130, 300, 260, types, masks=True)  # one segment a sequence
    check(c, types, *run(dk, c, types))


def layouts():
    def padded(t):
        wide = torch.full(t.shape[:2] + (t.shape[2] + 5,), float("nan"), dtype=t.dtype, device=t.device)
        wide[..., 3:-2] = t
        return wide[..., 3:-2]

    def times_first(t):
        return t.transpose(0, 1).contiguous().transpose(0, 1)

    def channels_first(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def every_second(t):
        wide = torch.full(t.shape[:2] + (2 * t.shape[2],), float("nan"), dtype=t.dtype, device=t.device)
        wide[..., ::2] = t
        return wide[..., ::2]

    return [padded, times_first, channels_first, every_second]


@pytest.mark.parametrize("types", TYPES, ids=NAMES)
@pytest.mark.parametrize("place", layouts(), ids=lambda f: f.__name__)
def test_layouts(dk, place, types):
    for T, W in ((45, 37), (600, 64)):
        c = inputs(5, 2, T, W, types, masks=True, initial=True)
        x, g = (place(dev(c[n], t)) for n, t in (("x", types[0]), ("g", types[1])))
        d = [dev(c[n]) for n in ("valid", "reset", "initial")]
        y, fin, ck = dk.gated_recurrence_forward(x, g, *d)
        grads = dk.gated_recurrence_backward(x, g, *d, ck, place(dev(c["dy"], types[0])), dev(c["df"]))
        check(c, types, y, fin, *grads)


@pytest.mark.parametrize("types", TYPES, ids=NAMES)
def test_broadcast_inputs(dk, types):
    """A decay a channel, expanded; its gradient is the sum over what it was expanded to."""
    B, T, W = 3, 200, 40
    c = inputs(6, B, T, W, types, initial=True)
    one = c["g"][0, 0]
    c["g"] = np.broadcast_to(one, (B, T, W))
    g = dev(one, types[1]).requires_grad_(True)
    row = dev(c["initial"][0]).requires_grad_(True)
    c["initial"] = np.broadcast_to(c["initial"][0], (B, W))
    c["dy"] = np.ones((B, T, W))
    x = dev(c["x"], types[0]).requires_grad_(True)
    y, fin = dk.gated_recurrence(x, g.expand(B, T, W), None, None, row.expand(B, W))
    dg, dx, di = torch.autograd.grad([y.sum(), (fin * dev(c["df"])).sum()], [g, x, row])
    check(c, types, y, fin, dx, torch.tensor(ro.recurrence_backward(
        c["x"], c["g"], None, None, c["initial"], c["dy"], c["df"])[1]))
    n = (200 + T / 4) * E
    rdg, rdi = ro.recurrence_backward(c["x"], c["g"], None, None, c["initial"], c["dy"], c["df"])[1:]
    mdx, _, mdi = ro.recurrence_backward(c["x"], c["g"], None, None, c["initial"], c["dy"], np.abs(c["df"]))
    mc = ro.recurrence(np.abs(c["x"]), c["g"], None, None, np.abs(c["initial"]))[2]
    # torch adds the expanded gradient up, in float32, and rounds it to g's type: each part and the sum
    sums = (2 * n * mc * mdx).sum((0, 1)) + 64 * E * np.abs(rdg).sum((0, 1))
    if types[1] == H:
        sums = sums + 2.0 ** -8 * (np.abs(rdg).sum((0, 1)) + np.abs(rdg.sum((0, 1))))
    assert np.all(np.abs(host(dg) - rdg.sum((0, 1))) <= sums)
    assert np.all(np.abs(host(di) - rdi.sum(0)) <= (n * mdi).sum(0) + 4 * E * np.abs(rdi).sum(0))


def test_wanted_gradients(dk):
    c = inputs(8, 2, 300, 20, (F, F), masks=True, initial=True)
    d = [dev(c[n]) for n in ("x", "g", "valid", "reset", "initial")]
    _, _, ck = dk.gated_recurrence_forward(*d)
    full = dk.gated_recurrence_backward(*d, ck, dev(c["dy"]), dev(c["df"]))
    for n in range(3):
        wanted = [i == n for i in range(3)]
        got = dk.gated_recurrence_backward(*d, ck, dev(c["dy"]), dev(c["df"]), wanted)
        for i in range(3):
            assert (got[i] is None) != wanted[i]
            assert got[i] is None or torch.equal(got[i], full[i])
    assert dk.gated_recurrence_backward(*d[:4], None, ck, dev(c["dy"]))[2] is None


def test_unused_outputs(dk):
    c = inputs(9, 2, 90, 20, (F, F), initial=True)
    x, g, initial = (dev(c[n]).requires_grad_(True) for n in ("x", "g", "initial"))
    y, fin = dk.gated_recurrence(x, g, None, None, initial)
    got = torch.autograd.grad(fin, [x, g, initial], dev(c["df"]), retain_graph=True)
    c0 = dict(c, dy=np.zeros_like(c["dy"]))
    check(c0, (F, F), y, fin, *got)
    got = torch.autograd.grad(y, [x, g, initial], dev(c["dy"]))
    check(dict(c, df=np.zeros_like(c["df"])), (F, F), y, fin, *got)


# ---- masks and values at the edges -----------------------------------------------------------


@pytest.mark.parametrize("types", TYPES[:2], ids=NAMES[:2])
@pytest.mark.parametrize("T", [1, 40, 700])
def test_padding_alone_keeps_the_state(dk, T, types):
    c = inputs(10, 3, T, 12, types, initial=True)
    c["valid"] = np.ones((3, T))
    c["valid"][1] = 0
    c["reset"] = np.zeros((3, T))
    c["reset"][1] = 1  # a reset on padding is none
    c["reset"][2, 0] = 1
    y, fin, dx, dg, di = run(dk, c, types)
    check(c, types, y, fin, dx, dg, di)
    assert torch.equal(fin[1], dev(c["initial"])[1]) and torch.equal(di[1], dev(c["df"])[1])
    assert not y[1].any() and not dx[1].any() and not dg[1].any() and not di[2].any()


@pytest.mark.parametrize("types", TYPES[:2], ids=NAMES[:2])
@pytest.mark.parametrize("T", [50, 900])
def test_what_is_not_finite_stays_where_it_is_seen(dk, T, types):
    nan, inf = float("nan"), float("inf")
    c = inputs(11, 2, T, 10, types)
    c["valid"], c["reset"] = np.ones((2, T)), np.zeros((2, T))
    cut = T // 2
    c["reset"][0, cut] = 1
    c["valid"][1, 7] = 0
    clean = {n: None if v is None else v.copy() for n, v in c.items()}
    c["x"][0, 5, 0], c["x"][0, 6, 1], c["x"][0, 4, 2] = nan, inf, -inf
    c["g"][0, 9, 3] = nan
    c["g"][0, cut, 4] = nan  # at a reset
    for n in ("x", "g", "dy"):
        c[n][1, 7] = nan  # at padding
    c["dy"][0, cut + 3, 5], c["dy"][0, cut + 3, 6] = nan, inf
    y, fin, dx, dg, _ = run(dk, dict(c, initial=np.zeros((2, 10))), types)
    good = run(dk, dict(clean, initial=np.zeros((2, 10))), types)
    y, dx, dg, fin = (t.detach() for t in (y, dx, dg, fin))
    for t in (y, dx, dg, fin):
        assert torch.isfinite(t[1]).all()
    for a, b in zip((y[1], fin[1], dx[1], dg[1]), (good[0][1], good[1][1], good[2][1], good[3][1])):
        assert torch.equal(a, b)
    # the first document sees it from its token on, the second not at all
    for ch, at in ((0, 5), (1, 6), (2, 4), (3, 9)):
        assert torch.equal(y[0, :at, ch], good[0][0, :at, ch])
        bad = y[0, at:cut, ch].float()
        assert not torch.isfinite(bad).any()
        if ch in (1, 2):
            assert (bad == (inf if ch == 1 else -inf)).all()
        assert torch.equal(y[0, cut:, ch], good[0][0, cut:, ch])
    assert torch.equal(y[0, :, 4], good[0][0, :, 4])
    assert torch.equal(fin, good[1])
    # the adjoint from token cut + 3 back to the reset, and not before it
    for ch, what in ((5, nan), (6, inf)):
        assert torch.equal(dx[0, :cut, ch], good[2][0, :cut, ch])
        assert torch.equal(dx[0, cut + 4:, ch], good[2][0, cut + 4:, ch])
        got = dx[0, cut:cut + 4, ch].float()
        assert got.isnan().all() if what != what else (got == inf).all()
    # a gate that is NaN spoils the adjoint before it
    assert dx[0, :9, 3].isnan().all() and torch.equal(dx[0, 9:, 3], good[2][0, 9:, 3])


@pytest.mark.parametrize("T", [40, 600])
def test_gates_that_empty_the_state(dk, T):
    c = inputs(12, 1, T, 6, (F, F), initial=True)
    c["initial"][0, 0] = float("inf")
    c["g"][0, 3] = [-np.inf, -1e30, -104, -87.5, -87.0, -60]
    y, fin, dx, dg, di = run(dk, c, (F, F))
    cc = dict(c, initial=np.where(np.isinf(c["initial"]), 0, c["initial"]))
    g = [t.detach().clone() for t in (y, dx, dg)]
    for t in g:
        t[0, :4, 0] = 0  # the channel that starts from infinity, up to its cut
    ref = ro.recurrence(cc["x"], cc["g"], None, None, cc["initial"])[0]
    assert np.allclose(host(g[0])[0, 4:], ref[0, 4:], rtol=1e-4, atol=1e-5)
    assert torch.isfinite(y[0, 3:]).all() and torch.isfinite(dx).all()
    assert not dg[0, 3, :4].any()
    # the initial state is seen by the three tokens before the cut
    rdi = ro.recurrence_backward(cc["x"], cc["g"], None, None, cc["initial"], c["dy"], c["df"])[2]
    assert np.allclose(host(di), rdi, rtol=1e-4, atol=1e-5)
    assert (y[0, :3, 0] == float("inf")).all()


def test_decay_past_float32_and_growth(dk):
    """A state of 1e30 under a decay of e^-150 over a block, and growth by e^150 from 1e-30: neither
    the decay nor the growth is a float32, the results are."""
    T = 150
    for sign, start in ((-1.0, 1e30), (1.0, 1e-30)):
        c = dict(x=np.zeros((1, T, 3)), g=np.full((1, T, 3), sign * 0.96), valid=None, reset=None,
                 initial=np.array([[start, 0.0, -start]]), dy=np.zeros((1, T, 3)),
                 df=np.zeros((1, 3)))
        c["g"] = rounded(c["g"], F)
        c["initial"] = rounded(c["initial"], F)
        y, fin, _, _, _ = run(dk, c, (F, F))
        check(c, (F, F), y, fin)
        assert not fin[0, 1].any()
    T = 700  # far past it: everything but zero becomes infinite
    g = torch.full((1, T, 3), 1.0, device="cuda")
    first = torch.tensor([[1e-38, 0.0, -1e-38]], device="cuda")
    y, fin = dk.gated_recurrence(torch.zeros((1, T, 3), device="cuda"), g, None, None, first)
    assert fin.tolist() == [[float("inf"), 0.0, float("-inf")]] and not y[..., 1].any()


def test_long_memory_is_exact_to_few_roundings(dk):
    """A constant decay of 1 - 1e-5 over 20000 tokens: a decay rounded once a token would be off by
    2^-25 / 1e-5, 3e-3 of the state."""
    T = 20000
    c = inputs(14, 1, T, 4, (F, F))
    c["g"] = rounded(np.full((1, T, 4), -1e-5), F)
    c["x"] = rounded(np.ones((1, T, 4)), F)
    y, fin = dk.gated_recurrence(dev(c["x"]), dev(c["g"]))
    _, ref, _ = ro.recurrence(c["x"], c["g"])
    # a state goes past a block in 5 roundings (the root twice, two products, a sum), and what a block adds
    # has some 100: 100 + 5 * 79 = 495 of the 8 * 79 = 632 allowed
    assert np.all(np.abs(host(fin) - ref) <= 8 * 79 * E * ref)


# ---- calls -------------------------------------------------------------------------------------


def test_offsets_beyond_32_bits(dk):
    far = (1 << 31) + 8
    big = torch.empty((2 * far + 64,), dtype=H, device="cuda")
    x = big.as_strided((1, 3, 20), (0, far, 1))
    g = big.as_strided((1, 3, 20), (0, far, 1), 32)
    c = inputs(15, 1, 3, 20, (H, H))
    x.copy_(dev(c["x"], H)), g.copy_(dev(c["g"], H))
    y, fin, ck = dk.gated_recurrence_forward(x, g)
    check(c, (H, H), y, fin)
    grads = dk.gated_recurrence_backward(x, g, None, None, None, ck, dev(c["dy"], H), dev(c["df"]))
    check(c, (H, H), y, fin, *grads)


@pytest.mark.parametrize("T", [64, 3000])
def test_same_bits_each_time_and_on_other_streams(dk, T):
    c = inputs(16, 2, T, 70, (H, H), masks=True, initial=True)
    args = [dev(c["x"], H), dev(c["g"], H), dev(c["valid"]), dev(c["reset"]), dev(c["initial"])]
    dy, df = dev(c["dy"], H), dev(c["df"])

    def both():
        y, fin, ck = dk.gated_recurrence_forward(*args)
        return (y, fin) + dk.gated_recurrence_backward(*args, ck, dy, df)

    first = both()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for s in streams:  # two calls and more at once
        with torch.cuda.stream(s):
            results.append(both())
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(first, r))


def test_captured_and_replayed(dk):
    T = 700
    c = [inputs(s, 2, T, 40, (H, F), masks=True, initial=True) for s in (17, 18, 19)]
    static = [dev(c[0]["x"], H), dev(c[0]["g"]), dev(c[0]["valid"]), dev(c[0]["reset"]), dev(c[0]["initial"])]
    dy, df = dev(c[0]["dy"], H), dev(c[0]["df"])

    def both():
        y, fin, ck = dk.gated_recurrence_forward(*static)
        return (y, fin) + dk.gated_recurrence_backward(*static, ck, dy, df)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for n in (1, 2, 0, 1):
        for t, name in zip(static + [dy, df], ("x", "g", "valid", "reset", "initial", "dy", "df")):
            t.copy_(dev(c[n][name], t.dtype))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, both()))
        check(c[n], (H, F), *got)


# ---- one token ------------------------------------------------------------------------------------


@pytest.mark.parametrize("types", TYPES, ids=NAMES)
@pytest.mark.parametrize("B,W", [(1, 1), (3, 65), (16, 512)])
def test_steps_are_the_scan(dk, B, W, types):
    T = 6
    c = inputs(B + W, B, T, W, types, masks=True, initial=True)
    x, g = dev(c["x"], types[0]), dev(c["g"], types[1])
    valid, reset, state = dev(c["valid"]), dev(c["reset"]), dev(c["initial"])
    y = torch.cat([dk.gated_recurrence_step(state, x[:, t:t + 1], g[:, t:t + 1], valid[:, t:t + 1],
                                            reset[:, t:t + 1]) for t in range(T)], 1)
    check(c, types, y, state)


def test_step_leaves_what_padding_leaves(dk):
    state = torch.tensor([[1.0, float("nan")], [2.0, 3.0]], device="cuda")
    x = torch.full((2, 1, 2), float("nan"), device="cuda")
    valid = torch.tensor([[0.0], [1.0]], device="cuda")
    y = dk.gated_recurrence_step(state, x, x, valid)
    assert state[0, 0] == 1 and not y[0].any() and y[1].isnan().all()
    # a reset drops what is not finite
    state = torch.tensor([[float("nan"), float("inf")]], device="cuda")
    one = torch.ones((1, 1, 2), device="cuda")
    assert (dk.gated_recurrence_step(state, one, one, None, one[..., 0]) == 1).all()


def test_step_and_autograd(dk):
    state = torch.zeros((2, 4), device="cuda")
    x = torch.randn((2, 1, 4), device="cuda")
    h = torch.randn((2, 5, 4), device="cuda", requires_grad=True)
    y, _ = dk.gated_recurrence(h, h, None, None, state)
    dk.gated_recurrence_step(state, x, x)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    for name in ("state", "x", "g"):
        a = dict(state=torch.zeros((2, 4), device="cuda"), x=x.clone(), g=x.clone())
        a[name].requires_grad_(True)
        with pytest.raises(ValueError, match="no gradient"):
            dk.gated_recurrence_step(**a)
        with torch.no_grad():
            dk.gated_recurrence_step(**a)


# ---- refusals ---------------------------------------------------------------------------------------


def test_refusals(dk):
    x = torch.zeros((2, 5, 4), device="cuda")
    m = torch.zeros((2, 5), device="cuda")
    for args, error in (((x.cpu(), x), "GPU"), ((x, x.cpu()), "GPU"), ((x[0], x[0]), "batch, time"),
                        ((x, x[:, :4]), "shape"), ((x, x, m[:, :3]), "valid"), ((x, x, None, m.t()), "reset"),
                        ((x, x, None, None, m), "initial"), ((x, x, m.cpu()), "valid must live")):
        with pytest.raises(ValueError, match=error):
            dk.gated_recurrence(*args)
    with pytest.raises(TypeError):
        dk.gated_recurrence(x.half(), x)
    with pytest.raises(TypeError):
        dk.gated_recurrence(x, x.double())
    with pytest.raises(ValueError, match="nondifferentiable"):
        dk.gated_recurrence(x, x, m.clone().requires_grad_(True))
    with pytest.raises(dk._lib.Gdn2Error, match="nonempty"):
        dk.gated_recurrence(x[:, :0], x[:, :0])
    _, _, ck = dk.gated_recurrence_forward(x, x)
    with pytest.raises(dk._lib.Gdn2Error, match="checkpoint"):
        dk.gated_recurrence_backward(x, x, None, None, None, ck[:8], x)
    with pytest.raises(ValueError, match="dy"):
        dk.gated_recurrence_backward(x, x, None, None, None, ck, x[:, :4])
    for state in (torch.zeros((4, 2), device="cuda").t(), torch.zeros((2, 4), device="cuda", dtype=H)):
        with pytest.raises(ValueError, match="state"):
            dk.gated_recurrence_step(state, x[:, :1], x[:, :1])
    with pytest.raises(dk._lib.Gdn2Error, match="time == 1"):
        dk.gated_recurrence_step(torch.zeros((2, 4), device="cuda"), x, x)


def test_other_checkpoints_are_refused(dk):
    x = torch.zeros(2, 9, 40, device="cuda")
    _, _, ck = dk.gated_recurrence_forward(x, x)
    _, _, none = dk.gated_recurrence_forward(x, x, train=False)
    for other in (none, ck.view(torch.float32), ck.new_zeros(1).expand(ck.numel())):
        with pytest.raises(ValueError, match="checkpoint"):
            dk.gated_recurrence_backward(x, x, None, None, None, other, x)
    dk.gated_recurrence_backward(x, x, None, None, None, ck, x)


def test_other_derivatives_are_refused(dk):
    fwAD = pytest.importorskip("torch.autograd.forward_ad")
    x = torch.randn((2, 5, 4), device="cuda")
    with fwAD.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            dk.gated_recurrence(fwAD.make_dual(x, x), x)
        dk.gated_recurrence(x, x)
    x.requires_grad_(True)
    y, _ = dk.gated_recurrence(x, -x * x)
    for loss in ((y ** 2).sum(), y.sum()):  # an upstream gradient that depends on x, and one that does not
        (d,) = torch.autograd.grad(loss, x, create_graph=True)
        with pytest.raises(RuntimeError, match="twice"):
            (d ** 2).sum().backward(retain_graph=True)
