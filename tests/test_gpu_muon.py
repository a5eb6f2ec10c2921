"""Newton-Schulz products and Muon updates against the float64 oracle.

Tolerance, fixed before the first run.  Steps amplify roundings by up to 3.9 each (the quintic's largest slope
on [0, 1.2]), in directions that depend on the matrix, so the oracle says how far the arithmetic may be off: its
products of float16 pairs, summed in float32 by 32 columns, are the library's but for the order inside a sum.
Norm and largest value of the difference may be 4 times what they are there, with a floor of 64 e of the
result's, e = 2^-24 (the normalisation, the scales and the result's own rounding); half a step, 2^-8 of a value,
is added where results are bf16."""
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


def matrices(seed, count, rows, cols, dtype=F, size=1e-3):
    """Gradients: a few strong directions and noise."""
    r = np.random.default_rng(seed)
    k = min(3, rows, cols)
    u = r.normal(size=(count, rows, k)) @ r.normal(size=(count, k, cols)) * 0.3
    return rounded((u + r.normal(size=(count, rows, cols)) * (0.2 + r.random((count, rows, 1)))) * size, dtype)


def check(u, got, dtype, every=1, **args):
    """got of the matrices u; the emulated arithmetic of every so-manieth stands for all."""
    got = host(got)
    assert got.shape == u.shape and np.all(np.isfinite(got))
    norm = top = 0.0
    refs = [ro.orthogonalize(x, **args) for x in u]
    for x, ref in list(zip(u, refs))[::every]:
        d = ro.orthogonalize(x, product=ro.split_product, **args) - ref
        norm = max(norm, 4 * np.linalg.norm(d) + 64 * E * np.linalg.norm(ref))
        top = max(top, 4 * np.abs(d).max() + 64 * E * np.abs(ref).max())
    half = 2.0 ** -8 if dtype == H else 0
    for x, ref in zip(got, refs):
        err = np.abs(x - ref)
        over = np.maximum(err - half * np.abs(ref), 0)
        assert np.linalg.norm(over) <= norm, f"norm: {np.linalg.norm(over) / norm:.2f} of the bound"
        assert over.max() <= top, f"largest: {over.max() / top:.2f} of the bound"


@BOTH
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (7, 1), (2, 3), (16, 16), (17, 33), (63, 64), (64, 65),
                                       (65, 64), (100, 31), (128, 130), (200, 333), (333, 200), (40, 1001)])
def test_shapes(dk, rows, cols, dtype):
    u = matrices(rows * cols, 2, rows, cols, dtype)
    check(u, dk.orthogonalize(dev(u, dtype)), dtype)


@BOTH
@pytest.mark.parametrize("count,rows,cols", [(33, 20, 70), (70, 130, 5), (100, 129, 200), (26, 500, 530)])
def test_many(dk, count, rows, cols, dtype):
    """More matrices than one launch takes, and enough for the large tiles."""
    u = matrices(count, count, rows, cols, dtype)
    check(u, dk.orthogonalize(dev(u, dtype)), dtype, every=40)


@BOTH
@pytest.mark.parametrize("count,rows,cols", [(1, 16, 2000), (3, 64, 3001), (2, 2500, 8), (1, 65, 3000), (2, 3000, 120),
                                             (1, 1, 5000)])
def test_long_sums(dk, count, rows, cols, dtype):
    """Few tiles with long sums, which are made in parts; up to 64 rows the operands are float32."""
    u = matrices(rows + cols, count, rows, cols, dtype)
    check(u, dk.orthogonalize(dev(u, dtype)), dtype)


@pytest.mark.parametrize("rows,cols", [(8, 8), (8, 3000), (16, 2000), (40, 60), (64, 64), (64, 1000)])
def test_small_matrices_are_float32_s(dk, rows, cols):
    """Operands and sums of float32: over eight matrices the difference is no larger than that of the formulas in
    float32 (numpy), whose operands are the same and whose sums are no shorter."""
    u = matrices(rows, 8, rows, cols)
    got = host(dk.orthogonalize(dev(u)))
    own = plain = 0.0
    for x, y in zip(u, got):
        ref = ro.orthogonalize(x)
        z = x.astype(np.float32)
        z = z / (np.sqrt((z * z).sum()) + np.float32(1e-7))
        a, b, c = (np.float32(k) for k in ro.COEFFICIENTS)
        for _ in range(5):
            gram = z @ z.T
            z = a * z + (b * gram + c * (gram @ gram)) @ z
        own += np.linalg.norm(y - ref) ** 2
        plain += np.linalg.norm(z - ref) ** 2
    assert own <= plain


def test_a_large_matrix(dk):
    """1600 x 2100 has the large tiles' triangle with a rest on both sides."""
    u = matrices(5, 1, 1600, 2100)
    x = dev(u)
    check(u, dk.orthogonalize(x), F)
    many = torch.cat([x] * 4)  # 4 x 91 tiles
    out = dk.orthogonalize(many)
    check(u, out[3:], F)
    assert torch.equal(out[0], out[3])


@pytest.mark.parametrize("count,rows,cols", [(37, 20, 2500), (9, 130, 700), (35, 333, 90), (3, 1200, 1300)])
def test_equal_matrices_have_equal_results(dk, count, rows, cols):
    """Wherever they stand in a call, also behind the 32 of a launch, and whether or not sums are made in parts."""
    u = dev(matrices(rows, 1, rows, cols)).expand(count, rows, cols)
    out = dk.orthogonalize(u)
    assert torch.equal(out, out[:1].expand_as(out))


def test_spectrum(dk):
    u = matrices(6, 1, 96, 160)
    s = np.linalg.svd(host(dk.orthogonalize(dev(u)))[0], compute_uv=False)
    assert np.all((s > 0.6) & (s < 1.3))


@pytest.mark.parametrize("steps", [1, 2, 3, 8])
@pytest.mark.parametrize("coefficients", [ro.COEFFICIENTS, (1.5, -0.5, 0.0), (1.875, -1.25, 0.375), (0.01, 0.0, 0.0),
                                          (2.5, 0.0, 0.0), (-1.0, 0.25, 0.0)])
def test_steps_and_coefficients(dk, steps, coefficients):
    args = dict(steps=steps, coefficients=tuple(float(np.float32(c)) for c in coefficients))
    u = matrices(7, 1, 50, 90)
    check(u, dk.orthogonalize(dev(u), **args), F, **args)
    t = np.ascontiguousarray(u.transpose(0, 2, 1))
    check(t, dk.orthogonalize(dev(t), **args), F, **args)


@BOTH
@pytest.mark.parametrize("size", [1e-35, 1e-12, 1e12, 1e35])
def test_sizes_of_values(dk, size, dtype):
    u = matrices(8, 2, 30, 40, dtype, size)
    eps = 0.0 if size < 1 else 1e-7
    check(u, dk.orthogonalize(dev(u, dtype), epsilon=eps), dtype, epsilon=eps)


def test_nothing_and_not_finite(dk):
    u = dev(matrices(9, 4, 70, 80))
    good = dk.orthogonalize(u)
    u[0] = 0
    u[2, 3, 4], u[3, 1, 1] = float("nan"), float("inf")
    out = dk.orthogonalize(u)
    assert not out[0].any() and torch.equal(out[1], good[1])
    assert out[2].isnan().all() and out[3].isnan().all()
    assert dk.orthogonalize(u[:1], epsilon=0.0).isnan().all()


def layouts():
    def transposed(t):
        return t.transpose(-1, -2).contiguous().transpose(-1, -2)

    def padded(t):
        wide = torch.full(t.shape[:-2] + (t.shape[-2], t.shape[-1] + 5), float("nan"), dtype=t.dtype,
                          device=t.device)
        wide[..., 3:-2] = t
        return wide[..., 3:-2]

    def matrices_last(t):
        return t.movedim(0, -1).contiguous().movedim(-1, 0)

    return [transposed, padded, matrices_last]


@BOTH
@pytest.mark.parametrize("place", layouts(), ids=lambda f: f.__name__)
def test_layouts(dk, place, dtype):
    for rows, cols in ((30, 70), (70, 30)):
        u = matrices(10, 3, rows, cols, dtype)
        x = dev(u, dtype)
        out = dk.orthogonalize(place(x))
        assert out.is_contiguous() and torch.equal(out, dk.orthogonalize(x))
        check(u, out, dtype)


def test_axes(dk):
    u = dev(matrices(11, 6, 10, 12))
    full = dk.orthogonalize(u)
    assert torch.equal(dk.orthogonalize(u[2]), full[2])
    assert torch.equal(dk.orthogonalize(u.view(2, 3, 10, 12)), full.view(2, 3, 10, 12))
    assert torch.equal(dk.orthogonalize(u[0].expand(4, 10, 12)), full[:1].expand(4, 10, 12))
    assert dk.orthogonalize(u[:0]).shape == (0, 10, 12)


def test_offsets_beyond_32_bits(dk):
    far = (1 << 31) + 8
    big = torch.empty((far + 5000,), dtype=H, device="cuda")
    x = big.as_strided((2, 40, 60), (far, 60, 1))
    u = matrices(12, 2, 40, 60, H)
    x.copy_(dev(u, H))
    check(u, dk.orthogonalize(x), H)


@pytest.mark.parametrize("rows,cols", [(33, 90), (90, 33), (256, 256)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_update(dk, rows, cols, nesterov):
    r = np.random.default_rng(13)
    g = matrices(13, 3, rows, cols)
    p, m = rounded(r.normal(size=g.shape), F), rounded(5e-3 * r.normal(size=g.shape), F)
    args = dict(beta=0.9, nesterov=nesterov, decay=0.1)
    tp, tg, tm = ([t.clone() for t in dev(a)] for a in (p, g, m))
    assert dk.muon_update(tp, tg, tm, 0.05, **args) is None
    for i in range(3):
        wp, wm = ro.muon(p[i], g[i], m[i], 0.05, **args)
        sp, _ = ro.muon(p[i], g[i], m[i], 0.05, product=ro.split_product, **args)
        # two roundings of the momentum and of the parameter
        assert np.all(np.abs(host(tm[i]) - wm) <= 3 * E * (np.abs(wm) + 0.9 * np.abs(m[i])))
        d = np.abs(host(tp[i]) - wp)
        bound = 4 * np.abs(sp - wp).max() + 64 * E * np.abs(wp - (1 - 0.05 * 0.1) * p[i]).max() + 4 * E * np.abs(p[i])
        assert np.all(d <= bound), f"{(d / bound).max():.2f} of the bound"
        assert np.array_equal(host(tg[i]), g[i])
    # a matrix alone, and several updates
    one = [dev(a[0]) for a in (p, g, m)]
    dk.muon_update(*one, 0.05, **args)
    assert torch.equal(one[0], tp[0]) and torch.equal(one[2], tm[0])
    versions = [t._version for t in tp + tm + tg]
    dk.muon_update(tp, tg, tm, 0.05, **args)
    assert [t._version for t in tp + tm + tg] == [v + (i < 6) for i, v in enumerate(versions)]


def test_one_gradient_for_several(dk):
    g = dev(matrices(14, 1, 20, 30)[0])
    p, m = [torch.zeros_like(g) for _ in range(2)], [torch.zeros_like(g) for _ in range(2)]
    dk.muon_update(p, [g, g], m, 0.1)
    assert torch.equal(p[0], p[1]) and p[0].any()


def test_optimizer(dk):
    torch.manual_seed(0)
    shapes = [(20, 30), (30, 20), (20, 30), (64, 64), (20, 30)]
    params = [torch.nn.Parameter(torch.randn(s, device="cuda")) for s in shapes]
    start = [host(p) for p in params]
    opt = dk.Muon(params, lr=0.1, weight_decay=0.2, momentum=0.8)
    mom = [np.zeros(s) for s in shapes]
    for step in range(3):
        for i, p in enumerate(params):
            p.grad = None if i == 4 or (i == 2 and step == 0) else dev(matrices(step * 9 + i, 1, *shapes[i])[0])
        opt.step()
        for i, p in enumerate(params):
            if p.grad is not None:
                start[i], mom[i] = ro.muon(start[i], host(p.grad), mom[i], 0.1, beta=0.8, decay=0.2)
    for p, want in zip(params, start):
        assert np.abs(host(p) - want).max() <= 1e-4  # three steps of 0.1 of results to 2e-5 each
    assert params[4] not in opt.state and set(opt.state[params[0]]) == {"momentum"}
    other = dk.Muon([torch.nn.Parameter(p.detach().clone()) for p in params])
    other.load_state_dict(opt.state_dict())
    assert other.param_groups[0]["lr"] == 0.1
    assert opt.step(lambda: torch.tensor(3.0)) == 3
    with pytest.raises(ValueError, match="matrices"):
        dk.Muon([torch.nn.Parameter(torch.zeros(4, device="cuda"))])


def test_a_strided_gradient(dk):
    u = matrices(21, 1, 24, 40)[0]
    one, two = (torch.nn.Parameter(torch.zeros(24, 40, device="cuda")) for _ in range(2))
    one.grad, two.grad = dev(u), dev(u.T.copy()).T
    assert not two.grad.is_contiguous()
    dk.Muon([one, two]).step()
    assert torch.equal(one, two) and one.abs().max() > 0


def test_same_bits_each_time_and_on_other_streams(dk):
    u = dev(matrices(15, 3, 150, 90, H), H)
    first = dk.orthogonalize(u)
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams:
        with torch.cuda.stream(s):
            results.append(dk.orthogonalize(u))
    torch.cuda.synchronize()
    assert all(torch.equal(first, r) for r in results)


def test_captured_and_replayed(dk):
    g = [matrices(s, 2, 40, 70) for s in (16, 17, 18)]
    x = dev(g[0])
    p, m = [torch.zeros((40, 70), device="cuda") for _ in range(2)], [torch.zeros((40, 70), device="cuda")
                                                                     for _ in range(2)]
    q, n = [t.clone() for t in p], [t.clone() for t in m]

    def both(p, m):
        out = dk.orthogonalize(x)
        dk.muon_update(p, list(x), m, 0.1)
        return out

    both([t.clone() for t in p], [t.clone() for t in m])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(p, m)
    for i in (1, 2, 0, 1):
        x.copy_(dev(g[i]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, both(q, n))
        assert all(torch.equal(a, b) for a, b in zip(p + m, q + n))
        check(g[i], out, F)


def test_refusals(dk):
    x = torch.zeros((4, 6), device="cuda")
    for bad in (x[0], x.cpu()):
        with pytest.raises(ValueError):
            dk.orthogonalize(bad)
    with pytest.raises(TypeError):
        dk.orthogonalize(x.half())
    with pytest.raises(ValueError, match="no gradient"):
        dk.orthogonalize(x.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="three"):
        dk.orthogonalize(x, coefficients=(1.0, 2.0))
    for args, text in ((dict(steps=0), "steps"), (dict(steps=101), "steps"), (dict(epsilon=-1.0), "epsilon"),
                       (dict(epsilon=float("nan")), "epsilon"), (dict(coefficients=(100.0, 0, 0)), "grow"),
                       (dict(coefficients=(1.5, 0.5, 0.5), steps=9), "grow"),
                       (dict(coefficients=(float("nan"), 0, 0)), "grow")):
        with pytest.raises(dk._lib.Gdn2Error, match=text):
            dk.orthogonalize(x, **args)
    with pytest.raises(dk._lib.Gdn2Error, match="nonempty"):
        dk.orthogonalize(x[:, :0])
    y, z = torch.zeros_like(x), torch.zeros_like(x)
    for args in (([x, y], [y], [z]), (x, y, x), (x, x, z), ([x, x], [y, y], [z, z.clone()]), (x.t(), y.t(), z.t()),
                 (x, y[:3], z), (x, y.double(), z), (x.cpu(), y, z), (x[0], y[0], z[0])):
        with pytest.raises(ValueError):
            dk.muon_update(*args, 0.1)
    pool = torch.zeros((40,), device="cuda")
    with pytest.raises(ValueError, match="share"):
        dk.muon_update([pool[:24].view(4, 6), pool[16:].view(4, 6)], [y, y], [z, z.clone()], 0.1)
    dk.muon_update([], [], [], 0.1)
    assert not x.any() and not z.any()
