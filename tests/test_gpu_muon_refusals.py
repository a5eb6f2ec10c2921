"""What the Muon update takes and refuses."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_muon import dk, matrices  # noqa: E402, F401
from gpu_util import dev  # noqa: E402

pytestmark = pytest.mark.gpu


def test_gradients_that_share_memory(dk):  # noqa: F811
    """Two gradients that are parts of one buffer, and overlap: as two copies of them."""
    pool = dev(matrices(1, 1, 30, 40)[0])
    g = [pool[:20], pool[10:]]
    out = []
    for gs in (g, [t.clone() for t in g]):
        p, m = ([torch.zeros(20, 40, device="cuda") for _ in range(2)] for _ in range(2))
        dk.muon_update(p, gs, m, 0.1)
        out.append(p + m)
    assert all(torch.equal(a, b) for a, b in zip(*out)) and out[0][0].any()
    p, m = ([torch.zeros(20, 40, device="cuda") for _ in range(2)] for _ in range(2))
    for args in (([pool[5:25], p[0]], g, m), (p, g, [m[0], pool[10:]]), ([p[0], p[0]], g, m)):
        before = [t.clone() for t in args[0] + args[2]]
        with pytest.raises(ValueError, match="share"):
            dk.muon_update(*args, 0.1)
        assert all(torch.equal(a, b) for a, b in zip(before, args[0] + args[2]))


def test_derivatives_are_refused(dk):  # noqa: F811
    fwAD = pytest.importorskip("torch.autograd.forward_ad")
    u = dev(matrices(2, 1, 20, 30)[0])
    p, m = torch.nn.Parameter(torch.zeros_like(u)), torch.zeros_like(u)
    wants = u.clone().requires_grad_(True)
    for args in ((p, wants * 2, m), (p, wants, m), (p, u, wants * 0), (p * 1, u, m), ([p, p * 1], [u, u], [m, m.clone()])):
        with pytest.raises(ValueError, match="no gradient"):
            dk.muon_update(*args, 0.1)
    with fwAD.dual_level():
        with pytest.raises(ValueError, match="no gradient"):
            dk.muon_update(p.detach(), fwAD.make_dual(u, u), m, 0.1)
    assert not p.any() and not m.any()
    # a parameter and its gradient; under no_grad all of them
    dk.muon_update(p, u, m, 0.1)
    with torch.no_grad():
        dk.muon_update(p, wants, m, 0.1)
        dk.muon_update(p * 1, wants * 2, m, 0.1)
    assert p.any() and m.any()


def test_a_parameter_that_a_graph_holds(dk):  # noqa: F811
    """Autograd is told of its change."""
    u = dev(matrices(3, 1, 20, 30)[0])
    p = torch.nn.Parameter(u.clone())
    y = (p * p).sum()
    dk.muon_update(p, u, torch.zeros_like(u), 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()
