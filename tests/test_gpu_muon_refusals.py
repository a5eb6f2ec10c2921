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
