"""Which memory the Muon update may share (CPU)."""
import random

import pytest

pytest.importorskip("torch")


def test_what_is_written_shares_no_memory():
    from delta_kernels.muon_ops import _overlap
    r = random.Random(0)
    seen = [0, 0]
    for _ in range(3000):
        def spans(n):
            return [(b, b + 4) for b in (r.randrange(0, 40) for _ in range(n))]

        written, read = spans(r.randrange(1, 4)), spans(r.randrange(0, 5))
        cells = [set(range(*s)) for s in written]
        want = any(cells[i] & cells[j] for i in range(len(cells)) for j in range(i)) \
            or any(c & set(range(*s)) for c in cells for s in read)
        assert _overlap(written, read) == want, (written, read)
        seen[want] += 1
    assert min(seen) > 300


def test_gradients_may():
    from delta_kernels.muon_ops import _overlap
    assert not _overlap([(0, 96), (96, 192)], [(200, 296), (200, 296), (240, 336), (250, 346)])
    assert _overlap([(0, 96), (330, 426)], [(200, 296), (200, 296), (240, 336), (250, 346)])
