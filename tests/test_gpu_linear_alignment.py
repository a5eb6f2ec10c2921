"""Results of linear attention at any address of their type: the same bits as at an aligned one."""
import struct

import pytest

torch = pytest.importorskip("torch")

from gpu_util import dev  # noqa: E402
from test_gpu_linear import dk, problem  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("K,V", [(64, 64), (128, 128)])
def test_results_off_16_bytes(dk, K, V, dtype):  # noqa: F811
    from delta_kernels import linear_ops as ops
    B, T, H = 2, 150, 2
    p = problem(1, B, T, H, K, V, dtype)
    q, k, v, do = (dev(p[n], dtype) for n in ("q", "k", "v", "do"))
    g = dev(p["g"])
    out, fin, ck = dk.linear_attention_forward(q, k, v, g)
    grads = dk.linear_attention_backward(q, k, v, g, None, None, None, ck, do)

    def off(like):
        n = like.numel()
        return torch.zeros((n + 16,), dtype=like.dtype, device="cuda")[1:n + 1].view(like.shape)

    L, stream = dk.lib(), torch.cuda.current_stream().cuda_stream
    shape = struct.pack("5q", B, T, H, K, V)
    views = [ops._view(t) for t in (q, k, v)] + [ops._view(g), None, None, None]
    o, f, c = off(out), off(fin), torch.empty_like(ck)
    assert o.data_ptr() % 16 and f.data_ptr() % 16
    assert L.gdn2_linear_scan(shape, *views, o.data_ptr(), f.data_ptr(), 1, c.data_ptr(), c.numel(),
                              stream) == 0
    assert torch.equal(o, out) and torch.equal(f, fin)
    ws = torch.empty((ops._bytes("gdn2_linear_workspace_bytes", q, v, ops._CODES[dtype]),),
                     dtype=torch.uint8, device="cuda")
    for which in range(3):  # dq off, dk off, all off
        d = [off(t) if which == i or which == 2 else torch.empty_like(t)
             for i, t in enumerate(grads[:4])]
        assert L.gdn2_linear_backward(shape, *views, c.data_ptr(), c.numel(), ops._view(do), None,
                                      *[t.data_ptr() for t in d], None, None, ws.data_ptr(),
                                      ws.numel(), stream) == 0
        for a, b in zip(d, grads):
            assert torch.equal(a, b), which
