"""The adapters' projection at sizes that a launch could refuse."""
import pytest
import torch

import moe_overlap_b200 as mo
from tests.test_lora_gpu import V, assert_close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("wide", ["N", "K"])
def test_more_column_blocks_than_65535(cuda_device, wide):
    """Gradients of 256 columns a block; x, dy and the adapters are sums of few products."""
    M, r = 3, 8
    K, N = (8, 65536 * 256 + 24) if wide == "N" else (65536 * 256 + 24, 8)
    g = torch.Generator(device=cuda_device).manual_seed(4)

    def rand(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=cuda_device) * std).to(torch.bfloat16)

    x, w, a, b, dy = rand(M, K), rand(N, K, std=0.1), rand(1, r, K, std=0.1), rand(1, N, r, std=0.1), rand(M, N)
    ids = torch.zeros(M, dtype=torch.int64, device=cuda_device)
    for t in (x, a, b):
        t.requires_grad_(True)
    y = mo.lora_linear(x, w, a, b, ids)
    da, db = torch.autograd.grad(y, (a, b), dy)
    mo.check_status(cuda_device, sync=True)
    u, tiny = 2.0 ** -8, 2.0 ** -133
    xd, ad, bd, dyd = (t.detach().double() for t in (x, a[0], b[0], dy))
    s, t = xd @ ad.t(), dyd @ bd
    # as in test_lora_gpu.py: fp32 sums, 16 bits of s and of t, one rounding
    ds = K * V * (xd.abs() @ ad.abs().t()) + 2.0 ** -16 * s.abs() + tiny
    dt = N * V * (dyd.abs() @ bd.abs()) + 2.0 ** -16 * t.abs() + tiny
    want = t.t() @ xd
    assert_close(da[0], (want, (dt + (M + 4) * V * t.abs()).t() @ xd.abs() + u * want.abs() + tiny))
    want = dyd.t() @ s
    assert_close(db[0], (want, dyd.abs().t() @ (ds + (M + 4) * V * s.abs()) + u * want.abs() + tiny))
