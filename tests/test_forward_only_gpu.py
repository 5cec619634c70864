"""What the forward-only calls do to autograd: refuse gradients, and mark `out` as written."""
import pytest
import torch

import moe_overlap_b200 as mo
from tests.test_few_tokens_gpu import make

pytestmark = pytest.mark.gpu


def test_layer_refuses_a_gradient_and_runs_without_one(cuda_device):
    from moe_overlap_b200.layer import MoELayer

    layer = MoELayer(64, 72, 4, 2, micro_batch_size=16, router_bias=True).init_random(std=0.05, seed=1)
    try:
        x = make(3, 4, 64, 72, torch.bfloat16, device=cuda_device)[0]
        want = layer.forward_few(x)[0]
        for p in (layer.router_w, layer.router_b, layer.w1, layer.w2):
            p.requires_grad_(True)  # a layer being trained can still decode
        assert torch.equal(layer.forward_few(x)[0], want)
        x.requires_grad_(True)
        with pytest.raises(ValueError, match="forward only"):
            layer.forward_few(x)
        with torch.no_grad():
            assert torch.equal(layer.forward_few(x)[0], want)
    finally:
        layer.close()


def test_out_is_marked_as_written(cuda_device):
    """A product saved from `out` before the call may not be differentiated after it."""
    x, rw, w1, w2 = make(3, 4, 64, 72, torch.bfloat16, device=cuda_device)
    out = torch.ones(3, 64, dtype=x.dtype, device=cuda_device)
    p = torch.ones_like(out, requires_grad=True)
    y = (p * out).sum()
    mo.moe_few_tokens(x, rw, w1, w2, 2, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()
    with torch.inference_mode():
        again = torch.empty_like(x)
        mo.moe_few_tokens(x, rw, w1, w2, 2, out=again)
    assert torch.equal(again, out)
