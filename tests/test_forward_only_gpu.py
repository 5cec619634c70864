"""The forward-only calls and autograd."""
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
