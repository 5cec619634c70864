"""The routings that MoELayer.forward_few takes."""
import pytest
import torch

from tests.test_few_tokens_gpu import make

pytestmark = pytest.mark.gpu


def test_routing_as_forward_takes_it(cuda_device):
    from moe_overlap_b200.layer import MoELayer

    layer = MoELayer(64, 72, 4, 2, renormalize=True, micro_batch_size=16).init_random(std=0.05, seed=1)
    try:
        x = make(5, 4, 64, 72, torch.bfloat16, device=cuda_device)[0]
        routing = layer.route(x)
        out, idx, w = layer.forward_few(x, routing=routing)
        pair = layer.forward_few(x, routing=routing[1:])
        assert torch.equal(out, pair[0])
        for i, v in ((idx, w), pair[1:]):
            assert i is routing[1] and v is routing[2]
        for bad in ((routing[1],), (*routing, routing[1])):
            with pytest.raises(ValueError, match="routing must be"):
                layer.forward_few(x, routing=bad)
    finally:
        layer.close()
