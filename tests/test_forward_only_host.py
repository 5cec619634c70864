"""CPU-only: calls that would lose a gradient without a word are refused before anything else."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import moe_overlap_b200 as mo


def _few():
    z = torch.zeros
    return dict(x=z(2, 16), router_w=z(3, 16), w1=z(3, 24, 16), w2=z(3, 16, 24), router_bias=z(3), out=z(2, 16))


def _given():
    z = torch.zeros
    return dict(x=z(2, 16), w1=z(3, 24, 16), w2=z(3, 16, 24), topk_idx=z(2, 1, dtype=torch.int64), topk_w=z(2, 1),
                out=z(2, 16))


CASES = [(mo.moe_few_tokens, _few, dict(top_k=2), n) for n in ("x", "router_w", "w1", "w2", "router_bias", "out")]
CASES += [(mo.experts_few_tokens, _given, {}, n) for n in ("x", "w1", "w2", "topk_w", "out")]


@pytest.mark.parametrize("fn,make,more,name", CASES)
def test_few_token_calls_refuse_inputs_that_require_a_gradient(fn, make, more, name):
    args = make()
    args[name].requires_grad_(True)
    with pytest.raises(ValueError, match="forward only"):
        fn(**args, **more)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):  # the next check
        fn(**args, **more)


@pytest.mark.parametrize("fn,make,more,name", CASES)
def test_few_token_calls_refuse_tangents(fn, make, more, name):
    args = make()
    with fwd.dual_level():
        args[name] = fwd.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(ValueError, match="forward only"):
            fn(**args, **more)


@pytest.mark.parametrize("name", ["x", "weight", "lora_a", "lora_b", "scale"])
def test_lora_linear_refuses_tangents(name):
    z = torch.zeros
    args = dict(x=z(2, 8), weight=z(8, 8), lora_a=z(1, 8, 8), lora_b=z(1, 8, 8), scale=z(1))
    with fwd.dual_level(), torch.no_grad():
        args[name] = fwd.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(ValueError, match="forward-mode"):
            mo.lora_linear(adapter_ids=z(2, dtype=torch.int64), **args)
