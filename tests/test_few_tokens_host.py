"""CPU-only refusals of the few-token experts layer: no kernel is launched."""
import pytest
import torch

import moe_overlap_b200 as mo
from moe_overlap_b200 import _lib


def _args(T=2, E=3, H=16, F=24, dtype=torch.bfloat16):
    return (torch.zeros(T, H, dtype=dtype), torch.zeros(E, H, dtype=dtype),
            torch.zeros(E, F, H, dtype=dtype), torch.zeros(E, H, F, dtype=dtype))


def test_cpu_tensors_are_refused():
    x, rw, w1, w2 = _args()
    with pytest.raises(ValueError, match="CUDA"):
        mo.moe_few_tokens(x, rw, w1, w2, 2)
    with pytest.raises(ValueError, match="CUDA"):
        mo.experts_few_tokens(x, w1, w2, torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1))


def test_shapes_are_checked_before_anything_runs():
    x, rw, w1, w2 = _args()
    with pytest.raises(ValueError, match="router_w"):
        mo.moe_few_tokens(x, rw[:2], w1, w2, 2)
    with pytest.raises(ValueError, match="topk"):
        mo.experts_few_tokens(x, w1, w2, torch.zeros(3, 1, dtype=torch.int64), torch.zeros(3, 1))
    with pytest.raises(ValueError, match="int64 or int32"):
        mo.experts_few_tokens(x, w1, w2, torch.zeros(2, 1), torch.zeros(2, 1))


def _call(**kw):
    a = dict(x=16, ldx=64, rw=16, ldr=64, bias=None, w1=16, w1e=64 * 64, w1r=64, w2=16, w2e=64 * 64,
             w2r=64, dtype=0, T=2, H=64, F=64, E=4, k=2, renorm=0, idx=16, w=16, out=16, ldo=64,
             ws=16, nbytes=1 << 30, status=None, stream=None)
    a.update(kw)
    return _lib.load().moe_few_tokens(*a.values())


@pytest.mark.parametrize("kw", [
    dict(T=-1), dict(T=129), dict(H=12), dict(F=4), dict(H=0), dict(E=0), dict(E=257), dict(k=0),
    dict(k=5), dict(k=17, E=32), dict(dtype=2), dict(x=None), dict(x=8), dict(ldx=63), dict(ldx=56),
    dict(w1r=60), dict(w2=None), dict(w1e=64), dict(w2e=4097), dict(ldr=8), dict(out=2),
    dict(idx=None), dict(w=None), dict(ws=None), dict(ws=8)])
def test_c_entry_refuses_bad_arguments_on_the_host(kw):
    assert _call(**kw) == _lib.MOE_ERR_INVALID_ARG


def test_c_entry_checks_the_workspace_and_takes_no_tokens():
    lib = _lib.load()
    need = lib.moe_few_tokens_workspace(2, 64, 64, 4, 2)
    assert need > 0
    assert _call(nbytes=need - 1) == _lib.MOE_ERR_CAPACITY
    assert _call(T=0) == _lib.MOE_OK
    assert lib.moe_few_tokens_workspace(129, 64, 64, 4, 2) == -1
    assert lib.moe_few_tokens_workspace(2, 60, 64, 4, 2) == -1
