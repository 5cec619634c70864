"""CPU-only refusals of the adapters' projection: no kernel is launched."""
import pytest
import torch

import moe_overlap_b200 as mo
from moe_overlap_b200 import _lib


def test_cpu_tensors_are_refused():
    z = torch.zeros
    bf = torch.bfloat16
    with pytest.raises(ValueError, match="CUDA"):
        mo.lora_linear(z(2, 8, dtype=bf), z(8, 8, dtype=bf), z(1, 8, 8, dtype=bf), z(1, 8, 8, dtype=bf),
                       z(2, dtype=torch.int64))


def _shrink(**kw):
    a = dict(x=16, ldx=64, w=16, sl=8 * 64, sr=64, tr=0, perm=16, offs=16, dtype=0, m=4, k=64, L=3, r=8,
             s=16, stream=None)
    a.update(kw)
    return _lib.load().moe_lora_shrink(*a.values())


def _expand(**kw):
    a = dict(s=16, w=16, sl=64 * 8, sr=8, tr=0, scale=16, perm=16, offs=16, dtype=0, m=4, n=64, L=3, r=8,
             y=16, ldy=64, stream=None)
    a.update(kw)
    return _lib.load().moe_lora_expand(*a.values())


def _grad(**kw):
    a = dict(s=16, z=16, ldz=64, scale=16, perm=16, offs=16, dtype=0, m=4, n=64, L=3, r=8, g=16,
             gl=64 * 8, gr=8, tr=0, stream=None)
    a.update(kw)
    return _lib.load().moe_lora_grad(*a.values())


COMMON = [dict(dtype=2), dict(m=-1), dict(L=0), dict(L=1025), dict(r=12), dict(r=136), dict(r=0),
          dict(perm=None), dict(offs=None)]


@pytest.mark.parametrize("kw", COMMON + [
    dict(k=12), dict(k=0), dict(x=None), dict(x=8), dict(ldx=56), dict(ldx=65), dict(w=None), dict(sr=56),
    dict(sl=64), dict(tr=1, sr=4), dict(s=None)])
def test_shrink_refuses_bad_arguments_on_the_host(kw):
    assert _shrink(**kw) == _lib.MOE_ERR_INVALID_ARG


@pytest.mark.parametrize("kw", COMMON + [
    dict(n=12), dict(y=None), dict(y=2), dict(ldy=8), dict(w=8), dict(sr=4), dict(sl=8), dict(scale=None),
    dict(tr=1, sr=8), dict(s=None)])
def test_expand_refuses_bad_arguments_on_the_host(kw):
    assert _expand(**kw) == _lib.MOE_ERR_INVALID_ARG


@pytest.mark.parametrize("kw", COMMON + [
    dict(n=12), dict(z=None), dict(ldz=8), dict(g=None), dict(g=4), dict(gr=4), dict(gl=8),
    dict(scale=None), dict(tr=1, gr=8), dict(s=None)])
def test_grad_refuses_bad_arguments_on_the_host(kw):
    assert _grad(**kw) == _lib.MOE_ERR_INVALID_ARG


def test_plan_refuses_bad_arguments_and_empty_work_is_ok():
    plan = _lib.load().moe_lora_plan
    bad = _lib.MOE_ERR_INVALID_ARG
    assert plan(16, 0, -1, 3, 16, 16, 16, None, None) == bad
    assert plan(16, 0, 4, 0, 16, 16, 16, None, None) == bad
    assert plan(16, 0, 4, 1025, 16, 16, 16, None, None) == bad
    assert plan(None, 0, 4, 3, 16, 16, 16, None, None) == bad
    assert plan(16, 0, 4, 3, None, 16, 16, None, None) == bad
    assert plan(16, 0, 4, 3, 16, None, 16, None, None) == bad
    assert _shrink(m=0) == _lib.MOE_OK and _expand(m=0) == _lib.MOE_OK
