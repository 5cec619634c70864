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


def _forward(**kw):
    a = dict(x=16, ldx=64, w=16, ldw=64, a=16, asl=8 * 64, asr=64, b=16, bsl=72 * 8, bsr=8, ids=16, ids64=1,
             scale=16, scale_all=1.0, dtype=0, m=4, k=64, n=72, L=3, r=8, back=1, y=16, ldy=72, kept=16,
             status=None, stream=None)
    a.update(kw)
    return _lib.load().moe_lora_forward(*a.values())


def _backward(**kw):
    a = dict(dy=16, lddy=72, x=16, ldx=64, w=16, ldw=64, a=16, asl=8 * 64, asr=64, b=16, bsl=72 * 8, bsr=8,
             scale=16, scale_all=1.0, dtype=0, m=4, k=64, n=72, L=3, r=8, kept=16, dx=16,
             lddx=64, da=16, db=16, status=None, stream=None)
    a.update(kw)
    return _lib.load().moe_lora_backward(*a.values())


COMMON = [dict(dtype=2), dict(m=-1), dict(m=1 << 31), dict(k=12), dict(k=0), dict(n=20), dict(L=0),
          dict(L=1025), dict(r=12), dict(r=136), dict(r=0), dict(x=None), dict(x=8), dict(ldx=56),
          dict(ldx=65), dict(w=None), dict(ldw=60), dict(a=None), dict(asr=56), dict(asl=64),
          dict(asl=513), dict(b=8), dict(bsr=4), dict(bsl=64), dict(kept=None), dict(kept=4)]


@pytest.mark.parametrize("kw", COMMON + [dict(ids=None), dict(y=None), dict(y=2), dict(ldy=64)])
def test_forward_refuses_bad_arguments_on_the_host(kw):
    assert _forward(**kw) == _lib.MOE_ERR_INVALID_ARG


@pytest.mark.parametrize("kw", COMMON + [
    dict(dy=None), dict(dy=4), dict(lddy=64), dict(dx=8),
    dict(lddx=56), dict(da=2), dict(db=8)])
def test_backward_refuses_bad_arguments_on_the_host(kw):
    assert _backward(**kw) == _lib.MOE_ERR_INVALID_ARG


def test_nothing_to_form_is_ok():
    assert _backward(dx=None, da=None, db=None) == _lib.MOE_OK
    assert _backward(m=0, da=None, db=None) == _lib.MOE_OK


def test_buffer_sizes():
    fn = _lib.load().moe_lora_kept_bytes
    assert fn(0, 3, 8) >= 0 and fn(100, 3, 8) >= 2 * 4 * 100 * 8
    for bad in ((-1, 3, 8), (100, 0, 8), (100, 1025, 8), (100, 3, 12), (100, 3, 136), (1 << 31, 3, 8)):
        assert fn(*bad) == -1
