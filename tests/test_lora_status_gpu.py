"""Errors of the device around a backward pass of the adapters' projection."""
import ctypes

import pytest
import torch

import moe_overlap_b200 as mo
from moe_overlap_b200 import _lib
from tests.test_lora_gpu import make

pytestmark = pytest.mark.gpu


def _graph(device):
    x, w, a, b, dy, scale, ids = make(40, 64, 72, 3, 8, torch.bfloat16, device=device)
    p = [t.requires_grad_(True) for t in (x, a, b)]
    return mo.lora_linear(x, w, a, b, ids, scale=scale), p, dy


def test_a_backward_raises_what_was_recorded_before_it(cuda_device):
    y, p, dy = _graph(cuda_device)
    torch.cuda.synchronize()
    _lib.status_word(cuda_device)[0] = _lib.MOE_ERR_TIMEOUT
    with pytest.raises(mo.MoeError, match="earlier"):
        torch.autograd.grad(y, p, dy, retain_graph=True)
    assert int(_lib.status_word(cuda_device)[0]) == 0
    grads = torch.autograd.grad(y, p, dy)  # raised once; the graph is still good
    assert all(bool(g.isfinite().all()) for g in grads)


def _bound_with(ops, backward):
    lib = _lib.load()
    names = ("moe_few_tokens", "moe_few_tokens_workspace", "moe_lora_forward", "moe_lora_backward",
             "moe_lora_kept_bytes")
    fns = [backward if n == "moe_lora_backward" else getattr(lib, n) for n in names]
    ops.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in fns))


def test_a_backward_is_checked_at_once_where_that_is_asked_for(cuda_device, monkeypatch):
    """A stand-in for the library's backward that records an error as a kernel would, and one
    that returns an error."""
    y, p, dy = _graph(cuda_device)
    torch.cuda.synchronize()
    ops, real = _lib.torch_ops(), _lib.load().moe_lora_backward
    word = _lib.status_word(cuda_device)
    types = _lib.SIGNATURES["moe_lora_backward"][1]

    def records(*args):
        word[0] = _lib.MOE_ERR_TIMEOUT
        return _lib.MOE_OK

    fakes = [ctypes.CFUNCTYPE(ctypes.c_int32, *types)(f) for f in (records, lambda *args: _lib.MOE_ERR_CUDA)]
    try:
        _bound_with(ops, fakes[0])
        monkeypatch.setenv("MOE_B200_SYNC_CHECK", "1")
        with pytest.raises(mo.MoeError):
            torch.autograd.grad(y, p, dy, retain_graph=True)
        monkeypatch.delenv("MOE_B200_SYNC_CHECK")
        _bound_with(ops, fakes[1])
        with pytest.raises(mo.MoeError):
            torch.autograd.grad(y, p, dy, retain_graph=True)
    finally:
        _bound_with(ops, real)
        word[0] = 0
    monkeypatch.setenv("MOE_B200_SYNC_CHECK", "1")
    assert all(bool(g.isfinite().all()) for g in torch.autograd.grad(y, p, dy))
