"""Low-rank adapters of many requests beside a projection that they share.

``lora_linear`` is the projection of a model that serves or trains many adapters at
once (the attention and shared projections around the routed experts, or the gate):
every row of the batch carries the id of its request's adapter.  The shared product is
the grouped GEMM of one expert (``moe_grouped_gemm``); the adapters' part and its
gradients are this package's kernels.  The reference has no counterpart.
"""
from __future__ import annotations

from typing import Union

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["lora_linear"]

_DTYPE_CODE = {torch.bfloat16: _lib.MOE_DTYPE_BF16, torch.float16: _lib.MOE_DTYPE_F16}
MAX_RANK = 128
MAX_ADAPTERS = 1024


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with unit-stride rows (and adapters) that start on 16 bytes, copied if needed."""
    if t.is_contiguous() and t.shape[-1] % 8 == 0 and t.data_ptr() % 16 == 0:
        return t
    ok = t.stride(-1) == 1 and t.stride(-2) % 8 == 0 and t.stride(-2) >= t.shape[-1]
    if t.dim() == 3 and t.shape[0] > 1:
        ok = ok and t.stride(0) % 8 == 0 and t.stride(0) >= t.stride(1) * t.shape[1]
    if ok and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _forward(x, weight, lora_a, lora_b, ids, scale, for_backward):
    """(y, the buffer that the backward needs)."""
    (m, k), n = x.shape, weight.shape[0]
    adapters, rank, _ = lora_a.shape
    dev, dt = x.device, x.dtype
    lib = _lib.load()
    sa, sb = lora_a.stride(), lora_b.stride()
    each, all_ = (scale.data_ptr(), 0.0) if isinstance(scale, torch.Tensor) else (None, scale)
    y = torch.empty(m, n, dtype=dt, device=dev)
    kept = torch.empty(lib.moe_lora_kept_bytes(m, adapters, rank, for_backward), dtype=torch.uint8, device=dev)
    with _lib.on_device(dev):
        rc = lib.moe_lora_forward(
            x.data_ptr(), x.stride(0), weight.data_ptr(), weight.stride(0), lora_a.data_ptr(), sa[0], sa[1],
            lora_b.data_ptr(), sb[0], sb[1], ids.data_ptr(), ids.dtype == torch.int64, each, all_,
            _DTYPE_CODE[dt], m, k, n, adapters, rank, for_backward, y.data_ptr(), n, kept.data_ptr(),
            _lib.status_address(dev), _lib.stream_handle(dev))
    _lib.check_call(rc, "moe_lora_forward")
    return y, kept


class LoraLinear(torch.autograd.Function):
    """x [M, K], lora_a [L, r, K], lora_b [L, N, r] -> y [M, N]; the weight, the ids and
    the scale get no gradient."""

    @staticmethod
    def forward(ctx, x, weight, lora_a, lora_b, ids, scale):
        y, kept = _forward(x, weight, lora_a, lora_b, ids, scale, True)
        ctx.save_for_backward(x, weight, lora_a, lora_b, kept)
        ctx.scale = scale
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, lora_a, lora_b, kept = ctx.saved_tensors
        need = ctx.needs_input_grad
        (m, k), n = x.shape, weight.shape[0]
        adapters, rank, _ = lora_a.shape
        dev, dt, scale = x.device, x.dtype, ctx.scale
        sa, sb = lora_a.stride(), lora_b.stride()
        each, all_ = (scale.data_ptr(), 0.0) if isinstance(scale, torch.Tensor) else (None, scale)
        dy = _rows(dy)
        dx = torch.empty(m, k, dtype=dt, device=dev) if need[0] else None
        da = torch.empty(adapters, rank, k, dtype=dt, device=dev) if need[2] else None
        db = torch.empty(adapters, n, rank, dtype=dt, device=dev) if need[3] else None
        with _lib.on_device(dev):
            rc = _lib.load().moe_lora_backward(
                dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), weight.data_ptr(), weight.stride(0),
                lora_a.data_ptr(), sa[0], sa[1], lora_b.data_ptr(), sb[0], sb[1], each, all_,
                _DTYPE_CODE[dt], m, k, n, adapters, rank, kept.data_ptr(),
                dx.data_ptr() if dx is not None else None, k, da.data_ptr() if da is not None else None,
                db.data_ptr() if db is not None else None, _lib.status_address(dev), _lib.stream_handle(dev))
        _lib.check_call(rc, "moe_lora_backward")
        return dx, None, da, db, None, None


_EAGER = "moe_overlap_b200.lora_linear ran outside a capture"


def _guard_capture(y, inputs, given):
    """Refuses a capture that could not be used.

    The gradient accumulator of a leaf belongs to the stream that it was made on and
    lives as long as any graph of the leaf.  One left from a call outside would pull
    that stream into a captured backward and break the capture in the autograd engine;
    so a call outside marks the accumulators, and a call under capture that finds the
    mark is refused here instead.
    """
    capturing = torch.cuda.is_current_stream_capturing()
    edges = y.grad_fn.next_functions
    for at in (0, 2, 3):  # x, lora_a, lora_b
        t = given[at]
        if not (t.requires_grad and t.is_leaf):
            continue
        node = edges[at][0] if inputs[at] is t else torch.autograd.graph.get_gradient_edge(t).node
        if not capturing:
            node.metadata[_EAGER] = True
        elif _EAGER in node.metadata:
            raise RuntimeError("lora_linear: a graph of the same inputs from a call outside the capture "
                               "is alive; drop its outputs before capturing a training step")


def _pad(t: torch.Tensor, *by: int) -> torch.Tensor:
    """``t`` with its last dimensions padded by zeros at the end (last dimension first)."""
    if not any(by):
        return t
    return F.pad(t, [v for n in by for v in (0, n)])


def lora_linear(x: torch.Tensor, weight: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
                adapter_ids: torch.Tensor, *, scale: Union[float, torch.Tensor] = 1.0) -> torch.Tensor:
    """``y[m] = x[m] @ weight.T + scale[i] * (x[m] @ lora_a[i].T) @ lora_b[i].T``, i = adapter_ids[m].

    ``x`` [M, K], ``weight`` [N, K], ``lora_a`` [L, r, K] and ``lora_b`` [L, N, r] share a
    bf16 or fp16 type and a device; ranks up to 128 (pad smaller adapters with zeros),
    up to 1024 adapters.  ``adapter_ids`` [M] (int32 or int64) is in any order; -1 is a
    row without adapter, and an id outside [-1, L) counts as -1 and raises ``MoeError``
    at a later call.  ``scale`` is a number or a float tensor [L].

    Differentiable in ``x``, ``lora_a`` and ``lora_b`` (sums in fp32, the gradients in
    the inputs' type; the product of rank r between the two is held in two parts of that
    type); the shared weight is frozen.  Sizes that are not multiples of 8, and rows that do not
    start on 16 bytes, are copied with padding on every call.

    A training step can be captured into a CUDA graph (forward and backward together);
    as for every autograd graph, no graph of the same leaves from before the capture
    may be alive then.
    """
    dev, dt = x.device, x.dtype
    if dev.type != "cuda":
        raise ValueError("lora_linear requires CUDA tensors.")
    if x.dim() != 2 or weight.dim() != 2 or lora_a.dim() != 3 or lora_b.dim() != 3:
        raise ValueError("Shapes must be x [M, K], weight [N, K], lora_a [L, r, K], lora_b [L, N, r].")
    (m, k), n = x.shape, weight.shape[0]
    adapters, rank, width = lora_a.shape
    if weight.shape != (n, k) or width != k or lora_b.shape != (adapters, n, rank):
        raise ValueError("Shapes must be x [M, K], weight [N, K], lora_a [L, r, K], lora_b [L, N, r].")
    if k == 0 or n == 0 or not 1 <= rank <= MAX_RANK or not 1 <= adapters <= MAX_ADAPTERS:
        raise ValueError(f"ranks go from 1 to {MAX_RANK}, adapters from 1 to {MAX_ADAPTERS}, and K "
                         "and N must not be 0")
    if dt not in _DTYPE_CODE:
        raise ValueError("x dtype must be bf16/fp16.")
    for name, t in (("weight", weight), ("lora_a", lora_a), ("lora_b", lora_b)):
        if t.dtype != dt or t.device != dev:
            raise ValueError(f"{name} must be a {dt} tensor on {dev}")
    if adapter_ids.shape != (m,) or adapter_ids.device != dev or \
            adapter_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"adapter_ids must be an int32 or int64 tensor [M] on {dev}")
    if weight.requires_grad and torch.is_grad_enabled():
        raise ValueError("the shared weight is frozen: lora_linear gives it no gradient")
    if isinstance(scale, torch.Tensor):
        if scale.shape != (adapters,) or not scale.is_floating_point():
            raise ValueError("scale must be a number or a float tensor [L]")
        if scale.requires_grad and torch.is_grad_enabled():
            raise ValueError("lora_linear gives the scale no gradient")
        if scale.dtype != torch.float32 or scale.device != dev or not scale.is_contiguous():
            scale = scale.to(device=dev, dtype=torch.float32).contiguous()
    else:
        scale = float(scale)
    _lib.check_status(dev)
    pk, pn, pr = -k % 8, -n % 8, -rank % 8
    if not (pk or pn or pr) and x.is_contiguous() and weight.is_contiguous() and lora_a.is_contiguous() \
            and lora_b.is_contiguous() and adapter_ids.is_contiguous() \
            and not (x.data_ptr() | weight.data_ptr() | lora_a.data_ptr() | lora_b.data_ptr()) & 15:
        args = (x, weight, lora_a, lora_b, adapter_ids, scale)
    elif pk or pn or pr:
        args = (_rows(_pad(x, pk)), _rows(_pad(weight, pk, pn)), _rows(_pad(lora_a, pk, pr)),
                _rows(_pad(lora_b, pr, pn)), adapter_ids.contiguous(), scale)
    else:
        args = (_rows(x), _rows(weight), _rows(lora_a), _rows(lora_b), adapter_ids.contiguous(), scale)
    if torch.is_grad_enabled() and (x.requires_grad or lora_a.requires_grad or lora_b.requires_grad):
        y = LoraLinear.apply(*args)
        _guard_capture(y, args, (x, weight, lora_a, lora_b))
    else:
        y, _ = _forward(*args, False)
    if _lib.sync_check_enabled():
        _lib.check_status(x.device, sync=True)
    return y[:, :n] if pn else y
