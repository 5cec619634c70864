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
    ok = t.stride(-1) == 1 and t.stride(-2) % 8 == 0 and t.stride(-2) >= t.shape[-1]
    if t.dim() == 3 and t.shape[0] > 1:
        ok = ok and t.stride(0) % 8 == 0 and t.stride(0) >= t.stride(1) * t.shape[1]
    if ok and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


class _Plan:
    """The batch's rows by adapter: ``perm`` [M], ``offs`` [L + 1] and ``base`` {0, M}."""

    def __init__(self, ids: torch.Tensor, adapters: int):
        m, dev = ids.shape[0], ids.device
        buf = torch.empty(m + adapters + 3, dtype=torch.int32, device=dev)
        self.perm, self.offs, self.base = buf[:m], buf[m:m + adapters + 1], buf[m + adapters + 1:]
        rc = _lib.load().moe_lora_plan(ids.data_ptr(), int(ids.dtype == torch.int64), m, adapters,
                                       self.perm.data_ptr(), self.offs.data_ptr(),
                                       self.base.data_ptr(), _lib.status_word(dev).data_ptr(),
                                       _lib.stream_handle(dev))
        _lib.check_call(rc, "moe_lora_plan")


def _shared(x, w, stride_k, stride_n, n, plan):
    """The shared product as the grouped GEMM of one expert, w[k, n] at the given strides.

    The C entry directly: a bad adapter id, which the plan may just have recorded, is
    raised by a later call and not by the middle of this one."""
    m, k = x.shape
    y = torch.empty(m, n, dtype=x.dtype, device=x.device)
    sms = torch.cuda.get_device_properties(x.device).multi_processor_count
    rc = _lib.load().moe_grouped_gemm(x.data_ptr(), x.stride(0), w.data_ptr(), 0, stride_k, stride_n,
                                      y.data_ptr(), n, plan.base.data_ptr(), 0, m, k, n, 1,
                                      _DTYPE_CODE[x.dtype], _lib.MOE_ACT_NONE, sms, 0, None,
                                      _lib.status_word(x.device).data_ptr(),
                                      _lib.stream_handle(x.device))
    _lib.check_call(rc, "moe_grouped_gemm")
    return y


def _shrink(x, w, transposed, plan, rank):
    m, k = x.shape
    s = torch.empty(2, m, rank, dtype=x.dtype, device=x.device)
    rc = _lib.load().moe_lora_shrink(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), w.stride(1),
                                     int(transposed), plan.perm.data_ptr(), plan.offs.data_ptr(),
                                     _DTYPE_CODE[x.dtype], m, k, w.shape[0], rank, s.data_ptr(),
                                     _lib.stream_handle(x.device))
    _lib.check_call(rc, "moe_lora_shrink")
    return s


def _expand(s, w, transposed, scale, plan, y):
    m, n = y.shape
    rc = _lib.load().moe_lora_expand(s.data_ptr(), w.data_ptr(), w.stride(0), w.stride(1),
                                     int(transposed), scale.data_ptr(), plan.perm.data_ptr(),
                                     plan.offs.data_ptr(), _DTYPE_CODE[y.dtype], m, n, w.shape[0],
                                     s.shape[2], y.data_ptr(), y.stride(0), _lib.stream_handle(y.device))
    _lib.check_call(rc, "moe_lora_expand")


def _grad(s, z, scale, plan, like, transposed):
    g = torch.empty(like.shape, dtype=like.dtype, device=like.device)
    m, n = z.shape
    rc = _lib.load().moe_lora_grad(s.data_ptr(), z.data_ptr(), z.stride(0), scale.data_ptr(),
                                   plan.perm.data_ptr(), plan.offs.data_ptr(), _DTYPE_CODE[z.dtype],
                                   m, n, like.shape[0], s.shape[2], g.data_ptr(), g.stride(0),
                                   g.stride(1), int(transposed), _lib.stream_handle(z.device))
    _lib.check_call(rc, "moe_lora_grad")
    return g


class LoraLinear(torch.autograd.Function):
    """x [M, K], lora_a [L, r, K], lora_b [L, N, r] -> y [M, N]; the weight, the ids and
    the scale get no gradient."""

    @staticmethod
    def forward(ctx, x, weight, lora_a, lora_b, ids, scale):
        with torch.cuda.device(x.device):
            plan = _Plan(ids, lora_a.shape[0])
            s = _shrink(x, lora_a, False, plan, lora_a.shape[1])
            y = _shared(x, weight, 1, weight.stride(0), weight.shape[0], plan)
            _expand(s, lora_b, False, scale, plan, y)
        ctx.save_for_backward(x, weight, lora_a, lora_b, scale, s)
        ctx.plan = plan
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, lora_a, lora_b, scale, s = ctx.saved_tensors
        plan = ctx.plan
        need_x, _, need_a, need_b, _, _ = ctx.needs_input_grad
        dx = da = db = None
        dy = _rows(dy)
        with torch.cuda.device(x.device):
            if need_x or need_a:
                back = _shrink(dy, lora_b, True, plan, lora_a.shape[1])
            if need_x:
                dx = _shared(dy, weight, weight.stride(0), 1, weight.shape[1], plan)
                _expand(back, lora_a, True, scale, plan, dx)
            if need_a:
                da = _grad(back, x, scale, plan, lora_a, True)
            if need_b:
                db = _grad(s, dy, scale, plan, lora_b, False)
        return dx, None, da, db, None, None


_EAGER = "moe_overlap_b200.lora_linear ran outside a capture"


def _leaf_nodes(*tensors):
    """The gradient accumulators of the leaves among ``tensors``, to be held until the
    forward's graph holds them.

    An accumulator belongs to the stream that it was made on and lives as long as any
    graph of its leaf.  One left from a call outside would pull that stream into a
    captured backward and break the capture in the autograd engine, so such a call
    marks it, and a call under capture that finds the mark is refused here instead.
    """
    if not torch.is_grad_enabled():
        return []
    capturing = torch.cuda.is_current_stream_capturing()
    nodes = [torch.autograd.graph.get_gradient_edge(t).node for t in tensors
             if t.requires_grad and t.is_leaf]
    for node in nodes:
        if not capturing:
            node.metadata[_EAGER] = True
        elif _EAGER in node.metadata:
            raise RuntimeError("lora_linear: a graph of the same inputs from a call outside the capture "
                               "is alive; drop its outputs before capturing a training step")
    return nodes


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
    if x.device.type != "cuda":
        raise ValueError("lora_linear requires CUDA tensors.")
    if x.dim() != 2 or weight.dim() != 2 or lora_a.dim() != 3 or lora_b.dim() != 3:
        raise ValueError("Shapes must be x [M, K], weight [N, K], lora_a [L, r, K], lora_b [L, N, r].")
    (m, k), n = x.shape, weight.shape[0]
    adapters, rank, _ = lora_a.shape
    if weight.shape != (n, k) or lora_a.shape[2] != k or lora_b.shape != (adapters, n, rank):
        raise ValueError("Shapes must be x [M, K], weight [N, K], lora_a [L, r, K], lora_b [L, N, r].")
    if k == 0 or n == 0 or not 1 <= rank <= MAX_RANK or not 1 <= adapters <= MAX_ADAPTERS:
        raise ValueError(f"ranks go from 1 to {MAX_RANK}, adapters from 1 to {MAX_ADAPTERS}, and K "
                         "and N must not be 0")
    if x.dtype not in _DTYPE_CODE:
        raise ValueError("x dtype must be bf16/fp16.")
    for name, t in (("weight", weight), ("lora_a", lora_a), ("lora_b", lora_b)):
        if t.dtype != x.dtype or t.device != x.device:
            raise ValueError(f"{name} must be a {x.dtype} tensor on {x.device}")
    if adapter_ids.shape != (m,) or adapter_ids.device != x.device or \
            adapter_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"adapter_ids must be an int32 or int64 tensor [M] on {x.device}")
    if weight.requires_grad and torch.is_grad_enabled():
        raise ValueError("the shared weight is frozen: lora_linear gives it no gradient")
    if isinstance(scale, torch.Tensor):
        if scale.shape != (adapters,) or not scale.is_floating_point():
            raise ValueError("scale must be a number or a float tensor [L]")
        if scale.requires_grad and torch.is_grad_enabled():
            raise ValueError("lora_linear gives the scale no gradient")
        scale = scale.to(device=x.device, dtype=torch.float32).contiguous()
    else:
        scale = torch.full((adapters,), float(scale), dtype=torch.float32, device=x.device)
    _lib.check_status(x.device)
    nodes = _leaf_nodes(x, lora_a, lora_b)
    pk, pn, pr = -k % 8, -n % 8, -rank % 8
    y = LoraLinear.apply(_rows(_pad(x, pk)), _rows(_pad(weight, pk, pn)), _rows(_pad(lora_a, pk, pr)),
                         _rows(_pad(lora_b, pr, pn)), adapter_ids.contiguous(), scale)
    del nodes
    if _lib.sync_check_enabled():
        _lib.check_status(x.device, sync=True)
    return y[:, :n] if pn else y
