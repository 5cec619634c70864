"""The routed-experts layer for a few tokens (decode batches).

``MoELayer.forward`` is built for thousands of rows: it exchanges them and runs
256-row tensor-core tiles.  At a handful of tokens the layer is a single pass over
the weights of the experts that some token takes, so these entry points stream those
weights once (src/train_moe_baseline.py:315-441 without the exchange):

* ``moe_few_tokens``: gate, top-k, experts and weighted sum;
* ``experts_few_tokens``: the same from a routing that the caller has.

Forward only.  Both can be captured into a CUDA graph and allocate only torch
tensors on the current stream.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib

__all__ = ["moe_few_tokens", "experts_few_tokens", "MAX_FEW_TOKENS"]

# Most tokens of one call; larger batches belong to MoELayer.forward.
MAX_FEW_TOKENS = 128

_DTYPE_CODE = {torch.bfloat16: _lib.MOE_DTYPE_BF16, torch.float16: _lib.MOE_DTYPE_F16}


def _row_strides(name: str, t: torch.Tensor, device, dtype):
    """The strides of ``t``, whose rows have to be unit-stride and start on 16 bytes (and
    whose matrices have to follow one another)."""
    if t.device != device or t.dtype != dtype:
        raise ValueError(f"{name} must be a {dtype} tensor on {device}")
    st, size = t.stride(), t.shape
    if st[-1] != 1 or st[-2] % 8 or st[-2] < size[-1] or t.data_ptr() % 16:
        raise ValueError(f"{name} needs unit-stride rows that start on 16 bytes")
    if len(st) == 3 and size[0] > 1 and (st[0] % 8 or st[0] < st[1] * size[1]):
        raise ValueError(f"{name}'s experts must follow one another")
    return st


def _run(x, router_w, router_bias, w1, w2, top_k, renormalize, idx, w, out):
    dev, dt = x.device, x.dtype
    if dev.type != "cuda":
        raise ValueError("few-token experts need CUDA tensors")
    if x.dim() != 2 or w1.dim() != 3 or w2.dim() != 3:
        raise ValueError("Shapes must be x [T, H], w1 [E, F, H], w2 [E, H, F].")
    tokens, hidden = x.shape
    experts, ffn, width = w1.shape
    if dt not in _DTYPE_CODE:
        raise ValueError("x must be bf16/fp16")
    if width != hidden or w2.shape != (experts, hidden, ffn):
        raise ValueError("Shapes must be x [T, H], w1 [E, F, H], w2 [E, H, F].")
    if hidden % 8 or ffn % 8 or hidden == 0 or ffn == 0:
        raise ValueError("hidden and ffn sizes must be multiples of 8")
    if tokens > MAX_FEW_TOKENS:
        raise ValueError(f"at most {MAX_FEW_TOKENS} tokens: use MoELayer.forward for larger batches")
    if not 1 <= top_k <= min(16, experts) or experts > 256:
        raise ValueError("top_k must be in 1..min(16, E), and E at most 256")
    ldx, unit = x.stride()
    if unit != 1 or ldx % 8 or ldx < hidden or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        ldx = hidden
    s1, s2 = _row_strides("w1", w1, dev, dt), _row_strides("w2", w2, dev, dt)
    if out is None:
        out = torch.empty(tokens, hidden, dtype=dt, device=dev)
        ldo = hidden
    elif out.shape != (tokens, hidden):
        raise ValueError("out must be [T, H]")
    else:
        ldo = _row_strides("out", out, dev, dt)[0]
    lib = _lib.load()
    _lib.check_status(dev)
    ws = torch.empty(lib.moe_few_tokens_workspace(tokens, hidden, ffn, experts, top_k),
                     dtype=torch.uint8, device=dev)
    with _lib.on_device(dev):
        rc = lib.moe_few_tokens(
            x.data_ptr(), ldx, router_w.data_ptr() if router_w is not None else None,
            router_w.stride(0) if router_w is not None else 0,
            router_bias.data_ptr() if router_bias is not None else None,
            w1.data_ptr(), s1[0], s1[1], w2.data_ptr(), s2[0], s2[1],
            _DTYPE_CODE[dt], tokens, hidden, ffn, experts, top_k, bool(renormalize),
            idx.data_ptr(), w.data_ptr(), out.data_ptr(), ldo, ws.data_ptr(), ws.numel(),
            _lib.status_address(dev), _lib.stream_handle(dev))
    _lib.check_call(rc, "moe_few_tokens")
    if _lib.sync_check_enabled():
        _lib.check_status(dev, sync=True)
    return out


def moe_few_tokens(x: torch.Tensor, router_w: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor,
                   top_k: int, *, router_bias: Optional[torch.Tensor] = None,
                   renormalize: bool = False, out: Optional[torch.Tensor] = None):
    """(out [T, H], topk_idx [T, k] int64, topk_w [T, k] fp32) of at most 128 tokens.

    ``x`` [T, H], ``router_w`` [E, H], ``w1`` [E, F, H] and ``w2`` [E, H, F] share a
    bf16 or fp16 type.  The gate's logits are held in 64 bits (``MoELayer.route``
    rounds them to bf16 first), the experts go by the logits with ties to the lower
    id; ``router_bias`` [E] and ``renormalize`` are as in ``router_topk``.  ``out``
    must not overlap ``x``.
    """
    top_k = int(top_k)
    if router_w.dim() != 2 or w1.dim() != 3 or router_w.shape != (w1.shape[0], x.shape[-1]):
        raise ValueError("router_w must be [E, H]")
    if x.device.type == "cuda":
        _row_strides("router_w", router_w, x.device, x.dtype)
    if router_bias is not None:
        if router_bias.shape != (router_w.shape[0],):
            raise ValueError("router bias must be [E]")
        router_bias = router_bias.to(device=x.device, dtype=torch.float32).contiguous()
    shape, dev = (x.shape[0], max(top_k, 0)), x.device
    idx = torch.empty(shape, dtype=torch.int64, device=dev)
    w = torch.empty(shape, dtype=torch.float32, device=dev)
    out = _run(x, router_w, router_bias, w1, w2, top_k, renormalize, idx, w, out)
    return out, idx, w


def experts_few_tokens(x: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, topk_idx: torch.Tensor,
                       topk_w: torch.Tensor, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[t] = sum_j topk_w[t, j] * (gelu(x[t] @ w1[e].T) @ w2[e].T)``, e = topk_idx[t, j].

    At most 128 tokens.  ``topk_idx`` [T, k] holds expert ids, -1 for a slot that is
    not routed (as the exchange takes them): a token whose slots are all -1, such as
    the padding of a batch, gets zeros.  The same expert may stand twice in a row.
    An id outside [-1, E) counts as -1 and raises ``MoeError`` at a later call.
    """
    if topk_idx.dim() != 2 or topk_idx.shape[0] != x.shape[0] or topk_w.shape != topk_idx.shape:
        raise ValueError("topk_idx and topk_w must be [T, k]")
    if topk_idx.device != x.device or topk_w.device != x.device:
        raise ValueError(f"topk_idx and topk_w must be on {x.device}")
    if topk_idx.dtype not in (torch.int64, torch.int32):
        raise ValueError("topk_idx must be int64 or int32")
    idx = topk_idx.to(torch.int64).contiguous()
    w = topk_w.to(torch.float32).contiguous()
    return _run(x, None, None, w1, w2, int(topk_idx.shape[1]), False, idx, w, out)
