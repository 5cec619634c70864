"""The routed-experts layer for a few tokens (decode batches).

``MoELayer.forward`` is built for thousands of rows: it exchanges them and runs
256-row tensor-core tiles.  At a handful of tokens the layer is a single pass over
the weights of the experts that some token takes, so these entry points stream those
weights (src/train_moe_baseline.py:315-441 without the exchange):

* ``moe_few_tokens``: gate, top-k, experts and weighted sum;
* ``experts_few_tokens``: the same from a routing that the caller has.

Forward only: inputs that require a gradient are refused while gradients are recorded.
Both can be captured into a CUDA graph and allocate only torch tensors on the current
stream.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib

__all__ = ["moe_few_tokens", "experts_few_tokens", "MAX_FEW_TOKENS"]

# Most tokens of one call; larger batches belong to MoELayer.forward.  Measured on one
# B200, forward and here: 128 tokens, top-2 of 16 x 2048 x 8192 335 and 221 us, top-8 of
# 64 x 2048 x 1024 324 and 141; with many slots an expert forward is the faster one
# earlier: top-8 of 9 x 1712 x 6320 335 and 206 us at 64 tokens, 327 and 394 at 128.
MAX_FEW_TOKENS = 128


def moe_few_tokens(x: torch.Tensor, router_w: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor,
                   top_k: int, *, router_bias: Optional[torch.Tensor] = None,
                   renormalize: bool = False, out: Optional[torch.Tensor] = None):
    """(out [T, H], topk_idx [T, k] int64, topk_w [T, k] fp32) of at most 128 tokens.

    ``x`` [T, H], ``router_w`` [E, H], ``w1`` [E, F, H] and ``w2`` [E, H, F] share a
    bf16 or fp16 type.  gelu(x W1^T) is held to 16 bits in bf16, in fp16 to 22 bits down
    to 2^-25 and up to 131008; the output is rounded once.  The gate's logits are held in 64 bits (``MoELayer.route``
    rounds them to bf16 first), the experts go by the logits with ties to the lower
    id; ``router_bias`` [E] and ``renormalize`` are as in ``router_topk``.  ``out``
    must not overlap ``x``.
    """
    return _lib.torch_ops().moe_few_tokens(x, router_w, w1, w2, top_k, router_bias, renormalize, out)


def experts_few_tokens(x: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, topk_idx: torch.Tensor,
                       topk_w: torch.Tensor, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[t] = sum_j topk_w[t, j] * (gelu(x[t] @ w1[e].T) @ w2[e].T)``, e = topk_idx[t, j].

    At most 128 tokens.  ``topk_idx`` [T, k] holds expert ids, -1 for a slot that is
    not routed (as the exchange takes them): a token whose slots are all -1, such as
    the padding of a batch, gets zeros.  The same expert may stand twice in a row.
    An id outside [-1, E) counts as -1 and raises ``MoeError`` at a later call.
    """
    return _lib.torch_ops().experts_few_tokens(x, w1, w2, topk_idx, topk_w, out)
