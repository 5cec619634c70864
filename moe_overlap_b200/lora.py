"""Low-rank adapters of many requests beside a projection that they share.

``lora_linear`` is the projection of a model that serves or trains many adapters at
once (the attention and shared projections around the routed experts, or the gate):
every row of the batch carries the id of its request's adapter.  The shared product is
the grouped GEMM of one expert, with the adapters' second product in its accumulator
where a tile of rows holds few adapters; decode batches have kernels of their own.
The reference has no counterpart.
"""
from __future__ import annotations

from typing import Union

import torch

from . import _lib

__all__ = ["lora_linear"]


def lora_linear(x: torch.Tensor, weight: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
                adapter_ids: torch.Tensor, *, scale: Union[float, torch.Tensor] = 1.0) -> torch.Tensor:
    """``y[m] = x[m] @ weight.T + scale[i] * (x[m] @ lora_a[i].T) @ lora_b[i].T``, i = adapter_ids[m].

    ``x`` [M, K], ``weight`` [N, K], ``lora_a`` [L, r, K] and ``lora_b`` [L, N, r] share a
    bf16 or fp16 type and a device; ranks up to 128 (pad smaller adapters with zeros),
    up to 1024 adapters.  ``adapter_ids`` [M] (int32 or int64) is in any order; -1 is a
    row without adapter, and an id outside [-1, L) counts as -1 and raises ``MoeError``
    at a later call.  ``scale`` is a number or a float tensor [L].

    Sums are fp32.  The product of rank r is rounded to the inputs' type, with its scale, as
    an operand of the shared product, whose sum is rounded once.  Decode batches hold it in
    fp32 instead; rows of tiles with too many adapters, and rows of fp16 whose operand the
    type does not hold (largest value beyond 65504 or below 2^-14), hold it in two parts of
    the type and are added to the rounded shared product.  So a row's last bit depends on
    the batch that it is in.

    Differentiable (once, in reverse mode) in ``x``, ``lora_a`` and ``lora_b``, with the
    gradients in the inputs' type.  For them the product of rank r is held in two parts of
    the type, in fp16 with a power of two, so that small gradients lose nothing.  The shared
    weight is frozen.  Sizes that are not multiples of 8, and rows that do not start on 16
    bytes, are copied with padding on every call.  The graph keeps about 10 r bytes a row
    beside its inputs, the workspace of its backward among them: passes over one graph may
    be repeated, but not from two threads at once.

    A training step can be captured into a CUDA graph (forward and backward together);
    as for every autograd graph, no graph of the same leaves from before the capture
    may be alive then, nor anything else that holds their gradient accumulators, which
    is refused: in the forward for inputs that are leaves, in the backward for leaves
    that the inputs were computed from.
    """
    if isinstance(scale, torch.Tensor):
        return _lib.torch_ops().lora_linear(x, weight, lora_a, lora_b, adapter_ids, scale, 0.0)
    return _lib.torch_ops().lora_linear(x, weight, lora_a, lora_b, adapter_ids, None, float(scale))
