"""Routing of tokens to experts, for ``moe_mlp``.

``route_experts(logits, top_k)`` returns ``(weights, ids)``: float32 and int32 ``[T, top_k]``, best first.  Per row x:

* scores ``s = softmax(x)`` or, with ``score="sigmoid"``, ``1 / (1 + exp(-x))``;
* choices ``c = s + bias`` (a bias that balances the experts' load changes who is chosen, not the weights);
* with ``num_groups`` > 1 only the experts of the ``top_groups`` best groups stay, a group's score being the sum of its
  ``group_top`` (1 or 2) largest choices;
* the ``top_k`` largest choices, ties to the lowest index; weights are their s, divided by their sum
  (``renormalize``), times ``scale``.

An expert whose logit or bias is -inf or NaN is off; a slot that no expert fills gets id -1 and weight 0, and
``moe_mlp`` skips it.  The ids are those of 64-bit arithmetic.
"""
from __future__ import annotations

import torch

from . import _lib

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_SCORES = {"softmax": 0, "sigmoid": 1}


def route_experts(logits: torch.Tensor, top_k: int, bias: torch.Tensor | None = None, score: str = "softmax",
                  num_groups: int = 1, top_groups: int = 1, group_top: int = 2, renormalize: bool = True,
                  scale: float = 1.0, weights: torch.Tensor | None = None, ids: torch.Tensor | None = None):
    if not isinstance(logits, torch.Tensor) or logits.dtype not in _DTYPES or logits.dim() != 2:
        raise TypeError("logits must be a 2-D float32, float16 or bfloat16 tensor [T, E]")
    index = logits.get_device()
    if index < 0:
        raise ValueError("logits must be a CUDA tensor")
    T, E = logits.shape
    strides = logits.stride()
    if E > 1 and strides[1] != 1:
        raise ValueError("logits must be contiguous along the experts")
    if score not in _SCORES:
        raise ValueError(f"score must be one of {sorted(_SCORES)}, got {score!r}")
    bias_at = None
    if bias is not None:
        if not isinstance(bias, torch.Tensor) or bias.dtype != torch.float32 or bias.shape != (E,) \
                or bias.get_device() != index or not bias.is_contiguous():
            raise ValueError(f"bias must be a contiguous float32 tensor [{E}] on the device of logits")
        bias_at = bias.data_ptr()
    if weights is None:
        weights = logits.new_empty((T, top_k), dtype=torch.float32)
    elif not isinstance(weights, torch.Tensor) or weights.dtype != torch.float32 or weights.shape != (T, top_k) \
            or weights.get_device() != index or not weights.is_contiguous():
        raise ValueError(f"weights must be a contiguous float32 tensor [{T}, {top_k}] on the device of logits")
    else:
        _lib.no_gradient("weights", weights)
    if ids is None:
        ids = logits.new_empty((T, top_k), dtype=torch.int32)
    elif not isinstance(ids, torch.Tensor) or ids.dtype != torch.int32 or ids.shape != (T, top_k) \
            or ids.get_device() != index or not ids.is_contiguous():
        raise ValueError(f"ids must be a contiguous int32 tensor [{T}, {top_k}] on the device of logits")
    _lib.call("nvfp4_route_experts", index, logits.data_ptr(), _DTYPES[logits.dtype], T, E, strides[0], bias_at,
              _SCORES[score], top_k, num_groups, top_groups, group_top, renormalize, scale, weights.data_ptr(),
              ids.data_ptr())
    return weights, ids
