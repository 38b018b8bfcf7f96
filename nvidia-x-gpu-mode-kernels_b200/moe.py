"""The experts' SiLU-gated MLP on NVFP4 weights, for tokens that chose their experts.

``moe_mlp(x, ids, weights, w_gate, w_up, w_down, scale_gate, scale_up, scale_down)`` returns fp16 ``[T, D]``:

    out[t] = sum_j weights[t, j] * (nvfp4(silu(xq . w_gate[e]^T) * (xq . w_up[e]^T)) . w_down[e]^T),
    e = ids[t, j],  xq = nvfp4(x[t])

* ``x`` fp16 ``[T, D]``; ``ids`` int32 and ``weights`` float32 ``[T, k]``, as ``route_experts`` returns them.  A slot
  with an id outside ``[0, E)`` is skipped; the same expert twice in a row counts twice.
* codes ``[E, F, D/2]`` (gate, up: same strides, so halves of one merged tensor will do) and ``[E, D, F/2]`` (down);
* scales per expert in the 128x4 blocked layout, ``[E, layout.blocked_numel(rows, K/16)]``, or plain ``[E, rows, K/16]``
  (converted here, which costs extra launches).

How many tokens an expert gets stays on the GPU: no synchronisation, and the call can be captured in a CUDA graph.  The
workspace comes from torch's allocator, on the current stream.
"""
from __future__ import annotations

import torch

from . import _lib
from .gemm import _FP4, _FP8
from .layout import blocked_numel, to_blocked


def _weights(name, w, shape, index):
    """Checks the codes of all experts' matrices of one kind; their strides."""
    if not isinstance(w, torch.Tensor) or w.dtype not in _FP4 or w.dim() != 3:
        raise TypeError(f"{name} must be a 3-D uint8 / float4_e2m1fn_x2 tensor [E, rows, K/2]")
    if w.shape != shape:
        raise ValueError(f"{name} has shape {tuple(w.shape)}, expected {shape}")
    strides = w.stride()
    if strides[2] != 1:
        raise ValueError(f"{name} must be contiguous along K")
    if w.get_device() != index:
        raise ValueError(f"{name} must be on the device of x")
    return strides


def _expert_scales(name, s, E, N, K, index):
    if not isinstance(s, torch.Tensor) or s.dtype not in _FP8:
        raise TypeError(f"{name} must be a uint8 / float8_e4m3fn tensor")
    if s.get_device() != index:
        raise ValueError(f"{name} must be on the device of x")
    if s.shape == (E, N, K // 16):
        return torch.stack([to_blocked(s[e]) for e in range(E)])
    if s.shape != (E, blocked_numel(N, K // 16)) or s.stride(1) != 1:
        raise ValueError(f"{name}: expected plain [{E}, {N}, {K // 16}] or blocked [{E}, {blocked_numel(N, K // 16)}] "
                         f"with contiguous bytes, got shape {tuple(s.shape)}")
    return s


def moe_mlp(x, ids, weights, w_gate, w_up, w_down, scale_gate, scale_up, scale_down, out=None):
    if not isinstance(x, torch.Tensor) or x.dtype != torch.float16 or x.dim() != 2:
        raise TypeError("x must be a 2-D float16 tensor [T, D]")
    index = x.get_device()
    if index < 0:
        raise ValueError("x must be a CUDA tensor")
    T, D = x.shape
    s_x = x.stride()
    if s_x[1] != 1:
        raise ValueError("x must be contiguous along D")
    if not isinstance(ids, torch.Tensor) or ids.dtype != torch.int32 or ids.dim() != 2:
        raise TypeError("ids must be a 2-D int32 tensor [T, k]")
    k = ids.shape[1]
    if ids.shape[0] != T or not ids.is_contiguous() or ids.get_device() != index:
        raise ValueError(f"ids must be contiguous [{T}, k] on the device of x, got {tuple(ids.shape)}")
    if not isinstance(weights, torch.Tensor) or weights.dtype != torch.float32:
        raise TypeError("weights must be a float32 tensor [T, k]")
    if weights.shape != ids.shape or not weights.is_contiguous() or weights.get_device() != index:
        raise ValueError(f"weights must be contiguous {tuple(ids.shape)} on the device of x, got {tuple(weights.shape)}")
    if not isinstance(w_gate, torch.Tensor) or w_gate.dim() != 3:
        raise TypeError("w_gate must be a 3-D uint8 / float4_e2m1fn_x2 tensor [E, F, D/2]")
    E, F, _ = w_gate.shape
    s_in = _weights("w_gate", w_gate, (E, F, D // 2), index)
    s_up = _weights("w_up", w_up, (E, F, D // 2), index)
    s_down = _weights("w_down", w_down, (E, D, F // 2), index)
    sg = _expert_scales("scale_gate", scale_gate, E, F, D, index)
    su = _expert_scales("scale_up", scale_up, E, F, D, index)
    sd = _expert_scales("scale_down", scale_down, E, D, F, index)
    sfe = sg.stride(0)
    if s_in != s_up or sfe != su.stride(0):
        raise ValueError("w_gate and w_up, and their scales, must have the same strides")
    if out is None:
        out = torch.empty((T, D), dtype=torch.float16, device=x.device)
    elif not isinstance(out, torch.Tensor) or out.dtype != torch.float16 or out.shape != (T, D) \
            or out.stride(1) != 1 or out.get_device() != index:
        raise ValueError(f"out must be a float16 [{T}, {D}] tensor with unit column stride on the device of x")
    else:
        _lib.no_gradient("out", out)
    need = _lib.query("nvfp4_moe_workspace", index, T, k, E, D, F)
    ws = x.new_empty(need, dtype=torch.uint8)
    _lib.call("nvfp4_moe_mlp", index, x.data_ptr(), s_x[0], ids.data_ptr(), weights.data_ptr(), T, k, E, D, F,
              w_gate.data_ptr(), w_up.data_ptr(), sg.data_ptr(), su.data_ptr(), s_in[1], s_in[0], sfe,
              w_down.data_ptr(), sd.data_ptr(), s_down[1], s_down[0], sd.stride(0), out.data_ptr(), out.stride(0),
              ws.data_ptr(), need)
    return out
