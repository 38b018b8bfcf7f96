"""Low-rank adapters of many requests beside a shared projection.

``lora_add(base, x, a, b, adapters)`` adds to ``base``, what ``skinny_gemm`` / ``grouped_gemm`` wrote for the shared
weights, each token's own low-rank term, from the activations before their quantisation:

    out[t] = base[t] + scales[i] * ((x[t] . a[i]^T) . b[i]^T),   i = adapters[t]

* ``base`` fp16 ``[T, N]``, ``x`` fp16 ``[T, K]``, ``a`` fp16 ``[n, r, K]``, ``b`` fp16 ``[n, N, r]``: ``r`` is the
  largest rank, padded to a multiple of 16 (up to 128); ``ranks`` int32 ``[n]`` says how much of it each adapter uses,
  what lies beyond may hold anything;
* ``adapters`` int32 ``[T]`` on the GPU: an index outside ``[0, n)``, such as -1, is a token without an adapter;
* ``out`` is ``base`` (in place) unless given; it may not overlap ``x``, nor require a gradient outside of
  ``torch.no_grad()``: there is no backward pass.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib


def _half(name, t, dim, index):
    """Checks a half-precision operand on device `index`; its strides."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float16 or t.dim() != dim:
        raise TypeError(f"{name} must be a {dim}-D float16 tensor")
    if t.get_device() != index:
        raise ValueError(f"{name} must be on the device of base")
    strides = t.stride()
    if strides[-1] != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must be contiguous along its last dimension")
    return strides


def _vector(name, t, n, dtype, index):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.shape != (n,):
        raise ValueError(f"{name} must be a {dtype} tensor [{n}]")
    if t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous on the device of base")
    return t.data_ptr()


def lora_add(base, x, a, b, adapters, scales=None, ranks=None, out=None):
    if not isinstance(base, torch.Tensor):
        raise TypeError("base must be a 2-D float16 tensor")
    index = base.get_device()
    if index < 0:
        raise ValueError("base must be a CUDA tensor")
    s_base, s_x = _half("base", base, 2, index), _half("x", x, 2, index)
    s_a, s_b = _half("a", a, 3, index), _half("b", b, 3, index)
    T, N = base.shape
    n, r, K = a.shape
    if x.shape[0] != T:
        raise ValueError(f"x has {x.shape[0]} rows, expected {T}")
    if x.shape[1] != K or b.shape != (n, N, r):
        raise ValueError(f"a {tuple(a.shape)} and b {tuple(b.shape)} do not fit [n, r, {x.shape[1]}] and [n, {N}, r]")
    if out is None:
        out, s_out = base, s_base
    else:
        s_out = _half("out", out, 2, index)
        if out.shape != base.shape:
            raise ValueError(f"out has shape {tuple(out.shape)}, expected {tuple(base.shape)}")
    _lib.no_gradient("out (base, in place)", out)
    ad = _vector("adapters", adapters, T, torch.int32, index)
    sc = None if scales is None else _vector("scales", scales, n, torch.float32, index)
    rk = None if ranks is None else _vector("ranks", ranks, n, torch.int32, index)
    need = ctypes.c_int64(0)
    _lib.check(_lib.lib().nvfp4_lora_workspace(T, r, n, ctypes.byref(need)))
    ws = base.new_empty(need.value, dtype=torch.uint8) if need.value else None
    _lib.call("nvfp4_lora_add", index, base.data_ptr(), s_base[0], x.data_ptr(), s_x[0], a.data_ptr(), s_a[1], s_a[0],
              b.data_ptr(), s_b[1], s_b[0], ad, sc, rk, T, K, N, r, n, out.data_ptr(), s_out[0],
              None if ws is None else ws.data_ptr(), need.value)
    return out
