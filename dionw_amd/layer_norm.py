"""Layer norm over the last dimension, and the norm whose output is quantized to 4 bits as it is made.

- ``layer_norm(x, weight, bias, eps)``: ``(x - mean) / sqrt(variance + eps) * weight + bias`` of each
  row, differentiable.
- ``LayerNorm``: ``nn.LayerNorm`` with it.
- ``float4_layer_norm``: the same rows as a ``Float4Matrix``, for ``float4_matmul`` with a kept weight:
  a prompt's norm and the quantization behind it in one reading of x.

x, the parameters and their gradients are float16, bfloat16 or float32, each in a type of its own;
statistics and sums are float32 throughout.
"""

from __future__ import annotations

import math
from functools import lru_cache
from typing import Any

import torch
from torch import Tensor, nn

from dionw_amd import _lib
from dionw_amd._operands import (
    CODES,
    call,
    check_unrecorded,
    check_vector,
    once_differentiable,
    pitch,
    readable,
    scratch,
    watched,
)
from dionw_amd.float4 import Float4Matrix, empty

__all__ = ["LayerNorm", "float4_layer_norm", "layer_norm"]


def _rows(x: Tensor, weight: Tensor | None, bias: Tensor | None) -> Tensor:
    """x as a matrix, once the arguments fit each other."""
    if x.dim() == 0 or x.shape[-1] == 0 or x.dtype not in CODES:
        raise ValueError("layer norm takes float16, bfloat16 or float32 rows of one value at least, got "
                         f"{x.dtype} of shape {tuple(x.shape)}")
    cols = x.shape[-1]
    check_vector("norm's weight", weight, cols, x.device)
    check_vector("norm's bias", bias, cols, x.device)
    return x if x.dim() == 2 else x.reshape(math.prod(x.shape[:-1]), cols)


def _parameter(p: Tensor | None) -> tuple[int, Tensor | None]:
    """A parameter as the kernels read it, held by the caller until the library call has returned."""
    return (_lib.F32, None) if p is None else (CODES[p.dtype], p if p.is_contiguous() else p.contiguous())


def _forward(x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float,
             keep: bool) -> tuple[Tensor, Tensor | None]:
    """y of a readable matrix, and its rows' means and reciprocal deviations, [2, rows]."""
    (m, n), device = x.shape, x.device
    stream = _lib.stream_handle(device)
    y = torch.empty(m, n, dtype=x.dtype, device=device)
    stats = torch.empty(2, m, dtype=torch.float32, device=device) if keep else None
    (w_code, weight), (b_code, bias) = _parameter(weight), _parameter(bias)
    at = (None, None) if stats is None else (stats.data_ptr(), stats.data_ptr() + 4 * m)
    call(device, "dionw_layer_norm_forward", CODES[x.dtype], x.data_ptr(), pitch(x), m, n, w_code,
         _lib.ptr(weight), b_code, _lib.ptr(bias), eps, y.data_ptr(), *at, stream)
    return y, stats


@lru_cache(maxsize=256)
def _backward_scratch(rows: int, cols: int) -> int:
    return _lib.library().dionw_layer_norm_backward_scratch(rows, cols)


class _Norm(torch.autograd.Function):
    """y = u g + b, u = (x - mean) / deviation; dx = (w - mean(w) - u mean(w u)) / deviation with
    w = dy g, dg = the sum of dy u over the rows, db = that of dy."""

    @staticmethod
    def forward(ctx: Any, x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float) -> Tensor:
        x = readable(x)
        y, stats = _forward(x, weight, bias, eps, any(ctx.needs_input_grad))
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.save_for_backward(x, weight, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dy: Tensor) -> tuple[Tensor | None, ...]:
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        x, weight, stats = ctx.saved_tensors
        (m, n), device = x.shape, x.device
        dy = readable(dy)
        w_code, gain = _parameter(weight)
        stream = _lib.stream_handle(device)
        dx = torch.empty(m, n, dtype=x.dtype, device=device) if need_x else None
        dg = torch.empty(n, dtype=weight.dtype, device=device) if need_w else None
        db = torch.empty(n, dtype=ctx.bias_dtype, device=device) if need_b else None
        size = _backward_scratch(m, n) if need_w or need_b else 0
        space = scratch(size, device)
        call(device, "dionw_layer_norm_backward", CODES[x.dtype], x.data_ptr(), pitch(x), dy.data_ptr(),
             pitch(dy), m, n, w_code, _lib.ptr(gain), stats.data_ptr(), stats.data_ptr() + 4 * m, _lib.ptr(dx),
             _lib.ptr(dg), CODES[ctx.bias_dtype] if need_b else _lib.F32, _lib.ptr(db), _lib.ptr(space), size,
             stream)
        return dx, dg, db, None


def layer_norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None,
               eps: float = 1e-5) -> Tensor:
    """``(x - mean) / sqrt(variance + eps) * weight + bias`` over the last dimension, in x's type.

    The variance is the biased one. ``weight`` and ``bias`` are vectors of that dimension in any of
    the types, or absent. Gradients flow to x, weight and bias, each in its own type. Under
    ``torch.autocast`` a 16-bit x is cast to float32, as for ``nn.LayerNorm``.

    Raises:
        ValueError: For shapes or types that do not fit, an empty last dimension, tensors off the
            GPU, forward-mode duals, or calls that ``torch.jit.trace`` or ``make_fx`` records.
    """
    if watched():
        check_unrecorded(x, weight, bias)
    if torch.is_autocast_enabled() and x.dtype in CODES:
        x = x.to(torch.float32)
    flat = _rows(x, weight, bias)
    if torch.is_grad_enabled():
        y = _Norm.apply(flat, weight, bias, eps)
    else:
        y = _forward(readable(flat), weight, bias, eps, False)[0]
    return y if x.dim() == 2 else y.view(x.shape)


def float4_layer_norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None,
                      eps: float = 1e-5) -> Float4Matrix:
    """``layer_norm``'s rows (all leading dimensions taken together) quantized to 4 bits as
    ``float4_quantize`` does to nearest, without being rounded to x's type first.

    Raises:
        ValueError: As ``layer_norm``; and for arguments that require a gradient, which it has not.
    """
    if watched():
        check_unrecorded(x, weight, bias)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        raise ValueError("float4_layer_norm is for inference: use layer_norm and float4_linear where "
                         "gradients are needed, or call under torch.no_grad()")
    flat = readable(_rows(x, weight, bias))
    (m, n), device = flat.shape, flat.device
    stream = _lib.stream_handle(device)
    q = empty(m, n, device)
    (w_code, weight), (b_code, bias) = _parameter(weight), _parameter(bias)
    call(device, "dionw_layer_norm_float4", CODES[flat.dtype], flat.data_ptr(), pitch(flat), m, n, w_code,
         _lib.ptr(weight), b_code, _lib.ptr(bias), eps, q.data.data_ptr(), q.scale.data_ptr(), q.scale.shape[1],
         stream)
    return q


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` on ``layer_norm``; several normalized dimensions are taken as one."""

    def forward(self, input: Tensor) -> Tensor:
        dims = len(self.normalized_shape)
        if input.shape[-dims:] != torch.Size(self.normalized_shape):
            raise ValueError(f"this norm takes [..., {', '.join(map(str, self.normalized_shape))}], got "
                             f"{tuple(input.shape)}")
        if dims == 1:
            return layer_norm(input, self.weight, self.bias, self.eps)
        weight, bias = (None if p is None else p.flatten() for p in (self.weight, self.bias))
        return layer_norm(input.flatten(-dims), weight, bias, self.eps).view(input.shape)
