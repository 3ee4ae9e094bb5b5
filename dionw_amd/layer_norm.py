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
    watched,
)
from dionw_amd.float4 import Float4Matrix, empty

__all__ = ["LayerNorm", "float4_layer_norm", "layer_norm"]


def _rows(x: Tensor, weight: Tensor | None, bias: Tensor | None) -> Tensor:
    """x as a matrix that the kernels read, once the arguments fit each other."""
    shape = x.shape
    if not shape or shape[-1] == 0 or x.dtype not in CODES:
        raise ValueError("layer norm takes float16, bfloat16 or float32 rows of one value at least, got "
                         f"{x.dtype} of shape {tuple(shape)}")
    cols = shape[-1]
    if weight is not None:
        check_vector("norm's weight", weight, cols, x.device)
    if bias is not None:
        check_vector("norm's bias", bias, cols, x.device)
    if len(shape) != 2:
        x = x.reshape(math.prod(shape[:-1]), cols)
    return x if x.is_contiguous() else readable(x)


def _parameter(p: Tensor | None) -> tuple[int, Tensor | None, int | None]:
    """A parameter's element code, and it as the kernels read it, held by the caller until the library
    call has returned."""
    if p is None:
        return _lib.F32, None, None
    if not p.is_contiguous():
        p = p.contiguous()
    return CODES[p.dtype], p, p.data_ptr()


def _forward(x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float,
             keep: bool) -> tuple[Tensor, Tensor | None]:
    """y of a readable matrix, and its rows' means and reciprocal deviations, [2, rows]."""
    (m, n), device = x.shape, x.device
    stream = _lib.stream_handle(device)
    y = torch.empty(m, n, dtype=x.dtype, device=device)
    stats, at = None, 0
    if keep:
        stats = torch.empty(2, m, dtype=torch.float32, device=device)
        at = stats.data_ptr()
    w_code, weight, w_at = _parameter(weight)
    b_code, bias, b_at = _parameter(bias)
    call(device, "dionw_layer_norm_forward", CODES[x.dtype], x.data_ptr(), pitch(x), m, n, w_code, w_at, b_code,
         b_at, eps, y.data_ptr(), at or None, at + 4 * m if at else None, stream)
    return y, stats


@lru_cache(maxsize=256)
def _backward_scratch(rows: int, cols: int) -> int:
    return _lib.library().dionw_layer_norm_backward_scratch(rows, cols)


class _Norm(torch.autograd.Function):
    """y = u g + b, u = (x - mean) / deviation; dx = (w - mean(w) - u mean(w u)) / deviation with
    w = dy g, dg = the sum of dy u over the rows, db = that of dy."""

    @staticmethod
    def forward(ctx: Any, x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float) -> Tensor:
        # What the backward needs is worked out here: it runs on a thread of torch's own, whose caches
        # hold none of this.
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        y, stats = _forward(x, weight, bias, eps, need_x or need_w or need_b)
        m, n = x.shape
        ctx.bias_dtype = bias.dtype if need_b else torch.float32
        ctx.room = _backward_scratch(m, n) if need_w or need_b else 0
        ctx.save_for_backward(x, weight, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dy: Tensor) -> tuple[Tensor | None, ...]:
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        x, weight, stats = ctx.saved_tensors
        (m, n), device, room = x.shape, x.device, ctx.room
        ld = n
        if not dy.is_contiguous():
            dy = readable(dy)
            ld = pitch(dy)
        dx = dg = db = space = dx_at = dg_at = db_at = space_at = None
        if need_x:
            dx = x.new_empty(m, n)
            dx_at = dx.data_ptr()
        if need_w:
            dg = torch.empty_like(weight, memory_format=torch.contiguous_format)
            dg_at = dg.data_ptr()
        if need_b:
            db = torch.empty(n, dtype=ctx.bias_dtype, device=device)
            db_at = db.data_ptr()
        if room:
            space = torch.empty(room, dtype=torch.uint8, device=device)
            space_at = space.data_ptr()
        w_code, weight, w_at = _parameter(weight)
        at = stats.data_ptr()
        # The engine runs this on x's device, and on the forward's stream.
        _lib.call("dionw_layer_norm_backward", CODES[x.dtype], x.data_ptr(), pitch(x), dy.data_ptr(), ld, m, n,
                  w_code, w_at, at, at + 4 * m, dx_at, dg_at, CODES[ctx.bias_dtype], db_at, space_at, room,
                  _lib.stream_handle(device))
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
        y = _forward(flat, weight, bias, eps, False)[0]
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
    flat = _rows(x, weight, bias)
    (m, n), device = flat.shape, flat.device
    stream = _lib.stream_handle(device)
    q = empty(m, n, device)
    w_code, weight, w_at = _parameter(weight)
    b_code, bias, b_at = _parameter(bias)
    call(device, "dionw_layer_norm_float4", CODES[flat.dtype], flat.data_ptr(), pitch(flat), m, n, w_code, w_at,
         b_code, b_at, eps, q.data.data_ptr(), q.scale.data_ptr(), q.scale.shape[1], stream)
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
