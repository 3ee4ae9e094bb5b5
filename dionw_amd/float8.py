"""8-bit floating-point matrices with a scale for each block of 128, and a linear layer on them.

The optimizer keeps float32 master weights; the layer here is a way to run the model over
them: weights, activations and gradients are quantized to e4m3 (4 exponent bits, 3 fraction
bits, largest 448) where a product reads them, and 16-bit results come from the scaled
8-bit matrix instructions, float32 ones (weight gradients) from bfloat16 ones on the same values. Scales are powers of two, so that scaling rounds nothing.

- ``float8_linear(x, weight, bias)``: ``x @ weight.T + bias``, differentiable. x and the
  gradient are quantized with a scale per row and 128 columns (for the weight's gradient, per
  column and 128 rows), the weight with one per 128 x 128 tile, whose transpose holds the same
  values. ``weight`` may also be a ``Float8Matrix`` (inference with the 8-bit copy alone).
- ``Float8Linear``: ``nn.Linear`` with that product.
- ``float8_quantize`` / ``float8_matmul``: its parts.

An input that is not finite becomes NaN and leaves its block's scale alone.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Any, Final

import torch
from torch import Tensor, nn
from torch.autograd.function import once_differentiable

from dionw_amd import _lib

__all__ = ["Float8Linear", "Float8Matrix", "float8_linear", "float8_matmul", "float8_quantize"]

TILE: Final = 128  # columns (and rows) that share a scale
_DTYPES: Final = (torch.float16, torch.bfloat16, torch.float32)


@dataclass(frozen=True, eq=False)
class Float8Matrix:
    """A ``[rows, cols]`` matrix in e4m3 with a power of two for each row and 128 columns.

    Attributes:
        data: float8_e4m3fn codes ``[rows, depth]``, ``depth`` being ``cols`` rounded up to
            128; the columns past ``cols`` hold zeros.
        scale: uint8 ``[depth / 128, rows rounded up to 16 or more]``: the exponent bytes of
            the float32 scales, by column block.
        cols: The number of columns.

    Raises:
        TypeError: For other element types.
        ValueError: For shapes or layouts that do not fit each other.
    """

    data: Tensor
    scale: Tensor
    cols: int

    def __post_init__(self) -> None:
        data, scale = self.data, self.scale
        if data.dtype is not torch.float8_e4m3fn or scale.dtype is not torch.uint8:
            raise TypeError("a Float8Matrix holds float8_e4m3fn codes and uint8 scale exponents, got "
                            f"{data.dtype} and {scale.dtype}")
        depth = -(-self.cols // TILE) * TILE
        if data.dim() != 2 or scale.dim() != 2 or data.shape[1] != depth:
            raise ValueError(f"the codes of {self.cols} columns are [rows, {depth}], got "
                             f"{tuple(data.shape)}")
        if scale.shape[0] != depth // TILE or scale.shape[1] < data.shape[0]:
            raise ValueError(f"the scales of {data.shape[0]} rows are [{depth // TILE}, rows or more], "
                             f"got {tuple(scale.shape)}")
        if scale.shape[1] % 16:
            raise ValueError(f"the scales of a column block lie at a multiple of 16, got {scale.shape[1]}")
        if not (data.is_contiguous() and scale.is_contiguous()) or data.device != scale.device:
            raise ValueError("a Float8Matrix's tensors are contiguous and on one device")

    @property
    def shape(self) -> tuple[int, int]:
        return self.data.shape[0], self.cols

    @property
    def device(self) -> torch.device:
        return self.data.device

    def values(self) -> Tensor:
        """The float32 values."""
        rows = self.data.shape[0]
        power = (self.scale[:, :rows].t().to(torch.int32) << 23).view(torch.float32)
        depth = self.data.shape[1]
        blocks = self.data.to(torch.float32).view(rows, depth // TILE, TILE)
        return (blocks * power[..., None]).view(rows, depth)[:, :self.cols]


def _empty(rows: int, cols: int, device: torch.device) -> Float8Matrix:
    depth = -(-cols // TILE) * TILE
    return Float8Matrix(
        torch.empty(rows, depth, dtype=torch.float8_e4m3fn, device=device),
        torch.empty(depth // TILE, -(-rows // 16) * 16, dtype=torch.uint8, device=device), cols)


def _expanded(rows: int, cols: int, device: torch.device) -> Tensor:
    return torch.empty(rows, -(-cols // TILE) * TILE, dtype=torch.bfloat16, device=device)


def _expand(q: Float8Matrix) -> Tensor:
    """The matrix as a product summed in float32 reads it: bfloat16 halves of the values."""
    rows, depth = q.data.shape
    out = _expanded(rows, depth, q.device)
    _lib.call("dionw_float8_expand", q.data.data_ptr(), depth, q.scale.data_ptr(), q.scale.shape[1],
              rows, depth, out.data_ptr(), depth, _lib.stream_handle(q.device))
    return out


def _product(m: int, n: int, depth: int, a: tuple[int, int | None, int], b: tuple[int, int | None, int],
             bias: Tensor | None, dtype: torch.dtype, device: torch.device) -> Tensor:
    """``a b.T + bias`` from the operands' addresses: (data, scale, scale pitch), the scale None
    for expanded operands."""
    expanded, stream = int(a[1] is None), _lib.stream_handle(device)
    out = torch.empty(m, n, dtype=dtype, device=device)
    size = _lib.library().dionw_float8_gemm_workspace(expanded, m, n, depth)
    space = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    _lib.call("dionw_float8_gemm", expanded, m, n, depth, a[0], depth, a[1], a[2], b[0], depth, b[1],
              b[2], _lib.ptr(bias), _lib.elem_code(dtype), out.data_ptr(), n, _lib.ptr(space), size,
              stream)
    return out


def _readable(x: Tensor) -> Tensor:
    """x as the kernels read it: rows of adjacent elements that do not overlap."""
    if x.dim() != 2 or x.dtype not in _DTYPES:
        raise ValueError("8-bit quantization takes a float16, bfloat16 or float32 matrix, got "
                         f"{x.dtype} of shape {tuple(x.shape)}")
    adjacent = x.shape[1] <= 1 or x.stride(1) == 1
    return x if adjacent and (x.shape[0] <= 1 or x.stride(0) >= x.shape[1]) else x.contiguous()


def _quantize(x: Tensor, tiles: bool, rows: bool, columns: bool, sums: torch.dtype | None = None,
              *, expand: bool = False,
              ) -> tuple[Float8Matrix | None, Float8Matrix | Tensor | None, Tensor | None]:
    """x quantized by rows, its transpose quantized by rows (``expand``: its codes expanded, as a
    product summed in float32 reads them), and its column sums, as asked."""
    x = _readable(x)
    m, n = x.shape
    stream = _lib.stream_handle(x.device)
    by_row = _empty(m, n, x.device) if rows else None
    by_column: Float8Matrix | Tensor | None = None
    if columns:
        by_column = _expanded(n, m, x.device) if expand else _empty(n, m, x.device)
    parts = torch.empty(-(-m // TILE), n, device=x.device) if sums else None
    ld = x.stride(0) if m > 1 else n

    def place(q: Float8Matrix | Tensor | None) -> tuple[Any, ...]:
        if isinstance(q, Tensor):
            return q.data_ptr(), q.shape[1], None, 0
        return (None, 0, None, 0) if q is None else (
            q.data.data_ptr(), q.data.shape[1], q.scale.data_ptr(), q.scale.shape[1])

    _lib.call("dionw_float8_quantize", _lib.elem_code(x.dtype), x.data_ptr(), m, n, max(ld, n),
              int(tiles), *place(by_row), *place(by_column), int(expand), _lib.ptr(parts), stream)
    total = None
    if sums:
        total = torch.empty(n, dtype=sums, device=x.device)
        _lib.call("dionw_sum_parts", parts.data_ptr(), parts.shape[0], n, _lib.elem_code(sums),
                  total.data_ptr(), stream)
    return by_row, by_column, total


def float8_quantize(x: Tensor, *, tiles: bool = False) -> Float8Matrix:
    """A float16, bfloat16 or float32 matrix rounded to nearest in e4m3, with a scale for each
    row and 128 columns, or (``tiles``) for each 128 x 128 tile.

    Raises:
        ValueError: For another shape or type, or a tensor off the GPU.
    """
    return _quantize(x.detach(), tiles, True, False)[0]


def float8_matmul(a: Float8Matrix, b: Float8Matrix, bias: Tensor | None = None, *,
                  dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """``a @ b.T + bias`` rounded once to ``dtype``.

    A float32 result is summed in float32 on operands expanded to bfloat16, which is exact. A
    16-bit one runs on the 8-bit matrix instructions, which cut the products of each 8 columns to
    13 bits below the exponent of the largest of them before they add (1e-5 to 6e-5 of the result).

    Raises:
        ValueError: For operands or a bias that do not fit each other, another dtype than
            float16, bfloat16 or float32, or tensors off the GPU.
    """
    m, n = a.shape[0], b.shape[0]
    if a.cols != b.cols or a.device != b.device:
        raise ValueError(f"float8_matmul takes matrices of one depth on one device, got {a.shape} on "
                         f"{a.device} and {b.shape} on {b.device}")
    bias = _bias(bias, n, a.device)
    _lib.elem_code(dtype)
    depth = a.data.shape[1]
    if dtype is torch.float32:
        ea, eb = _expand(a), _expand(b)
        return _product(m, n, depth, (ea.data_ptr(), None, 0), (eb.data_ptr(), None, 0), bias, dtype,
                        a.device)
    return _product(m, n, depth, (a.data.data_ptr(), a.scale.data_ptr(), a.scale.shape[1]),
                    (b.data.data_ptr(), b.scale.data_ptr(), b.scale.shape[1]), bias, dtype, a.device)


def _bias(bias: Tensor | None, n: int, device: torch.device) -> Tensor | None:
    """The bias as the product reads it: contiguous float32."""
    if bias is None:
        return None
    if bias.shape != (n,) or bias.dtype not in _DTYPES or bias.device != device:
        raise ValueError(f"the bias of {n} outputs is a float vector of that length on {device}, got "
                         f"{bias.dtype} {tuple(bias.shape)} on {bias.device}")
    return bias.detach().to(torch.float32).contiguous()


class _Linear(torch.autograd.Function):
    """y = x W^T + b; dx = dy W, dW = dy^T x, db = the sum of dy over the rows."""

    @staticmethod
    def forward(ctx: Any, x: Tensor, weight: Tensor, bias: Tensor | None) -> Tensor:
        need_x, need_w = ctx.needs_input_grad[:2]
        xq, xt, _ = _quantize(x, False, True, need_w)
        wq, wt, _ = _quantize(weight, True, True, need_x)
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.dtypes, ctx.sizes = (x.dtype, weight.dtype), (x.shape[0], *weight.shape)
        ctx.save_for_backward(*(t for q in (xt, wt) if q is not None for t in (q.data, q.scale)))
        return float8_matmul(xq, wq, bias, dtype=x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dy: Tensor) -> tuple[Tensor | None, Tensor | None, Tensor | None]:
        need_x, need_w, need_b = ctx.needs_input_grad
        m, n, k = ctx.sizes
        saved = list(ctx.saved_tensors)
        xt = Float8Matrix(*saved[:2], m) if need_w else None
        wt = Float8Matrix(*saved[-2:], n) if need_x else None
        exact = ctx.dtypes[1] is torch.float32
        rows, columns, db = _quantize(dy, False, need_x, need_w, ctx.bias_dtype if need_b else None,
                                      expand=exact)
        dx = float8_matmul(rows, wt, dtype=ctx.dtypes[0]) if need_x else None
        dw = None
        if need_w and exact:
            ex = _expand(xt)
            dw = _product(n, k, ex.shape[1], (columns.data_ptr(), None, 0), (ex.data_ptr(), None, 0),
                          None, torch.float32, dy.device)
        elif need_w:
            dw = float8_matmul(columns, xt, dtype=ctx.dtypes[1])
        return dx, dw, db


def float8_linear(x: Tensor, weight: Tensor | Float8Matrix, bias: Tensor | None = None) -> Tensor:
    """``x @ weight.T + bias`` in 8 bits, in x's type (float16, bfloat16 or float32).

    ``x`` is ``[..., in]``; its rows, all leading dimensions taken together, form the blocks of
    128 of the weight's gradient. ``weight`` is ``[out, in]``: a float tensor, quantized at
    every call (gradients flow to x, weight and bias, the weight's in its own type), or a
    ``Float8Matrix`` for inference.

    Raises:
        ValueError: For shapes or types that do not fit, tensors off the GPU, or an x that
            requires a gradient beside a ``Float8Matrix``.
    """
    if x.dim() == 0 or x.shape[-1] != weight.shape[-1] or len(weight.shape) != 2:
        raise ValueError(f"float8_linear takes x [..., in] and a weight [out, in], got "
                         f"{tuple(x.shape)} and {tuple(weight.shape)}")
    if x.device != weight.device:
        raise ValueError(f"x is on {x.device}, the weight on {weight.device}")
    flat = x.reshape(math.prod(x.shape[:-1]), x.shape[-1])
    if isinstance(weight, Float8Matrix):
        if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
            raise ValueError("a Float8Matrix weight is for inference: pass the float weight where "
                             "gradients are needed, or call under torch.no_grad()")
        out = float8_matmul(float8_quantize(flat), weight, bias, dtype=x.dtype)
    else:
        _bias(bias, weight.shape[0], x.device)
        out = _Linear.apply(flat, weight, bias)
    return out.view(*x.shape[:-1], weight.shape[0])


class Float8Linear(nn.Linear):
    """``nn.Linear`` whose products run in 8 bits (``float8_linear``); the parameters stay as
    they are, so the layer trains with any optimizer of float weights."""

    def forward(self, input: Tensor) -> Tensor:
        return float8_linear(input, self.weight, self.bias)

    def quantized_weight(self) -> Float8Matrix:
        """The weight as the layer's products read it, to be kept for inference."""
        return float8_quantize(self.weight, tiles=True)
