"""8-bit floating-point matrices with a scale for each block of 128, and a linear layer on them.

The optimizer keeps float32 master weights; the layer here is a way to run the model over
them: weights, activations and gradients are quantized to e4m3 (4 exponent bits, 3 fraction
bits, largest 448) where a product reads them, and 16-bit results come from the scaled
8-bit matrix instructions, float32 ones (weight gradients) from bfloat16 ones on the same
values. Scales are powers of two, so that scaling rounds nothing.

- ``float8_linear(x, weight, bias)``: ``x @ weight.T + bias``, differentiable. x and the
  gradient are quantized with a scale per row and 128 columns (for the weight's gradient, per
  column and 128 rows), the weight with one per 128 x 128 tile, whose transpose holds the same
  values. ``weight`` may also be a ``Float8Matrix`` (inference with the 8-bit copy alone).
- ``Float8Linear``: ``nn.Linear`` with that product.
- ``float8_quantize`` / ``float8_quantize_both`` / ``float8_matmul``: its parts.

An input that is not finite becomes NaN and leaves its block's scale alone.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from functools import lru_cache
from typing import Any, Final

import torch
from torch import Tensor, nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from dionw_amd import _lib

__all__ = ["Float8Linear", "Float8Matrix", "float8_linear", "float8_matmul", "float8_quantize",
           "float8_quantize_both"]

TILE: Final = 128  # columns (and rows) that share a scale
_DTYPES: Final = (torch.float16, torch.bfloat16, torch.float32)
_CODES: Final = {dtype: _lib.elem_code(dtype) for dtype in _DTYPES}


# Cheap signs of what _check_unrecorded looks for: torch.jit.trace, and function modes, which
# make_fx runs under (as harmless ones do).
_tracing = torch._C._is_tracing
_function_modes = torch._C._len_torch_function_stack


def _check_unrecorded(*tensors: Tensor | None) -> None:
    """Kernels run on addresses, which graph recorders and forward-mode derivatives do not see: a
    recorded graph would return the outputs' memory as it was allocated, a tangent would be lost."""
    if torch.jit.is_tracing() or (_function_modes() and _recorded_by_fx()):
        raise ValueError("the 8-bit kernels cannot be recorded by torch.jit.trace or make_fx: the "
                         "graph would lose them")
    if forward_ad._current_level >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError("the 8-bit operators have no forward-mode derivative: call them on plain "
                         "tensors, or use the backward pass")


def _recorded_by_fx() -> bool:
    from torch.fx.experimental.proxy_tensor import get_proxy_mode  # takes a second to import

    return get_proxy_mode() is not None


@dataclass(frozen=True, eq=False)
class Float8Matrix:
    """A ``[rows, cols]`` matrix in e4m3 with a power of two for each row and 128 columns.

    Attributes:
        data: float8_e4m3fn codes ``[rows, depth]``, ``depth`` being ``cols`` rounded up to
            128; the columns past ``cols`` hold zeros.
        scale: uint8 ``[depth / 128, rows rounded up to 16 or more]``: the exponent bytes of
            the (normal) float32 scales, 1 to 254, by column block.
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


def _expand(q: Float8Matrix) -> Tensor:
    """The matrix as a product summed in float32 reads it: bfloat16 halves of the values."""
    rows, depth = q.data.shape
    out = torch.empty(rows, depth, dtype=torch.bfloat16, device=q.device)
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


def _pitch(x: Tensor) -> int:
    """Elements between the rows of a readable matrix."""
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _quantize(x: Tensor, tiles: bool, both: bool) -> tuple[Float8Matrix, Float8Matrix | None]:
    """x quantized by rows, and its transpose quantized by rows where both are asked for."""
    if _tracing() or _function_modes():
        _check_unrecorded()
    x = _readable(x)
    m, n = x.shape
    stream = _lib.stream_handle(x.device)
    by_row = _empty(m, n, x.device)
    by_column = _empty(n, m, x.device) if both else None
    def place(q: Float8Matrix | None) -> tuple[Any, ...]:
        return (None, 0, None, 0) if q is None else (
            q.data.data_ptr(), q.data.shape[1], q.scale.data_ptr(), q.scale.shape[1])

    _lib.call("dionw_float8_quantize", _lib.elem_code(x.dtype), x.data_ptr(), m, n, _pitch(x),
              int(tiles), *place(by_row), *place(by_column), 0, None, stream)
    return by_row, by_column


def float8_quantize(x: Tensor, *, tiles: bool = False) -> Float8Matrix:
    """A float16, bfloat16 or float32 matrix rounded to nearest in e4m3, with a scale for each
    row and 128 columns, or (``tiles``) for each 128 x 128 tile.

    Raises:
        ValueError: For another shape or type, a tensor off the GPU, or a call that
            ``torch.jit.trace`` or ``make_fx`` records.
    """
    return _quantize(x.detach(), tiles, False)[0]


def float8_quantize_both(x: Tensor, *, tiles: bool = False) -> tuple[Float8Matrix, Float8Matrix]:
    """``float8_quantize`` of x and of its transpose, from one reading of x: what a product and its
    gradients take. With ``tiles`` both hold the same values.

    Raises:
        ValueError: For another shape or type, a tensor off the GPU, or a call that
            ``torch.jit.trace`` or ``make_fx`` records.
    """
    by_row, by_column = _quantize(x.detach(), tiles, True)
    return by_row, by_column


def float8_matmul(a: Float8Matrix, b: Float8Matrix, bias: Tensor | None = None, *,
                  dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """``a @ b.T + bias`` rounded once to ``dtype``.

    A float32 result is summed in float32 on operands expanded to bfloat16, which is exact. A
    16-bit one runs on the 8-bit matrix instructions, which cut the products of each 8 columns to
    13 bits below the exponent of the largest of them before they add (1e-5 to 6e-5 of the result
    on random data, more where large products cancel).

    Raises:
        ValueError: For operands or a bias that do not fit each other, another dtype than
            float16, bfloat16 or float32, tensors off the GPU, a bias that requires a gradient,
            a forward-mode dual, or a call that ``torch.jit.trace`` or ``make_fx`` records.
    """
    if _tracing() or _function_modes() or forward_ad._current_level >= 0:
        _check_unrecorded(bias)
    m, n = a.shape[0], b.shape[0]
    if a.cols != b.cols or a.device != b.device:
        raise ValueError(f"float8_matmul takes matrices of one depth on one device, got {a.shape} on "
                         f"{a.device} and {b.shape} on {b.device}")
    if bias is not None and bias.requires_grad and torch.is_grad_enabled():
        raise ValueError("float8_matmul gives its bias no gradient: pass it detached, or use "
                         "float8_linear on the float weight")
    bias = _bias(bias, n, a.device)
    _lib.elem_code(dtype)
    depth = a.data.shape[1]
    if dtype is torch.float32:
        ea, eb = _expand(a), _expand(b)
        return _product(m, n, depth, (ea.data_ptr(), None, 0), (eb.data_ptr(), None, 0), bias, dtype,
                        a.device)
    return _product(m, n, depth, (a.data.data_ptr(), a.scale.data_ptr(), a.scale.shape[1]),
                    (b.data.data_ptr(), b.scale.data_ptr(), b.scale.shape[1]), bias, dtype, a.device)


def _check_bias(bias: Tensor | None, n: int, device: torch.device) -> None:
    if bias is not None and (bias.shape != (n,) or bias.dtype not in _DTYPES or bias.device != device):
        raise ValueError(f"the bias of {n} outputs is a float vector of that length on {device}, got "
                         f"{bias.dtype} {tuple(bias.shape)} on {bias.device}")


def _bias(bias: Tensor | None, n: int, device: torch.device) -> Tensor | None:
    """The bias as the product reads it: contiguous float32, which the caller holds until the
    library call has returned (a temporary freed before it may be another thread's by then)."""
    _check_bias(bias, n, device)
    return None if bias is None else bias.detach().to(torch.float32).contiguous()


@lru_cache(maxsize=256)
def _sizes(x_code: int, w_code: int, m: int, n: int, k: int, need_x: bool, need_w: bool,
           need_b: bool) -> tuple[int, int, int]:
    """Bytes of what the forward saves and of both passes' scratch."""
    sizes = (ctypes.c_size_t * 3)()
    _lib.library().dionw_float8_linear_sizes(x_code, w_code, m, n, k, need_x, need_w, need_b, sizes)
    return sizes[0], sizes[1], sizes[2]


def _scratch(size: int, device: torch.device) -> Tensor | None:
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def _forward(x: Tensor, weight: Tensor, bias: Tensor | None, need_x: bool, need_w: bool,
             need_b: bool) -> tuple[Tensor, Tensor | None, int]:
    """y, what the gradients asked for need of x and W, and the bytes of the backward's scratch."""
    x, weight = _readable(x), _readable(weight)
    m, k = x.shape
    n, device = weight.shape[0], x.device
    x_code, w_code = _CODES[x.dtype], _CODES[weight.dtype]
    stream = _lib.stream_handle(device)
    keep, room, backward_room = _sizes(x_code, w_code, m, n, k, need_x, need_w, need_b)
    saved, scratch = _scratch(keep, device), _scratch(room, device)
    y = torch.empty(m, n, dtype=x.dtype, device=device)
    added = _bias(bias, n, device)
    _lib.call("dionw_float8_linear_forward", x_code, x.data_ptr(), _pitch(x), w_code,
              weight.data_ptr(), _pitch(weight), _lib.ptr(added), m, n, k, need_x, need_w,
              y.data_ptr(), _lib.ptr(saved), _lib.ptr(scratch), room, stream)
    return y, saved, backward_room


class _Linear(torch.autograd.Function):
    """y = x W^T + b; dx = dy W, dW = dy^T x, db = the sum of dy over the rows."""

    @staticmethod
    def forward(ctx: Any, x: Tensor, weight: Tensor, bias: Tensor | None) -> Tensor:
        y, saved, ctx.room = _forward(x, weight, bias, *ctx.needs_input_grad)
        ctx.codes = _CODES[x.dtype], _CODES[weight.dtype]
        ctx.sizes, ctx.dtypes = (x.shape[0], *weight.shape), (x.dtype, weight.dtype)
        ctx.bias_dtype = bias.dtype if ctx.needs_input_grad[2] else None
        ctx.save_for_backward(*([] if saved is None else [saved]))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dy: Tensor) -> tuple[Tensor | None, Tensor | None, Tensor | None]:
        need_x, need_w, need_b = ctx.needs_input_grad
        m, n, k = ctx.sizes
        dy, device = _readable(dy), dy.device
        saved = ctx.saved_tensors[0] if ctx.saved_tensors else None
        scratch = _scratch(ctx.room, device)
        dx = torch.empty(m, k, dtype=ctx.dtypes[0], device=device) if need_x else None
        dw = torch.empty(n, k, dtype=ctx.dtypes[1], device=device) if need_w else None
        db = torch.empty(n, dtype=ctx.bias_dtype, device=device) if need_b else None
        _lib.call("dionw_float8_linear_backward", ctx.codes[0], dy.data_ptr(), _pitch(dy), ctx.codes[1],
                  m, n, k, need_x, need_w, _lib.ptr(saved), _lib.ptr(dx), _lib.ptr(dw),
                  _lib.elem_code(ctx.bias_dtype) if need_b else 0, _lib.ptr(db), _lib.ptr(scratch),
                  ctx.room, _lib.stream_handle(device))
        return dx, dw, db


@lru_cache(maxsize=256)
def _kept_scratch(code: int, m: int, n: int, k: int) -> int:
    return _lib.library().dionw_float8_linear_kept_scratch(code, m, n, k)


def _kept_linear(x: Tensor, weight: Float8Matrix, bias: Tensor | None) -> Tensor:
    # Decoding waits for the host here: every attribute is read once.
    data, scale, k, dtype = weight.data, weight.scale, weight.cols, x.dtype
    device, shape, code = data.device, x.shape, _CODES.get(dtype)
    n, depth = data.shape
    if not shape or shape[-1] != k or x.device != device or code is None:
        raise ValueError(f"float8_linear takes float x [..., {k}] on {device} for this weight, got "
                         f"{dtype} {tuple(shape)} on {x.device}")
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
        raise ValueError("a Float8Matrix weight is for inference: pass the float weight where "
                         "gradients are needed, or call under torch.no_grad()")
    stream = _lib.stream_handle(device)
    if len(shape) == 2:
        m, out = shape[0], (shape[0], n)
    else:
        m, out = math.prod(shape[:-1]), (*shape[:-1], n)
        x = x.reshape(m, k)
    pitch = k
    if not x.is_contiguous():
        x = _readable(x)
        pitch = _pitch(x)
    if bias is not None:
        bias = _bias(bias, n, device)
    room = _kept_scratch(code, m, n, k)
    scratch = _scratch(room, device) if room else None
    y = x.new_empty(out)
    _lib.call("dionw_float8_linear_kept", code, x.data_ptr(), pitch, data.data_ptr(), depth,
              scale.data_ptr(), scale.shape[1], None if bias is None else bias.data_ptr(), m, n, k,
              y.data_ptr(), _lib.ptr(scratch), room, stream)
    return y


def float8_linear(x: Tensor, weight: Tensor | Float8Matrix, bias: Tensor | None = None) -> Tensor:
    """``x @ weight.T + bias`` in 8 bits, in x's type (float16, bfloat16 or float32).

    ``x`` is ``[..., in]``; its rows, all leading dimensions taken together, form the blocks of
    128 of the weight's gradient. Under ``torch.autocast`` x is cast to its type first, as for
    ``nn.Linear``; the weight and the bias stay as they are. ``weight`` is ``[out, in]``: a float
    tensor, quantized at every call (gradients flow to x, weight and bias, the weight's in its
    own type), or a ``Float8Matrix`` for inference. A 16-bit x sums as ``float8_matmul`` does for
    its type; ``x.float()`` has the same codes and float32 sums.

    Raises:
        ValueError: For shapes or types that do not fit, tensors off the GPU, an x or bias that
            requires a gradient beside a ``Float8Matrix``, forward-mode duals, calls that
            ``torch.jit.trace`` or ``make_fx`` records, or sums of 8 M products (4 M for a
            float32 result) and more, a gradient's included.
    """
    kept = isinstance(weight, Float8Matrix)
    if _tracing() or _function_modes() or forward_ad._current_level >= 0:
        _check_unrecorded(x, None if kept else weight, bias)
    if torch.is_autocast_enabled() and x.dtype in _CODES:
        x = x.to(torch.get_autocast_dtype("cuda"))
    if kept:
        return _kept_linear(x, weight, bias)
    shape = x.shape
    if not shape or weight.dim() != 2 or shape[-1] != weight.shape[1]:
        raise ValueError(f"float8_linear takes x [..., in] and a weight [out, in], got "
                         f"{tuple(shape)} and {tuple(weight.shape)}")
    if x.device != weight.device:
        raise ValueError(f"x is on {x.device}, the weight on {weight.device}")
    _check_bias(bias, weight.shape[0], x.device)
    flat = x if len(shape) == 2 else x.reshape(math.prod(shape[:-1]), shape[-1])
    # Asked here: inside the function gradients are off, and what it is told of its inputs' needs
    # does not know whether they were on.
    if torch.is_grad_enabled():
        y = _Linear.apply(flat, weight, bias)
    else:
        y = _forward(flat, weight, bias, False, False, False)[0]
    return y if len(shape) == 2 else y.view(*shape[:-1], weight.shape[0])


class Float8Linear(nn.Linear):
    """``nn.Linear`` whose products run in 8 bits (``float8_linear``); the parameters stay as
    they are, so the layer trains with any optimizer of float weights."""

    def forward(self, input: Tensor) -> Tensor:
        return float8_linear(input, self.weight, self.bias)

    def quantized_weight(self) -> Float8Matrix:
        """The weight as the layer's products read it, to be kept for inference."""
        return float8_quantize(self.weight, tiles=True)
