"""4-bit floating-point matrices with a scale for each block of 32, and a linear layer on them.

The microscaled format: codes are e2m1 (a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6), each 32 of a
row with a power of two, which the matrix instructions multiply by on the way. Half the bytes of an
8-bit matrix, and twice its rate. As in ``dionw_amd.float8`` the optimizer keeps float32 master weights
and the model runs over them in fewer bits; the values here have two significant bits, so that
which layers take them is the model's choice.

- ``float4_linear(x, weight, bias)``: ``x @ weight.T + bias``, differentiable. x is quantized with a
  scale per row and 32 columns (for the weight's gradient, per column and 32 rows), the weight with
  one per 32 x 32 tile, whose transpose holds the same values, and the gradient like x, but rounded
  up or down by chance: to nearest, small gradients would vanish from every sum. ``weight`` may also
  be a ``Float4Matrix`` (inference with the 4-bit copy alone).
- ``Float4Linear``: ``nn.Linear`` with that product.
- ``float4_quantize`` / ``float4_quantize_both`` / ``float4_matmul``: its parts.

A block that holds a value that is not finite is NaN as a whole: codes have none of their own.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from functools import lru_cache
from typing import Any, Final

import torch
from torch import Tensor, nn

from dionw_amd import _lib
from dionw_amd._operands import (
    CODES,
    call,
    check_unrecorded,
    check_vector,
    float_bias,
    once_differentiable,
    pitch,
    readable,
    scratch as _scratch,
    tie,
    watched,
)

__all__ = ["Float4Linear", "Float4Matrix", "float4_linear", "float4_matmul", "float4_quantize",
           "float4_quantize_both"]

BLOCK: Final = 32  # columns (and rows) that share a scale
STAGE: Final = 256  # columns that a matrix's rows are padded to a multiple of
_NEAREST, _TILES, _STOCHASTIC = 0, 1, 2


def depth_of(cols: int) -> int:
    return -(-cols // STAGE) * STAGE


@dataclass(frozen=True, eq=False)
class Float4Matrix:
    """A ``[rows, cols]`` matrix in e2m1 with a power of two for each row and 32 columns.

    Attributes:
        data: uint8 ``[rows, depth / 2]``, ``depth`` being ``cols`` rounded up to 256: two codes
            a byte, the first column's in the low half; the columns past ``cols`` hold zeros.
        scale: uint8 ``[depth / 32, rows rounded up to 16 or more]``: the exponent bytes of
            the (normal) float32 scales, 1 to 254, by column block; 255 makes a block NaN.
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
        if data.dtype is not torch.uint8 or scale.dtype is not torch.uint8:
            raise TypeError("a Float4Matrix holds uint8 pairs of codes and uint8 scale exponents, got "
                            f"{data.dtype} and {scale.dtype}")
        depth = depth_of(self.cols)
        if data.dim() != 2 or scale.dim() != 2 or data.shape[1] != depth // 2:
            raise ValueError(f"the codes of {self.cols} columns are [rows, {depth // 2}], got "
                             f"{tuple(data.shape)}")
        if scale.shape[0] != depth // BLOCK or scale.shape[1] < data.shape[0]:
            raise ValueError(f"the scales of {data.shape[0]} rows are [{depth // BLOCK}, rows or more], "
                             f"got {tuple(scale.shape)}")
        if scale.shape[1] % 16:
            raise ValueError(f"the scales of a column block lie at a multiple of 16, got {scale.shape[1]}")
        if not (data.is_contiguous() and scale.is_contiguous()) or data.device != scale.device:
            raise ValueError("a Float4Matrix's tensors are contiguous and on one device")

    @property
    def shape(self) -> tuple[int, int]:
        return self.data.shape[0], self.cols

    @property
    def device(self) -> torch.device:
        return self.data.device

    def values(self) -> Tensor:
        """The float32 values.

        Raises:
            ValueError: For a matrix off the GPU, or a call that ``torch.jit.trace`` or ``make_fx``
                records.
        """
        if watched():
            check_unrecorded()
        data, scale, cols = self.data, self.scale, self.cols
        rows, device = data.shape[0], data.device
        stream = _lib.stream_handle(device)
        out = torch.empty(rows, cols, dtype=torch.float32, device=device)
        call(device, "dionw_float4_values", data.data_ptr(), scale.data_ptr(), scale.shape[1], rows, cols,
             out.data_ptr(), stream)
        return out


def empty(rows: int, cols: int, device: torch.device) -> Float4Matrix:
    """An unwritten matrix: its parts fit each other, so that nothing is checked."""
    depth = -(-cols // STAGE) * STAGE
    q = object.__new__(Float4Matrix)
    put = object.__setattr__
    put(q, "data", torch.empty(rows, depth // 2, dtype=torch.uint8, device=device))
    put(q, "scale", torch.empty(depth // BLOCK, -(-rows // 16) * 16, dtype=torch.uint8, device=device))
    put(q, "cols", cols)
    return q


def _readable(x: Tensor) -> Tensor:
    """x as the kernels read it: rows of adjacent elements that do not overlap."""
    if x.dim() != 2 or x.dtype not in CODES:
        raise ValueError("4-bit quantization takes a float16, bfloat16 or float32 matrix, got "
                         f"{x.dtype} of shape {tuple(x.shape)}")
    return readable(x)


def _seed(seed: int | Tensor, device: torch.device) -> tuple[int, int | None]:
    """The seed as the kernels take it: a number, or an address."""
    if not isinstance(seed, Tensor):
        return int(seed) & (1 << 64) - 1, None
    if seed.dtype is not torch.int64 or seed.numel() != 1 or seed.device != device:
        raise ValueError(f"a seed is a number or one int64 on {device}, got {seed.dtype} "
                         f"{tuple(seed.shape)} on {seed.device}")
    return 0, seed.data_ptr()


def _quantize(x: Tensor, tiles: bool, seed: int | Tensor | None,
              both: bool) -> tuple[Float4Matrix, Float4Matrix | None]:
    """x quantized by rows, and its transpose quantized by rows where both are asked for."""
    if watched():
        check_unrecorded()
    if tiles and seed is not None:
        raise ValueError("tiles are rounded to nearest: they take no seed")
    x, device = _readable(x), x.device
    m, n = x.shape
    stream = _lib.stream_handle(device)
    number, address = (0, None) if seed is None else _seed(seed, device)
    by_row, by_column = empty(m, n, device), None
    data, scale = by_row.data, by_row.scale
    transpose: tuple[Any, ...] = None, None, 0
    if both:
        by_column = empty(n, m, device)
        transpose = by_column.data.data_ptr(), by_column.scale.data_ptr(), by_column.scale.shape[1]
    rounding = _TILES if tiles else _NEAREST if seed is None else _STOCHASTIC
    call(device, "dionw_float4_quantize", CODES[x.dtype], x.data_ptr(), m, n, pitch(x), rounding, number,
         address, data.data_ptr(), scale.data_ptr(), scale.shape[1], *transpose, stream)
    return by_row, by_column


def float4_quantize(x: Tensor, *, tiles: bool = False, seed: int | Tensor | None = None) -> Float4Matrix:
    """A float16, bfloat16 or float32 matrix rounded to e2m1, with a scale for each row and 32
    columns, or (``tiles``) for each 32 x 32 tile.

    To nearest without a ``seed``: the scale is the smallest power of two that brings the block's
    largest magnitude to 7 at most, and what is above 6 becomes 6. With one, each value is rounded
    up or down by chance, so that it is right on average, and the scale brings the largest to 6 at
    most; the random bits are a hash of the seed (a number, or one int64 on x's device, which the
    kernel reads) and the element's place.

    Raises:
        ValueError: For another shape or type, a tensor off the GPU, both ``tiles`` and a seed, or a
            call that ``torch.jit.trace`` or ``make_fx`` records.
    """
    return _quantize(x, tiles, seed, False)[0]


def float4_quantize_both(x: Tensor, *, tiles: bool = False,
                         seed: int | Tensor | None = None) -> tuple[Float4Matrix, Float4Matrix]:
    """``float4_quantize`` of x and of its transpose, from one reading of x: what a product and its
    gradients take. With ``tiles`` both hold the same values; with a seed an element's random bits
    are the same in both.

    Raises:
        ValueError: As ``float4_quantize``.
    """
    by_row, by_column = _quantize(x, tiles, seed, True)
    return by_row, by_column


def float4_matmul(a: Float4Matrix, b: Float4Matrix, bias: Tensor | None = None, *,
                  dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """``a @ b.T + bias``, summed in float32 and rounded once to ``dtype``.

    Raises:
        ValueError: For operands or a bias that do not fit each other, another dtype than
            float16, bfloat16 or float32, rows of 16 M columns or more, tensors off the GPU, a bias
            that requires a gradient, a forward-mode dual, or a call that ``torch.jit.trace`` or
            ``make_fx`` records.
    """
    if watched():
        check_unrecorded(bias)
    a_data, a_scale, b_data, b_scale = a.data, a.scale, b.data, b.scale
    m, n, device = a_data.shape[0], b_data.shape[0], a_data.device
    if a.cols != b.cols or device != b_data.device:
        raise ValueError(f"float4_matmul takes matrices of one depth on one device, got {a.shape} on "
                         f"{device} and {b.shape} on {b.device}")
    if bias is not None:
        if bias.requires_grad and torch.is_grad_enabled():
            raise ValueError("float4_matmul gives its bias no gradient: pass it detached, or use "
                             "float4_linear on the float weight")
        bias = float_bias(bias, n, device)
    code, depth = _lib.elem_code(dtype), 2 * a_data.shape[1]
    stream = _lib.stream_handle(device)
    out = torch.empty(m, n, dtype=dtype, device=device)
    size = _workspace(m, n, depth)
    space = _scratch(size, device) if size else None
    call(device, "dionw_float4_gemm", m, n, depth, a_data.data_ptr(), a_scale.data_ptr(), a_scale.shape[1],
         b_data.data_ptr(), b_scale.data_ptr(), b_scale.shape[1], _lib.ptr(bias), code, out.data_ptr(), n,
         _lib.ptr(space), size, stream)
    return out


@lru_cache(maxsize=256)
def _workspace(m: int, n: int, depth: int) -> int:
    return _lib.library().dionw_float4_gemm_workspace(m, n, depth)


@lru_cache(maxsize=256)
def _sizes(m: int, n: int, k: int, need_x: bool, need_w: bool, need_b: bool) -> tuple[int, int, int]:
    """Bytes of what the forward saves and of both passes' scratch."""
    sizes = (ctypes.c_size_t * 3)()
    _lib.library().dionw_float4_linear_sizes(m, n, k, need_x, need_w, need_b, sizes)
    return sizes[0], sizes[1], sizes[2]


def _forward(x: Tensor, weight: Tensor, bias: Tensor | None, need_x: bool, need_w: bool,
             need_b: bool) -> tuple[Tensor, Tensor | None, int]:
    """y, what the gradients asked for need of x and W, and the bytes of the backward's scratch."""
    if not x.is_contiguous():
        x = readable(x)
    if not weight.is_contiguous():
        weight = readable(weight)
    m, k = x.shape
    n, device = weight.shape[0], x.device
    stream = _lib.stream_handle(device)
    keep, room, backward_room = _sizes(m, n, k, need_x, need_w, need_b)
    saved, scratch = _scratch(keep, device), _scratch(room, device)
    y = torch.empty(m, n, dtype=x.dtype, device=device)
    added = None if bias is None else float_bias(bias, n, device)
    call(device, "dionw_float4_linear_forward", CODES[x.dtype], x.data_ptr(), pitch(x), CODES[weight.dtype],
         weight.data_ptr(), pitch(weight), _lib.ptr(added), m, n, k, need_x, need_w, y.data_ptr(),
         _lib.ptr(saved), _lib.ptr(scratch), room, stream)
    return y, saved, backward_room


class _Linear(torch.autograd.Function):
    """y = x W^T + b; dx = dy W, dW = dy^T x, db = the sum of dy over the rows."""

    @staticmethod
    def forward(ctx: Any, x: Tensor, weight: Tensor, bias: Tensor | None,
                seed: int | Tensor | None) -> tuple[Tensor, Tensor]:
        # What the backward needs is worked out here: it runs on a thread of torch's own, whose caches
        # hold none of this.
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        y, saved, room = _forward(x, weight, bias, need_x, need_w, need_b)
        if seed is None:
            seed = int(torch.empty((), dtype=torch.int64, device="cpu").random_()) if need_x or need_w else 0
        # A seed on the device is read when the backward runs, whatever it holds then.
        ctx.seed = seed.detach() if isinstance(seed, Tensor) else seed
        ctx.number, ctx.seed_at = _seed(ctx.seed, x.device)
        ctx.sizes, ctx.room = (x.shape[0], *weight.shape), room
        ctx.dtypes = x.dtype, weight.dtype, bias.dtype if need_b else torch.float32
        ctx.device = x.device
        tied = tie(y)
        ctx.save_for_backward(saved, tied)
        ctx.set_materialize_grads(False)
        return y, tied

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dy: Tensor | None, _: None) -> tuple[Tensor | None, ...]:
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        m, n, k = ctx.sizes
        x_dtype, w_dtype, b_dtype = ctx.dtypes
        device, room = ctx.device, ctx.room
        saved, tied = ctx.saved_tensors
        if dy is None:
            dy = tied.new_zeros(m, n)
        ld = n
        if not dy.is_contiguous():
            dy = readable(dy)
            ld = pitch(dy)
        dx = dw = db = scratch = dx_at = dw_at = db_at = scratch_at = None
        if need_x:
            dx = torch.empty(m, k, dtype=x_dtype, device=device)
            dx_at = dx.data_ptr()
        if need_w:
            dw = torch.empty(n, k, dtype=w_dtype, device=device)
            dw_at = dw.data_ptr()
        if need_b:
            db = torch.empty(n, dtype=b_dtype, device=device)
            db_at = db.data_ptr()
        if room:
            scratch = torch.empty(room, dtype=torch.uint8, device=device)
            scratch_at = scratch.data_ptr()
        # The engine runs this on x's device, and on the forward's stream.
        _lib.call("dionw_float4_linear_backward", CODES[x_dtype], dy.data_ptr(), ld, CODES[w_dtype], m, n, k,
                  need_x, need_w, ctx.number, ctx.seed_at, None if saved is None else saved.data_ptr(), dx_at,
                  dw_at, CODES[b_dtype], db_at, scratch_at, room, _lib.stream_handle(device))
        return dx, dw, db, None


@lru_cache(maxsize=256)
def _kept_scratch(m: int, n: int, k: int) -> int:
    return _lib.library().dionw_float4_linear_kept_scratch(m, n, k)


def _kept_linear(x: Tensor, weight: Float4Matrix, bias: Tensor | None) -> Tensor:
    # Decoding waits for the host here: every attribute is read once.
    data, scale, k = weight.data, weight.scale, weight.cols
    device, shape, code = data.device, x.shape, CODES.get(x.dtype)
    n = data.shape[0]
    if not shape or shape[-1] != k or x.device != device or code is None:
        raise ValueError(f"float4_linear takes float x [..., {k}] on {device} for this weight, got "
                         f"{x.dtype} {tuple(shape)} on {x.device}")
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
        raise ValueError("a Float4Matrix weight is for inference: pass the float weight where "
                         "gradients are needed, or call under torch.no_grad()")
    stream = _lib.stream_handle(device)
    if len(shape) == 2:
        m, out = shape[0], (shape[0], n)
    else:
        m, out = math.prod(shape[:-1]), (*shape[:-1], n)
        x = x.reshape(m, k)
    ld = k
    if not x.is_contiguous():
        x = readable(x)
        ld = pitch(x)
    if bias is not None:
        bias = float_bias(bias, n, device)
    room = _kept_scratch(m, n, k)
    scratch = _scratch(room, device) if room else None
    y = x.new_empty(out)
    call(device, "dionw_float4_linear_kept", code, x.data_ptr(), ld, data.data_ptr(), scale.data_ptr(),
         scale.shape[1], None if bias is None else bias.data_ptr(), m, n, k, y.data_ptr(), _lib.ptr(scratch),
         room, stream)
    return y


def float4_linear(x: Tensor, weight: Tensor | Float4Matrix, bias: Tensor | None = None, *,
                  seed: int | Tensor | None = None) -> Tensor:
    """``x @ weight.T + bias`` in 4 bits, summed in float32, in x's type (float16, bfloat16 or float32).

    ``x`` is ``[..., in]``; its rows, all leading dimensions taken together, form the blocks of
    32 of the weight's gradient. Under ``torch.autocast`` x is cast to its type first, as for
    ``nn.Linear``; the weight and the bias stay as they are. ``weight`` is ``[out, in]``: a float
    tensor, quantized at every call (gradients flow to x, weight and bias, the weight's in its
    own type), or a ``Float4Matrix`` for inference. From a ``Float4Matrix`` up to 8 rows are served by
    one launch (16 of up to 8192 columns for 4096 outputs or less, of up to 2048 for 5105 to 16384 outputs, of
    up to 4096 for others), in which a row's bits do not depend on the rows beside it; more rows are
    summed in an order that their number chooses, so that a row's last bits may change with it.

    ``seed`` chooses the random bits of the gradient's rounding (see ``float4_quantize``). Without
    one a number is drawn from torch's CPU generator at every call that records gradients, as
    dropout draws its own; in a HIP graph it would be the recorded one at every replay. One int64 on
    x's device is read when the backward pass runs, also in a replay.

    Raises:
        ValueError: For shapes or types that do not fit, tensors off the GPU, an x or bias that
            requires a gradient beside a ``Float4Matrix``, forward-mode duals, calls that
            ``torch.jit.trace`` or ``make_fx`` records, or sums of 16 M products and more, a
            gradient's included.
    """
    kept = isinstance(weight, Float4Matrix)
    if watched():
        check_unrecorded(x, None if kept else weight, bias)
    if torch.is_autocast_enabled() and x.dtype in CODES:
        x = x.to(torch.get_autocast_dtype("cuda"))
    if kept:
        return _kept_linear(x, weight, bias)
    shape = x.shape
    if not shape or weight.dim() != 2 or shape[-1] != weight.shape[1]:
        raise ValueError(f"float4_linear takes x [..., in] and a weight [out, in], got "
                         f"{tuple(shape)} and {tuple(weight.shape)}")
    if x.device != weight.device:
        raise ValueError(f"x is on {x.device}, the weight on {weight.device}")
    check_vector("bias", bias, weight.shape[0], x.device)
    if isinstance(seed, Tensor):
        _seed(seed, x.device)
    for t in (x, weight):
        if t.dtype not in CODES:
            raise ValueError(f"float4_linear takes float16, bfloat16 or float32 tensors, got {t.dtype}")
    flat = x if len(shape) == 2 else x.reshape(math.prod(shape[:-1]), shape[-1])
    # Asked here: inside the function gradients are off, and what it is told of its inputs' needs
    # does not know whether they were on.
    if torch.is_grad_enabled():
        y, _ = _Linear.apply(flat, weight, bias, seed)
    else:
        y = _forward(flat, weight, bias, False, False, False)[0]
    return y if len(shape) == 2 else y.view(*shape[:-1], weight.shape[0])


class Float4Linear(nn.Linear):
    """``nn.Linear`` whose products run in 4 bits (``float4_linear``); the parameters stay as
    they are, so the layer trains with any optimizer of float weights.

    Attributes:
        seed: ``float4_linear``'s, None unless set. Recorded in a HIP graph, a layer without one (or
            with a number) rounds its gradients by the recorded bits at every replay: set it to one
            int64 on the GPU, which layers may share, and change that between replays. It is no
            buffer: neither moved nor saved with the module.
    """

    seed: int | Tensor | None = None

    def forward(self, input: Tensor) -> Tensor:
        return float4_linear(input, self.weight, self.bias, seed=self.seed)

    def quantized_weight(self) -> Float4Matrix:
        """The weight as the layer's products read it, to be kept for inference."""
        return float4_quantize(self.weight, tiles=True)
