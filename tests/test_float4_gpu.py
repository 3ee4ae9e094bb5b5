"""4-bit matrices, their products and the linear layer against float64 (GPU).

Quantization is exact: every code and scale must be the definition's, the stochastic one's too. A
product of two e2m1 values is exact in float32; the sums' error is bounded, whatever their order and
even if the adders truncate, by ``(depth + 1) x 2^-23 x sum |a| |b|``, and the result is rounded once
more to the output's type.
"""

from __future__ import annotations

import ctypes

import pytest
import torch

from dionw_amd import (
    Float4Linear,
    Float4Matrix,
    float4_linear,
    float4_matmul,
    float4_quantize,
    float4_quantize_both,
)
from tests import float4_oracle as oracle

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
SMALLEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}  # half a subnormal
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
BLOCK = oracle.BLOCK


def _random(m, n, seed, dtype=torch.float32, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(m, n, generator=gen) * torch.exp(spread * torch.randn(m, 1, generator=gen))
    x = x * torch.exp(spread * torch.randn(1, n, generator=gen))
    return x.to(dtype).cuda()


def _check(got, a, b, bias=None):
    """``got`` against ``a @ b.T + bias`` of float64 values."""
    want, size = a @ b.T, a.abs() @ b.abs().T
    if bias is not None:
        bias = bias.detach().cpu().double()
        want, size = want + bias, size + bias.abs()
    bound = (a.shape[1] + 1) * 2.0 ** -23 * size
    bound = bound + UNIT[got.dtype] * (want.abs() + bound) + SMALLEST[got.dtype]
    error = (got.detach().cpu().double() - want).abs()
    assert got.shape == want.shape and bool((error <= bound).all()), float((error - bound).max())


def _same(q: Float4Matrix, source, rows=1, bits=None):
    values, byte = oracle.quantize(source, rows, bits)
    assert q.shape == tuple(source.shape)
    assert torch.equal(q.scale[:byte.shape[0], :source.shape[0]].cpu().int(), byte.int())
    assert torch.equal(q.values().cpu().double(), values)
    codes = torch.stack([q.data & 15, q.data >> 4], 2).view(q.data.shape[0], -1)
    assert not codes[:, q.cols:].any()


SHAPES = [(1, 1), (1, 256), (256, 1), (127, 129), (128, 128), (200, 300), (3, 1000), (257, 512), (640, 77),
          (31, 33), (500, 2100)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("tiles", [False, True])
def test_quantization_is_the_definitions(shape, dtype, tiles) -> None:
    x = _random(*shape, 1, dtype)
    rows, columns = float4_quantize_both(x, tiles=tiles)
    side = BLOCK if tiles else 1
    _same(rows, x, side)
    _same(columns, x.t(), side)
    alone = float4_quantize(x, tiles=tiles)
    assert torch.equal(alone.data, rows.data)
    assert torch.equal(alone.scale[:, :shape[0]], rows.scale[:, :shape[0]])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("seed", [0, 123456789012345, -7])
def test_stochastic_quantization_is_the_definitions(shape, dtype, seed) -> None:
    x = _random(*shape, 2, dtype)
    bits = oracle.noise(seed, *shape)
    rows, columns = float4_quantize_both(x, seed=seed)
    _same(rows, x, bits=bits)
    _same(columns, x.t(), bits=bits.t())
    at = torch.tensor([seed], device="cuda")
    for other in (float4_quantize(x, seed=seed), float4_quantize(x, seed=at)):
        assert torch.equal(other.data, rows.data)


def test_a_large_matrix_in_rows_alone() -> None:
    """Enough rows for the workgroups of 32."""
    x = _random(5003, 4100, 3, torch.bfloat16)
    q = float4_quantize(x)
    for part in (slice(0, 100), slice(2500, 2600), slice(4903, 5003)):
        values, byte = oracle.quantize(x[part])
        assert torch.equal(q.values()[part].cpu().double(), values)
        assert torch.equal(q.scale[:byte.shape[0], part].cpu().int(), byte.int())


def _edges():
    x = torch.zeros(32, 256)
    x[1, 0] = 7.0
    x[2, 0] = torch.nextafter(torch.tensor(7.0), torch.tensor(1e9))
    x[3, 0], x[3, 1] = 2.0 ** -149, -(2.0 ** -140)
    x[4, 0], x[4, 1] = 3.4e38, -3.3e38
    x[5, 0], x[5, 1], x[5, 40] = float("inf"), 2.0, -1.0
    x[6, 100], x[6, 101], x[6, 3] = float("nan"), -float("inf"), 3.0
    x[7, :32] = torch.arange(32) * 0.25  # every tie
    x[8] = torch.arange(256) * 2.0 ** -6 + 2.0 ** -3
    x[9] = 2.0 ** -126
    x[10, 0] = -0.0
    x[11] = float("nan")
    x[12, 0], x[12, 1] = 6.0, 5.999
    x[13, 0] = torch.nextafter(torch.tensor(6.0), torch.tensor(1e9))
    x[14, 0], x[14, 1:32] = 6.0, 2.0 ** -24 * torch.arange(1, 32)
    x[15, 255] = -3.4e38
    return x


def test_quantization_of_values_at_the_edges() -> None:
    """Maxima at a power's carry, zeros, the smallest and largest floats, values that are not
    finite, ties."""
    x = _edges().cuda()
    got = float4_quantize(x)
    values, byte = oracle.quantize(x)
    assert torch.equal(got.scale[:, :32].cpu().int(), byte.int())
    now = got.values().cpu().double()
    assert torch.equal(now.isnan(), values.isnan())
    values = values.float().double()  # as float32 holds them
    assert torch.equal(now.nan_to_num(), values.nan_to_num())
    # A block's NaN reaches its row's outputs alone.
    eye = torch.eye(256, device="cuda")
    out = float4_matmul(got, float4_quantize(eye), dtype=torch.float32)
    assert torch.equal(out.isnan().any(1).cpu(), values.isnan().any(1))
    finite = ~values.isnan().any(1)
    assert torch.equal(out.cpu().double()[finite], values[finite])


def test_stochastic_quantization_of_values_at_the_edges() -> None:
    x = _edges().cuda()
    bits = oracle.noise(3, *x.shape)
    for got, source, noise in zip(float4_quantize_both(x, seed=3), (x, x.t()), (bits, bits.t())):
        values, byte = oracle.quantize(source, 1, noise)
        assert torch.equal(got.scale[:byte.shape[0], :source.shape[0]].cpu().int(), byte.int())
        now = got.values().cpu().double()
        assert torch.equal(now.isnan(), values.isnan())
        assert torch.equal(now.nan_to_num(), values.float().double().nan_to_num())


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_inputs(dtype) -> None:
    base = _random(300, 700, 2, dtype)
    for x in (base[:, :333], base[:, 1:334], base[::2, 4:400], base.t(), base[5:6], base[:, 3:4],
              base[0].expand(50, 700), base[:, :1].expand(300, 200)):
        _same(float4_quantize(x), x)
        bits = oracle.noise(1, *x.shape)
        rows, columns = float4_quantize_both(x, seed=1)
        _same(rows, x, bits=bits)
        _same(columns, x.t(), bits=bits.t())


def test_rows_behind_the_last_are_left_alone() -> None:
    """The scales' padding apart, nothing is written past a matrix."""
    from dionw_amd import _lib

    x = _random(100, 300, 4)
    data = torch.full((110, 256), 77, dtype=torch.uint8, device="cuda")
    scale = torch.full((17, 112), 77, dtype=torch.uint8, device="cuda")
    data_t = torch.full((310, 128), 77, dtype=torch.uint8, device="cuda")
    scale_t = torch.full((9, 304), 77, dtype=torch.uint8, device="cuda")
    for rounding in range(3):
        _lib.call("dionw_float4_quantize", 2, x.data_ptr(), 100, 300, 300, rounding, 5, None, data.data_ptr(),
                  scale.data_ptr(), 112, data_t.data_ptr(), scale_t.data_ptr(), 304,
                  _lib.stream_handle(x.device))
        assert (data[100:] == 77).all() and (data_t[300:] == 77).all()
        assert (scale[16] == 77).all() and (scale_t[8] == 77).all()


# (tokens, depth, outputs): one, ragged, around every tile size, deep, wide, many tokens.
PRODUCTS = [(1, 1, 1), (1, 4096, 64), (2, 128, 16), (5, 300, 1000), (16, 256, 17), (17, 128, 128), (33, 1024, 65),
            (64, 384, 64), (65, 512, 129), (100, 14336, 256), (127, 200, 255), (128, 128, 128),
            (129, 1152, 257), (255, 640, 511), (256, 256, 256), (257, 1000, 513), (300, 2048, 300),
            (512, 896, 768), (1000, 128, 1000), (1025, 2304, 1031), (2048, 512, 2048), (8, 32768, 40),
            (4096, 768, 4100), (64, 4096, 4096)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", PRODUCTS, ids=str)
def test_products(size, dtype) -> None:
    m, k, n = size
    a, b = _random(m, k, 3, spread=0.5), _random(n, k, 4, spread=0.5) * k ** -0.5
    bias = torch.randn(n, device="cuda") if m % 2 else None
    qa, qb = float4_quantize(a), float4_quantize(b, tiles=n % 2 == 0)
    got = float4_matmul(qa, qb, bias, dtype=dtype)
    _check(got, qa.values().cpu().double(), qb.values().cpu().double(), bias)


@pytest.mark.parametrize("extents", [(64, 2048, 64), (1024, 2048, 1024), (1536, 1280, 768), (4096, 1024, 4096),
                                     (100, 16384, 200), (2304, 8192, 768)], ids=str)
def test_small_whole_numbers_are_exact_on_every_tile(extents) -> None:
    """Values of the format with powers of two by row and block: layouts and scales must give the
    very float64 results."""
    m, k, n = extents
    gen = torch.Generator(device="cuda").manual_seed(5)
    values = torch.tensor([0.0, 1, 2, 3, 4, 6, -1, -2, -3, -4, -6], device="cuda")

    def whole(rows, cols):
        v = values[torch.randint(11, (rows, cols), generator=gen, device="cuda")]
        v.view(rows, -1, BLOCK)[..., 0] = 6  # every block's scale is its power
        p = torch.randint(-1, 2, (rows, cols // BLOCK, 1), generator=gen, device="cuda")
        return (v.view(rows, -1, BLOCK) * 2.0 ** p).view(rows, cols)

    a, b = whole(m, k), whole(n, k)
    got = float4_matmul(float4_quantize(a), float4_quantize(b), dtype=torch.float32)
    # Multiples of 1/4 up to k 144: exact in float32 up to 2^22.
    assert torch.equal(got.double(), a.double() @ b.double().t())


def test_small_whole_numbers_are_exact_in_the_layer() -> None:
    """Whole numbers that the format holds beside each other give both gradients exactly, rounded
    stochastically too: a value of the format is kept."""
    gen = torch.Generator().manual_seed(5)
    for m, k, n in ((1, 300, 200), (130, 200, 99), (513, 640, 770), (300, 1024, 256)):
        def whole(*shape):
            return torch.randint(-3, 4, shape, generator=gen).float()

        x, w, dy = whole(m, k), whole(n, k), whole(m, n)
        xp, wp = (torch.nn.Parameter(t.cuda()) for t in (x, w))
        y = float4_linear(xp, wp)
        assert torch.equal(y.cpu().double(), x.double() @ w.double().t())
        dx, dw = torch.autograd.grad(y, (xp, wp), dy.cuda())
        assert torch.equal(dx.cpu().double(), dy.double() @ w.double())
        assert torch.equal(dw.cpu().double(), dy.double().t() @ x.double())


def test_gradients_are_the_differences() -> None:
    """On whole numbers the layer is exactly bilinear, so that the change of a loss along any
    whole step is the gradient's product with it (and half the second-order term, taken out by
    a central difference)."""
    gen = torch.Generator().manual_seed(6)
    m, k, n = 70, 260, 140
    x, w = (torch.randint(-2, 3, s, generator=gen).float().cuda() for s in ((m, k), (n, k)))
    b, dy = torch.randint(-3, 4, (n,), generator=gen).float().cuda(), torch.randint(-3, 4, (m, n), generator=gen).float().cuda()
    steps = [torch.randint(-1, 2, s.shape, generator=gen).float().cuda() for s in (x, w, b)]
    args = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(float4_linear(*args), args, dy)

    def loss(sign):
        return (float4_linear(*[t + sign * s for t, s in zip((x, w, b), steps)]).double() * dy.double()).sum()

    slope = sum((g.double() * s.double()).sum() for g, s in zip(grads, steps))
    assert float(loss(1) - loss(-1)) == 2 * float(slope)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [(1, 64, 64), (130, 200, 99), (257, 512, 385), (1000, 300, 1111)], ids=str)
def test_the_layer_trains(size, dtype) -> None:
    m, k, n = size
    x = (_random(m, k, 7, spread=0.5)).to(dtype).requires_grad_()
    w = torch.nn.Parameter(_random(n, k, 8, spread=0.3) * k ** -0.5)
    b = torch.nn.Parameter(torch.randn(n, device="cuda"))
    dy = (_random(m, n, 9, spread=0.5) * 1e-2).to(dtype)
    y = float4_linear(x, w, b, seed=77)
    y.backward(dy)
    assert y.dtype is dtype and x.grad.dtype is dtype and w.grad.dtype is torch.float32
    bits = oracle.noise(77, m, n)
    xq, wq = oracle.quantize(x)[0], oracle.quantize(w, BLOCK)[0]
    _check(y, xq, wq, b)
    _check(x.grad, oracle.quantize(dy, 1, bits)[0], wq.T.contiguous())
    _check(w.grad, oracle.quantize(dy.t(), 1, bits.t())[0], oracle.quantize(x.t())[0])
    exact = dy.double().sum(0)
    assert bool(((b.grad.double() - exact).abs() <= (m + 1) * 2.0 ** -24 * dy.double().abs().sum(0)).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 70, 128, 129, 257, 300, 520])
def test_nothing_is_written_past_the_buffers(rows, dtype) -> None:
    """Of both passes, whatever gradients are asked for: each buffer of exactly its size, and what lies
    behind it stays."""
    from itertools import product as every

    from dionw_amd import _lib

    n, k, code, guard = 200, 300, _lib.elem_code(dtype), 1 << 16
    x, dy = _random(rows, k, 1, dtype), _random(rows, n, 2, dtype)
    w, b = _random(n, k, 3), torch.randn(n, device="cuda")
    stream = _lib.stream_handle(x.device)

    def room(size):
        return torch.full((size + guard,), 77, dtype=torch.uint8, device="cuda")

    for need_x, need_w, need_b in every((0, 1), repeat=3):
        sizes = (ctypes.c_size_t * 3)()
        _lib.library().dionw_float4_linear_sizes(rows, n, k, need_x, need_w, need_b, sizes)
        saved, forward, backward = map(room, sizes)
        y, dx, dw, db = (room(size) for size in (x.itemsize * rows * n, x.itemsize * rows * k, 4 * n * k, 4 * n))
        _lib.call("dionw_float4_linear_forward", code, x.data_ptr(), k, 2, w.data_ptr(), k, b.data_ptr(), rows, n, k,
                  need_x, need_w, y.data_ptr(), saved.data_ptr(), forward.data_ptr(), sizes[1], stream)
        _lib.call("dionw_float4_linear_backward", code, dy.data_ptr(), n, 2, rows, n, k, need_x, need_w, 5, None,
                  saved.data_ptr(), dx.data_ptr() if need_x else None, dw.data_ptr() if need_w else None, 2,
                  db.data_ptr() if need_b else None, backward.data_ptr(), sizes[2], stream)
        for buffer in (saved, forward, backward, y, dx, dw, db):
            assert bool((buffer[-guard:] == 77).all())


def test_gradients_are_right_on_average() -> None:
    """Over many seeds the gradient approaches that of unrounded dy: each of S sums of n terms has a
    deviation of half a step of each term at most. A block's step is at most a third of its
    largest value; six deviations."""
    m, k, n, seeds = 64, 32, 96, 256
    x, w = _random(m, k, 1, spread=0.2), _random(n, k, 2, spread=0.2)
    dy = _random(m, n, 3, spread=0.2)
    xp = x.clone().requires_grad_()
    total = torch.zeros(m, k, dtype=torch.float64, device="cuda")
    for seed in range(seeds):
        total += torch.autograd.grad(float4_linear(xp, w, seed=seed), xp, dy)[0].double()
    wq = oracle.quantize(w, BLOCK)[0].cuda()
    most = dy.double().abs().view(m, -1, BLOCK).amax(2).repeat_interleave(BLOCK, 1)
    deviation = ((most / 3 / 2) ** 2 @ wq ** 2).sqrt() / seeds ** 0.5
    assert bool(((total / seeds - dy.double() @ wq).abs() <= 6 * deviation).all())


@pytest.mark.parametrize("kinds", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.bfloat16),
                                   (torch.float32, torch.float16)], ids=str)
def test_weights_and_biases_of_16_bits(kinds) -> None:
    """Gradients come in the weight's and the bias's own types."""
    dtype, held = kinds
    m, k, n = 300, 260, 130
    x = _random(m, k, 7, spread=0.5).to(dtype).requires_grad_()
    w = (_random(n, k, 8, spread=0.3) * k ** -0.5).to(held).requires_grad_()
    b = torch.randn(n, device="cuda").to(held).requires_grad_()
    dy = (_random(m, n, 9, spread=0.5) * 1e-2).to(dtype)
    y = float4_linear(x, w, b, seed=5)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert (dx.dtype, dw.dtype, db.dtype) == (dtype, held, held)
    bits = oracle.noise(5, m, n)
    xq, wq = oracle.quantize(x)[0], oracle.quantize(w, BLOCK)[0]
    _check(y, xq, wq, b)
    _check(dx, oracle.quantize(dy, 1, bits)[0], wq.T.contiguous())
    _check(dw, oracle.quantize(dy.t(), 1, bits.t())[0], oracle.quantize(x.t())[0])
    exact = dy.double().sum(0)
    bound = (m + 1) * 2.0 ** -24 * dy.double().abs().sum(0)
    assert bool(((db.double() - exact).abs() <= bound + UNIT[held] * (exact.abs() + bound)).all())


def test_only_the_gradients_asked_for() -> None:
    x, w, b = _random(40, 130, 1), _random(50, 130, 2), torch.randn(50, device="cuda")
    dy = _random(40, 50, 3)
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(float4_linear(*full, seed=1), full, dy)
    for mask in range(1, 8):
        args = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b))]
        asked = [t for t in args if t.requires_grad]
        got = torch.autograd.grad(float4_linear(*args, seed=1), asked, dy)
        for g, t in zip(got, asked):
            assert torch.equal(g, want[[t is a for a in args].index(True)])


def test_leading_dimensions_broadcast_gradients_and_shared_weights() -> None:
    x = _random(60, 130, 1).view(3, 4, 5, 130).requires_grad_()
    w = torch.nn.Parameter(_random(50, 130, 2))
    y = float4_linear(x, w, seed=9)
    assert y.shape == (3, 4, 5, 50)
    y.sum().backward()  # a gradient of stride 0
    flat = x.detach().reshape(60, 130).requires_grad_()
    v = torch.nn.Parameter(w.detach().clone())
    float4_linear(flat, v, seed=9).backward(torch.ones(60, 50, device="cuda"))
    assert torch.equal(x.grad.view(60, 130), flat.grad) and torch.equal(w.grad, v.grad)
    # A weight used twice sums its gradients.
    u = torch.nn.Parameter(w.detach().clone())
    twice = [float4_linear(flat.detach(), u, seed=9) for _ in range(2)]
    (twice[0] + twice[1]).backward(torch.ones(60, 50, device="cuda"))
    assert torch.equal(u.grad, 2 * v.grad)


def test_empty_extents() -> None:
    w = torch.nn.Parameter(_random(50, 130, 2))
    b = torch.nn.Parameter(torch.randn(50, device="cuda"))
    x = torch.zeros(0, 130, device="cuda", requires_grad=True)
    y = float4_linear(x, w, b)
    assert y.shape == (0, 50)
    y.sum().backward()
    assert x.grad.shape == (0, 130) and not w.grad.any() and not b.grad.any()
    empty = float4_linear(torch.zeros(4, 0, device="cuda"), torch.zeros(50, 0, device="cuda"), b.detach())
    assert torch.equal(empty, b.detach().expand(4, 50))
    assert float4_linear(torch.zeros(4, 130, device="cuda"), torch.zeros(0, 130, device="cuda")).shape == (4, 0)
    kept = float4_quantize(torch.zeros(50, 0, device="cuda"))
    for rows in (1, 40):
        assert torch.equal(float4_linear(torch.zeros(rows, 0, device="cuda"), kept, b.detach()),
                           b.detach().expand(rows, 50))
    assert kept.values().shape == (50, 0) and float4_quantize(torch.zeros(0, 9, device="cuda")).values().shape == (0, 9)


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_rows_of_an_input_without_a_gradient(dtype) -> None:
    """Whichever of weight and bias are trained: their gradients are zeros, in their own types."""
    x = torch.zeros(0, 130, dtype=dtype, device="cuda")
    for mask in range(1, 4):
        w, b = _random(50, 130, 2, dtype), torch.randn(50, device="cuda")
        trained = [t.requires_grad_() for i, t in enumerate((w, b)) if mask >> i & 1]
        y = float4_linear(x, w, b)
        assert y.shape == (0, 50) and y.dtype is dtype
        for t, g in zip(trained, torch.autograd.grad(y, trained, torch.zeros_like(y))):
            assert g.shape == t.shape and g.dtype is t.dtype and not g.any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [(1, 64, 64), (1, 4096, 1024), (3, 1000, 99), (8, 4096, 336), (16, 14336, 128),
                                  (17, 640, 77), (40, 5000, 100), (64, 4096, 600), (100, 2048, 1031),
                                  (1, 200, 20000), (5, 1, 40), (16, 31, 5000)], ids=str)
def test_a_kept_weight_serves(size, dtype) -> None:
    m, k, n = size
    x, w = _random(m, k, 10, dtype, 0.5), _random(n, k, 11, spread=0.3) * k ** -0.5
    bias = torch.randn(n, device="cuda", dtype=dtype) if n % 2 else None
    kept = float4_quantize(w, tiles=True)
    y = float4_linear(x, kept, bias)
    assert y.dtype is dtype
    _check(y, oracle.quantize(x)[0], oracle.quantize(w, BLOCK)[0], bias)
    # The same rows from a strided x.
    wide = torch.cat([x, x], 1)[:, :k]
    assert torch.equal(float4_linear(wide, kept, bias), y)
    assert torch.equal(float4_linear(torch.cat([x, x], 1)[:, k:], kept, bias), y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [(2, 300, 5104), (3, 520, 5105), (1, 2400, 5121), (16, 257, 10240), (5, 1300, 10245),
                                  (7, 700, 16384), (1, 256, 16385), (16, 1281, 16399), (9, 600, 33001),
                                  (4, 1000, 65520), (16, 513, 65521), (2, 770, 70001), (1, 31, 131073)], ids=str)
def test_a_few_rows_on_weights_of_many(size, dtype) -> None:
    """Around the weight's rows at which the kernel's form changes, and past each form's workgroups;
    whole and ragged depths, from one stage to more than every wave takes."""
    m, k, n = size
    x, w = _random(m, k, 10, dtype, 0.5), _random(n, k, 11, spread=0.3) * k ** -0.5
    bias = torch.randn(n, device="cuda") if n % 2 else None
    kept = float4_quantize(w, tiles=True)
    _check(float4_linear(x, kept, bias), oracle.quantize(x)[0], kept.values().cpu().double(), bias)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_rows_output_does_not_depend_on_the_rows_beside_it(dtype) -> None:
    """Among the few rows that one launch serves."""
    x, w = _random(16, 3000, 10, dtype, 0.5), _random(700, 3000, 11, spread=0.3)
    kept = float4_quantize(w)
    y = float4_linear(x, kept)
    assert all(torch.equal(float4_linear(x[i:i + 1], kept), y[i:i + 1]) for i in range(16))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [(16, 8192, 4096), (16, 4096, 5104), (8, 4097, 5104), (16, 2048, 5105), (8, 2049, 16384), (16, 300, 16385),
                                  (8, 4100, 16390), (16, 256, 66000), (8, 5000, 66000)], ids=str)
def test_a_rows_output_does_not_depend_on_the_rows_beside_it_up_to_those_of_one_launch(size, dtype) -> None:
    """The most rows that one launch serves, for each of the kernel's forms and on both sides of where they end."""
    m, k, n = size
    x, w = _random(m, k, 10, dtype, 0.5), _random(n, k, 11, spread=0.3)
    kept = float4_quantize(w, tiles=True)
    y = float4_linear(x, kept)
    for rows in (1, 2, 5, m - 1):
        assert torch.equal(float4_linear(x[:rows], kept), y[:rows])
    assert torch.equal(float4_linear(x[m - 1:], kept), y[m - 1:])


@pytest.mark.parametrize("rows", [3, 40])
def test_a_tokens_nan_stays_its_own(rows) -> None:
    x, kept = _random(rows, 500, 1), float4_quantize(_random(99, 500, 2))
    want = float4_linear(x, kept)
    x[1, 300], x[2, 0] = float("nan"), -float("inf")
    got = float4_linear(x, kept)
    assert got[1:3].isnan().all()
    keep = [i for i in range(rows) if i not in (1, 2)]
    assert torch.equal(got[keep], want[keep])


def test_the_module() -> None:
    layer = Float4Linear(130, 70).cuda()
    x = _random(20, 130, 1)
    y = layer(x)
    assert torch.equal(y, float4_linear(x, layer.weight, layer.bias))
    with torch.no_grad():
        assert torch.allclose(layer(x), float4_linear(x, layer.quantized_weight(), layer.bias), rtol=1e-5, atol=1e-5)
    torch.manual_seed(3)
    first = torch.autograd.grad(layer(x).square().sum(), layer.weight)[0]
    torch.manual_seed(3)
    assert torch.equal(torch.autograd.grad(layer(x).square().sum(), layer.weight)[0], first)


def test_another_stream_and_a_graph() -> None:
    kept = float4_quantize(_random(500, 640, 1), tiles=True)
    x = _random(9, 640, 2, torch.bfloat16)
    w = torch.nn.Parameter(_random(300, 640, 3))
    dy = _random(9, 300, 4, torch.bfloat16)
    xg = x.clone().requires_grad_()
    seed = torch.tensor([11], device="cuda")

    def train():
        return torch.autograd.grad(float4_linear(xg, w, seed=seed), (xg, w), dy)

    want = [float4_linear(x, kept), *train()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [float4_linear(x, kept), *train()]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [float4_linear(x, kept), *train()]
    seen = []
    for k in range(4):
        with torch.no_grad():
            if k % 2 == 0:
                x.copy_(_random(9, 640, 20 + k, torch.bfloat16))
                xg.copy_(x)
            seed += 1  # read by the replay: new bits for the same gradient
        graph.replay()
        torch.cuda.synchronize()
        now = [float4_linear(x, kept), *train()]
        assert all(torch.equal(a, b) for a, b in zip(out, now))
        seen.append(out[2].clone())
    assert not torch.equal(seen[0], seen[1])


def test_a_modules_seed_gives_a_replayed_graph_new_bits() -> None:
    layer, x, dy = Float4Linear(300, 200).cuda(), _random(40, 300, 1).requires_grad_(), _random(40, 200, 2)
    layer.seed = torch.tensor([3], device="cuda")

    def train():
        return torch.autograd.grad(layer(x), (x, layer.weight, layer.bias), dy)

    first = train()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = train()
    seen = [first]
    for seed in (3, 4, 5, 4):
        layer.seed.fill_(seed)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, train()))
        seen.append([t.clone() for t in out])
    assert all(torch.equal(a, b) for a, b in zip(seen[0], seen[1]))
    assert all(torch.equal(a, b) for a, b in zip(seen[2], seen[4]))
    for i in (0, 1):  # db is a plain sum
        assert not torch.equal(seen[1][i], seen[2][i]) and not torch.equal(seen[2][i], seen[3][i])


def test_two_graphs_keep_their_scratch_apart() -> None:
    x, y = _random(100, 4096, 1, torch.bfloat16), _random(100, 4096, 2, torch.bfloat16)
    kept = float4_quantize(_random(512, 4096, 3), tiles=True)
    want = [float4_linear(t, kept) for t in (x, y)]
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph, t in zip(graphs, (x, y)):
        with torch.cuda.graph(graph):
            outs.append(float4_linear(t, kept))
    for _ in range(3):
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for graph, stream in zip(graphs, streams):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_runs_repeat_bit_for_bit() -> None:
    x, w = _random(1000, 1000, 1).requires_grad_(), _random(700, 1000, 2).requires_grad_()
    b = torch.randn(700, device="cuda", requires_grad=True)
    dy = _random(1000, 700, 3)
    runs = [[y := float4_linear(x, w, b, seed=2), *torch.autograd.grad(y, (x, w, b), dy)] for _ in range(3)]
    for other in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(runs[0], other))


def test_operands_past_32_bit_offsets() -> None:
    """Codes past 2^32 bytes: the last rows of a tall operand must be read from their place."""
    rows, depth = (1 << 25) + 100, 256
    data = torch.zeros(rows, depth // 2, dtype=torch.uint8, device="cuda")
    scale = torch.full((8, rows + 12), 127, dtype=torch.uint8, device="cuda")
    tail = float4_quantize(_random(200, depth, 1))
    data[-200:] = tail.data
    scale[:, rows - 200:rows] = tail.scale[:, :200]
    tall = Float4Matrix(data, scale, depth)
    x = float4_quantize(_random(3, depth, 2))
    for got in (float4_matmul(x, tall)[:, -200:], float4_matmul(tall, x)[-200:].t(),
                float4_linear(x.values(), tall)[:, -200:]):
        _check(got, x.values().cpu().double(), tail.values().cpu().double())


def test_a_matrix_past_32_bit_offsets_is_quantized_from_its_place() -> None:
    """More than 2^32 elements, and 2^32 pairs of them for the noise."""
    rows, cols = (1 << 25) + 200, 256 + 2
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-300:] = _random(300, cols, 1, torch.bfloat16)
    tail = slice(rows - 300, rows)
    q = float4_quantize(x)
    values, byte = oracle.quantize(x[tail])
    assert torch.equal(q.scale[:byte.shape[0], tail].cpu().int(), byte.int())
    part = Float4Matrix(q.data[tail].clone(), torch.nn.functional.pad(q.scale[:, tail], (0, 4)).contiguous(), cols)
    assert torch.equal(part.values().cpu().double(), values)
    del q
    q = float4_quantize(x, seed=4)
    bits = oracle.noise(4, 300, cols, first_row=rows - 300)
    values, byte = oracle.quantize(x[tail], 1, bits)
    part = Float4Matrix(q.data[tail].clone(), torch.nn.functional.pad(q.scale[:, tail], (0, 4)).contiguous(), cols)
    assert torch.equal(part.values().cpu().double(), values)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_small_values_of_16_bits_are_rounded_before_the_noise(dtype) -> None:
    """By chance a scaled magnitude below 1 is rounded to a multiple of 2^-23 first. Where that rounding decides:
    values that go up to 0.5 rounded, and down to 0 if what is below 2^-23 were cut."""
    rows, cols, seed = 2048, 2048, 3
    bits = oracle.noise(seed, rows, cols)
    least = 2 ** 22 - bits  # multiples of 2^-23 from which on the value goes up
    x = torch.full((rows, cols), 6 * 2.0 ** 12)  # every block's scale is 2^12
    near = least < 1024
    x[near] = (least[near] - 0.25).float() * 2.0 ** (12 - 23)
    x = x.to(dtype)
    parts = x[near].double() * 2.0 ** (23 - 12)
    decided = (parts.round() >= least[near]) & (parts.floor() < least[near])
    assert int(decided.sum()) > 20
    got = float4_quantize_both(x.cuda(), seed=seed)
    _same(got[0], x, bits=bits)
    _same(got[1], x.t(), bits=bits.t())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("seed", [None, 3])
def test_quantization_of_16_bit_values_at_the_edges(dtype, seed) -> None:
    """The largest and smallest values of a type, its subnormals alone and beside normal ones, ties, and
    values that are not finite."""
    most, least = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    step = least * torch.finfo(dtype).eps  # the smallest subnormal
    x = torch.zeros(32, 256, dtype=torch.float64)
    x[0, 0], x[0, 1], x[0, 2] = most, -most, most / 2
    x[1] = torch.arange(256) % 128 * step
    x[2, 0], x[2, 1:100] = -least, torch.arange(1, 100) * step
    x[3, 0], x[3, 1] = step, -step
    x[4, 0], x[4, 1:] = 6.0, torch.arange(1, 256) * step
    x[5] = 2.0 ** -torch.arange(0, 256).clamp(max=140).double()
    x[6, 0], x[6, 40], x[6, 41] = float("inf"), 2.0, -1.0
    x[7, 5], x[7, 100] = float("nan"), -float("inf")
    x[8, :32] = torch.arange(32) * 0.25
    x[9] = least
    x[10, 0], x[10, 1] = 7.0, 6.96875
    x = x.to(dtype)
    bits = None if seed is None else oracle.noise(seed, *x.shape)
    got = float4_quantize_both(x.cuda(), seed=seed)
    for q, source, noise in zip(got, (x, x.t()), (bits, None if bits is None else bits.t())):
        values, byte = oracle.quantize(source, 1, noise)
        assert torch.equal(q.scale[:byte.shape[0], :source.shape[0]].cpu().int(), byte.int())
        now = q.values().cpu().double()
        assert torch.equal(now.isnan(), values.isnan())
        assert torch.equal(now.nan_to_num(), values.float().double().nan_to_num())
    if seed is None:
        alone = float4_quantize(x.cuda())
        assert torch.equal(alone.data, got[0].data) and torch.equal(alone.scale[:, :32], got[0].scale[:, :32])
