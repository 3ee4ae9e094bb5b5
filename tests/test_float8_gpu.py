"""8-bit matrices, their products and the linear layer against float64 (GPU).

Quantization is exact: every code and scale must be the definition's. A product of two e4m3
values is exact in float32; the sums' error is bounded, whatever their order and even if the
adders truncate, by ``(depth + 1) x 2^-23 x sum |a| |b|``, and the result is rounded once more
to the output's type. 16-bit outputs are summed by an instruction that cuts the products of each
8 columns to 13 bits below the exponent of the largest of them: 7 products each lose less than
``2^-13`` of that largest one, which adds ``7 x 2^-13 x sum over the groups of max |a| max |b|``.
"""

from __future__ import annotations

import pytest
import torch

from dionw_amd import (
    Float8Linear,
    Float8Matrix,
    float8_linear,
    float8_matmul,
    float8_quantize,
    float8_quantize_both,
)
from tests import float8_oracle as oracle

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
SMALLEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}  # half a subnormal


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
    if got.dtype is not torch.float32:
        most = [torch.nn.functional.pad(t, (0, -t.shape[1] % 8)).abs().view(t.shape[0], -1, 8).amax(2)
                for t in (a, b)]
        bound = bound + 7 * 2.0 ** -13 * (most[0] @ most[1].T)
    bound = bound + UNIT[got.dtype] * (want.abs() + bound) + SMALLEST[got.dtype]
    error = (got.detach().cpu().double() - want).abs()
    assert got.shape == want.shape and bool((error <= bound).all()), float((error - bound).max())


SHAPES = [(1, 1), (1, 128), (128, 1), (127, 129), (128, 128), (200, 300), (3, 1000), (257, 512), (640, 77)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("tiles", [False, True])
def test_quantization_is_the_definitions(shape, dtype, tiles) -> None:
    x = _random(*shape, 1, dtype)
    rows, columns = float8_quantize_both(x, tiles=tiles)
    for got, source in ((rows, x), (columns, x.t())):
        values, byte = oracle.quantize(source, oracle.TILE if tiles else 1)
        assert got.shape == tuple(source.shape)
        assert torch.equal(got.scale[:, :source.shape[0]].cpu().int(), byte.int())
        assert torch.equal(got.values().cpu().double(), values)
        assert not got.data[:, got.cols:].view(torch.uint8).any()
    assert torch.equal(float8_quantize(x, tiles=tiles).data.view(torch.uint8), rows.data.view(torch.uint8))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_biass_gradient_is_the_sum_of_the_rows(shape, dtype) -> None:
    dy = _random(*shape, 1, dtype)
    x, w = torch.ones(shape[0], 8, device="cuda", dtype=dtype), torch.ones(shape[1], 8, device="cuda")
    b = torch.zeros(shape[1], device="cuda", requires_grad=True)
    (sums,) = torch.autograd.grad(float8_linear(x, w, b), (b,), dy)
    exact = dy.double().sum(0)
    bound = (shape[0] + 1) * 2.0 ** -24 * dy.double().abs().sum(0)
    assert bool(((sums.double() - exact).abs() <= bound).all())


def test_quantization_of_values_at_the_edges() -> None:
    """Maxima at a binade's carry, zeros, the smallest and largest floats, values that are not
    finite, ties."""
    x = torch.zeros(24, 128)
    x[1, 0] = 448.0
    x[2, 0] = torch.nextafter(torch.tensor(448.0), torch.tensor(1e9))
    x[3, 0], x[3, 1] = 2.0 ** -149, -(2.0 ** -140)
    x[4, 0], x[4, 1] = 3.4e38, -3.3e38
    x[5, 0], x[5, 1], x[5, 2] = float("inf"), 2.0, -1.0
    x[6, 0], x[6, 1], x[6, 2] = float("nan"), -float("inf"), 3.0
    x[7, :64] = torch.arange(64) * 0.5 + 416
    x[8] = 256 + torch.arange(128) * 1.0  # ties between codes 32 apart
    x[9] = torch.arange(128) * 2.0 ** -12 + 2.0 ** -3  # subnormal values beside a large one
    x[9, 0] = 448.0
    x[10] = 2.0 ** -126
    x[11, 0] = -0.0
    x[12] = float("nan")
    x = x.cuda()
    got = float8_quantize(x)
    values, byte = oracle.quantize(x)
    values = values.float().double()  # as float32 holds them: 3.4e38 rounds to 2^128
    assert torch.equal(got.scale[:, :24].cpu().int(), byte.int())
    now = got.values().cpu().double()
    assert torch.equal(now.isnan(), values.isnan())
    assert torch.equal(now.nan_to_num(), values.nan_to_num())
    # A row's values that are not finite reach its outputs alone.
    eye = torch.eye(128, device="cuda")
    out = float8_matmul(got, float8_quantize(eye), dtype=torch.float32)
    assert torch.equal(out.isnan().any(1).cpu(), values.isnan().any(1))
    finite = ~values.isnan().any(1)
    assert torch.equal(out.cpu().double()[finite], values[finite])


def test_strided_inputs() -> None:
    base = _random(300, 700, 2)
    for x in (base[:, :333], base[:, 1:334], base[::2, 4:400], base.t(), base[5:6], base[:, 3:4],
              base[0].expand(50, 700), base[:, :1].expand(300, 200)):
        got = float8_quantize(x)
        values, _ = oracle.quantize(x)
        assert torch.equal(got.values().cpu().double(), values)


# (tokens, depth, outputs): one, ragged, around every tile size, deep, wide, many tokens.
PRODUCTS = [(1, 1, 1), (1, 4096, 64), (2, 128, 16), (5, 300, 1000), (16, 256, 17), (17, 128, 128), (33, 1024, 65),
            (64, 384, 64), (65, 512, 129), (100, 14336, 256), (127, 200, 255), (128, 128, 128),
            (129, 1152, 257), (255, 640, 511), (256, 256, 256), (257, 1000, 513), (300, 2048, 300),
            (512, 896, 768), (1000, 128, 1000), (1025, 2304, 1031), (2048, 256, 2048), (8, 16384, 40)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("size", PRODUCTS, ids=str)
def test_products(size, dtype) -> None:
    m, k, n = size
    a, b = _random(m, k, 3, spread=0.5), _random(n, k, 4, spread=0.5) * k ** -0.5
    bias = torch.randn(n, device="cuda") if m % 2 else None
    qa, qb = float8_quantize(a), float8_quantize(b, tiles=n % 2 == 0)
    got = float8_matmul(qa, qb, bias, dtype=dtype)
    _check(got, qa.values().cpu().double(), qb.values().cpu().double(), bias)


def test_small_whole_numbers_are_exact() -> None:
    """Whole numbers up to 8 are exact in e4m3 beside each other, and their products' sums in
    float32: layouts, scales and both gradients must give the very float64 results."""
    gen = torch.Generator().manual_seed(5)
    for m, k, n in ((1, 300, 200), (130, 200, 99), (513, 640, 770), (300, 1024, 256)):
        def whole(*shape):
            return torch.randint(-8, 9, shape, generator=gen).float()

        # Different powers of two by row and block: the scales have to land on their rows.
        def powers(rows, cols):
            p = torch.randint(-6, 7, (rows, -(-cols // 128)), generator=gen)
            return (2.0 ** p.float()).repeat_interleave(128, 1)[:, :cols]

        x, w, dy = whole(m, k), whole(n, k), whole(m, n)
        xs = x * powers(m, k)
        got = float8_matmul(float8_quantize(xs.cuda()), float8_quantize(w.cuda()), dtype=torch.float32)
        assert torch.equal(got.cpu().double(), xs.double() @ w.double().t())
        xp, wp = (torch.nn.Parameter(t.cuda()) for t in (x, w))
        y = float8_linear(xp, wp)
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
    x, w = (torch.randint(-3, 4, s, generator=gen).float().cuda() for s in ((m, k), (n, k)))
    b, dy = torch.randint(-3, 4, (n,), generator=gen).float().cuda(), torch.randint(-3, 4, (m, n), generator=gen).float().cuda()
    steps = [torch.randint(-1, 2, s.shape, generator=gen).float().cuda() for s in (x, w, b)]
    args = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(float8_linear(*args), args, dy)

    def loss(sign):
        return (float8_linear(*[t + sign * s for t, s in zip((x, w, b), steps)]).double() * dy.double()).sum()

    slope = sum((g.double() * s.double()).sum() for g, s in zip(grads, steps))
    assert float(loss(1) - loss(-1)) == 2 * float(slope)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("size", [(1, 64, 64), (130, 200, 99), (257, 512, 385), (1000, 300, 1111)], ids=str)
def test_the_layer_trains(size, dtype) -> None:
    m, k, n = size
    x = (_random(m, k, 7, spread=0.5)).to(dtype).requires_grad_()
    w = torch.nn.Parameter(_random(n, k, 8, spread=0.3) * k ** -0.5)
    b = torch.nn.Parameter(torch.randn(n, device="cuda"))
    dy = (_random(m, n, 9, spread=0.5) * 1e-2).to(dtype)
    y = float8_linear(x, w, b)
    y.backward(dy)
    assert y.dtype is dtype and x.grad.dtype is dtype and w.grad.dtype is torch.float32
    (xq, _), (wq, _) = oracle.quantize(x), oracle.quantize(w, oracle.TILE)
    _check(y, xq, wq, b)
    _check(x.grad, oracle.quantize(dy)[0], wq.T.contiguous())
    _check(w.grad, oracle.quantize(dy.t())[0], oracle.quantize(x.t())[0])
    exact = dy.double().sum(0)
    assert bool(((b.grad.double() - exact).abs() <= (m + 1) * 2.0 ** -24 * dy.double().abs().sum(0)).all())


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
    y = float8_linear(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert (dx.dtype, dw.dtype, db.dtype) == (dtype, held, held)
    (xq, _), (wq, _) = oracle.quantize(x), oracle.quantize(w, oracle.TILE)
    _check(y, xq, wq, b)
    _check(dx, oracle.quantize(dy)[0], wq.T.contiguous())
    _check(dw, oracle.quantize(dy.t())[0], oracle.quantize(x.t())[0])
    exact = dy.double().sum(0)
    bound = (m + 1) * 2.0 ** -24 * dy.double().abs().sum(0)
    assert bool(((db.double() - exact).abs() <= bound + UNIT[held] * (exact.abs() + bound)).all())


def test_only_the_gradients_asked_for() -> None:
    x, w, b = _random(40, 130, 1), _random(50, 130, 2), torch.randn(50, device="cuda")
    dy = _random(40, 50, 3)
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(float8_linear(*full), full, dy)
    for mask in range(1, 8):
        args = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b))]
        asked = [t for t in args if t.requires_grad]
        got = torch.autograd.grad(float8_linear(*args), asked, dy)
        for g, t in zip(got, asked):
            assert torch.equal(g, want[[t is a for a in args].index(True)])


def test_leading_dimensions_broadcast_gradients_and_shared_weights() -> None:
    x = _random(60, 130, 1).view(3, 4, 5, 130).requires_grad_()
    w = torch.nn.Parameter(_random(50, 130, 2))
    y = float8_linear(x, w)
    assert y.shape == (3, 4, 5, 50)
    y.sum().backward()  # a gradient of stride 0
    flat = x.detach().reshape(60, 130).requires_grad_()
    v = torch.nn.Parameter(w.detach().clone())
    float8_linear(flat, v).backward(torch.ones(60, 50, device="cuda"))
    assert torch.equal(x.grad.view(60, 130), flat.grad) and torch.equal(w.grad, v.grad)
    # A weight used twice sums its gradients.
    u = torch.nn.Parameter(w.detach().clone())
    (float8_linear(flat.detach(), u) + float8_linear(flat.detach(), u)).backward(torch.ones(60, 50, device="cuda"))
    assert torch.equal(u.grad, 2 * v.grad)


def test_empty_extents() -> None:
    w = torch.nn.Parameter(_random(50, 130, 2))
    b = torch.nn.Parameter(torch.randn(50, device="cuda"))
    x = torch.zeros(0, 130, device="cuda", requires_grad=True)
    y = float8_linear(x, w, b)
    assert y.shape == (0, 50)
    y.sum().backward()
    assert x.grad.shape == (0, 130) and not w.grad.any() and not b.grad.any()
    empty = float8_linear(torch.zeros(4, 0, device="cuda"), torch.zeros(50, 0, device="cuda"), b.detach())
    assert torch.equal(empty, b.detach().expand(4, 50))
    assert float8_linear(torch.zeros(4, 130, device="cuda"), torch.zeros(0, 130, device="cuda")).shape == (4, 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("held", [torch.bfloat16, torch.float32])
def test_no_rows_of_an_input_without_a_gradient(dtype, held) -> None:
    """Whichever of weight and bias are trained: their gradients are zeros, in their own types."""
    x = torch.zeros(0, 130, dtype=dtype, device="cuda")
    for mask in range(1, 4):
        w, b = _random(50, 130, 2).to(held), torch.randn(50, device="cuda")
        trained = [t.requires_grad_() for i, t in enumerate((w, b)) if mask >> i & 1]
        y = float8_linear(x, w, b)
        assert y.shape == (0, 50) and y.dtype is dtype
        for t, g in zip(trained, torch.autograd.grad(y, trained, torch.zeros_like(y))):
            assert g.shape == t.shape and g.dtype is t.dtype and not g.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("size", [(1, 64, 64), (1, 4096, 1024), (3, 1000, 99), (8, 4096, 336), (16, 14336, 128),
                                  (17, 640, 77), (40, 5000, 100), (100, 2048, 1031), (1, 200, 20000)], ids=str)
def test_a_kept_weight_serves(size, dtype) -> None:
    m, k, n = size
    x, w = _random(m, k, 10, dtype, 0.5), _random(n, k, 11, spread=0.3) * k ** -0.5
    bias = torch.randn(n, device="cuda", dtype=dtype) if n % 2 else None
    kept = float8_quantize(w, tiles=True)
    y = float8_linear(x, kept, bias)
    assert y.dtype is dtype
    _check(y, oracle.quantize(x)[0], oracle.quantize(w, oracle.TILE)[0], bias)
    # The same rows alone and together, and from a strided x.
    wide = torch.cat([x, x], 1)[:, :k]
    assert torch.equal(float8_linear(wide, kept, bias), y)


def test_the_module() -> None:
    layer = Float8Linear(130, 70).cuda()
    x = _random(20, 130, 1)
    y = layer(x)
    assert torch.equal(y, float8_linear(x, layer.weight, layer.bias))
    with torch.no_grad():
        assert torch.allclose(layer(x), float8_linear(x, layer.quantized_weight(), layer.bias), rtol=1e-5, atol=1e-5)


def test_another_stream_and_a_graph() -> None:
    kept = float8_quantize(_random(500, 640, 1), tiles=True)
    x = _random(9, 640, 2, torch.bfloat16)
    w = torch.nn.Parameter(_random(300, 640, 3))
    dy = _random(9, 300, 4, torch.bfloat16)
    xg = x.clone().requires_grad_()

    def train():
        return torch.autograd.grad(float8_linear(xg, w), (xg, w), dy)

    want = [float8_linear(x, kept), *train()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [float8_linear(x, kept), *train()]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [float8_linear(x, kept), *train()]
    for k in range(4):
        with torch.no_grad():
            x.copy_(_random(9, 640, 20 + k, torch.bfloat16))
            xg.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        now = [float8_linear(x, kept), *train()]
        assert all(torch.equal(a, b) for a, b in zip(out, now))


def test_runs_repeat_bit_for_bit() -> None:
    x, w = _random(1000, 1000, 1).requires_grad_(), _random(700, 1000, 2).requires_grad_()
    b = torch.randn(700, device="cuda", requires_grad=True)
    dy = _random(1000, 700, 3)
    runs = [[y := float8_linear(x, w, b), *torch.autograd.grad(y, (x, w, b), dy)] for _ in range(3)]
    for other in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(runs[0], other))


def test_operands_past_32_bit_offsets() -> None:
    """Codes past 2^32 bytes: the last rows of a tall operand must be read from their place."""
    rows, depth = (1 << 25) + 100, 128
    data = torch.zeros(rows, depth, dtype=torch.uint8, device="cuda")
    scale = torch.full((1, rows + 12), 127, dtype=torch.uint8, device="cuda")
    tail = float8_quantize(_random(200, depth, 1))
    data[-200:] = tail.data.view(torch.uint8)
    scale[:, rows - 200:rows] = tail.scale[:, :200]
    tall = Float8Matrix(data.view(torch.float8_e4m3fn), scale, depth)
    x = float8_quantize(_random(3, depth, 2))
    for got in (float8_matmul(x, tall, dtype=torch.bfloat16)[:, -200:],
                float8_matmul(tall, x, dtype=torch.bfloat16)[-200:].t()):
        _check(got, x.values().cpu().double(), tail.values().cpu().double())
