"""The 8-bit linear layer as evaluation and 16-bit models call it (GPU)."""

from __future__ import annotations

import pytest
import torch

from dionw_amd import Float8Linear, _lib, float8_linear, float8_quantize, float8_quantize_both
from tests.test_float8_gpu import _random
from tests.test_float8_tiles_gpu import _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_a_forward_without_gradients_gives_the_same(dtype) -> None:
    layer = Float8Linear(260, 130).cuda()
    x = _random(300, 260, 1, dtype)
    y = layer(x)
    for grad in (torch.no_grad, torch.inference_mode):
        with grad():
            assert torch.equal(layer(x), y)
    shaped = x.view(3, 4, 25, 260)
    with torch.no_grad():
        assert torch.equal(layer(shaped), y.view(3, 4, 25, 130))


def test_rows_that_only_a_gradient_could_not_sum_are_served() -> None:
    """A weight's gradient would sum over the rows, of which products take fewer than 2^22 in
    float32: a forward without gradients has no such sum."""
    rows = (1 << 22) + 5
    x, w = torch.zeros(rows, 8, device="cuda"), torch.nn.Parameter(_random(3, 8, 2))
    x[-2:] = _random(2, 8, 3)
    with pytest.raises(ValueError, match="8 MB"):
        float8_linear(x, w)
    with torch.no_grad():
        y = float8_linear(x, w)
        assert torch.equal(y[-2:], float8_linear(x[-2:], w)) and not y[:-2].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_autocast_is_heeded(dtype) -> None:
    """A float32 activation under autocast goes the way of a 16-bit one, and gets a float32 gradient."""
    layer, kept_layer = Float8Linear(260, 130).cuda(), torch.nn.Linear(260, 130).cuda()
    x, half = _random(300, 260, 1).requires_grad_(), _random(300, 260, 1).to(dtype).requires_grad_()
    dy = _random(300, 130, 2).to(dtype)
    with torch.autocast("cuda", dtype):
        y = layer(x)
        assert y.dtype is kept_layer(x).dtype is dtype
        with torch.no_grad():
            served = float8_linear(x, layer.quantized_weight(), layer.bias)
    want = layer(half)
    assert torch.equal(y, want)
    with torch.no_grad():
        assert torch.equal(served, float8_linear(half, layer.quantized_weight(), layer.bias))
    got = torch.autograd.grad(y, (x, layer.weight, layer.bias), dy)
    for g, w in zip(got, torch.autograd.grad(want, (half, layer.weight, layer.bias), dy)):
        assert g.dtype is torch.float32 and torch.equal(g, w.float())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tiles", [0, 1])
@pytest.mark.parametrize("shape", [(1, 128), (130, 200), (257, 384)])
def test_the_library_quantizes_into_expanded_values_and_sums(shape, tiles, dtype) -> None:
    """The entry's outputs that the Python functions do not ask for: bfloat16 halves of the
    values, which are exact in it, and the sums of each 128 rows' columns."""
    (m, n), x = shape, _random(*shape, 1, dtype)
    depth, depth_t = -(-n // 128) * 128, -(-m // 128) * 128
    rows, columns = float8_quantize_both(x, tiles=bool(tiles))
    for expanded in (1, 2, 3):
        data = torch.empty(m, depth, dtype=torch.bfloat16 if expanded & 1 else torch.uint8, device="cuda")
        data_t = torch.empty(n, depth_t, dtype=torch.bfloat16 if expanded & 2 else torch.uint8, device="cuda")
        scale, scale_t = torch.empty_like(rows.scale), torch.empty_like(columns.scale)
        sums = torch.empty(-(-m // 128), n, device="cuda")
        _lib.call("dionw_float8_quantize", _lib.elem_code(dtype), x.data_ptr(), m, n, n, tiles,
                  data.data_ptr(), depth, scale.data_ptr(), scale.shape[1], data_t.data_ptr(), depth_t,
                  scale_t.data_ptr(), scale_t.shape[1], expanded, sums.data_ptr(), _lib.stream_handle(x.device))
        for got, want, bit in ((data, rows, 1), (data_t, columns, 2)):
            if expanded & bit:
                assert torch.equal(2 * got[:, :want.cols].float(), want.values())
                assert not got[:, want.cols:].any()
            else:
                assert torch.equal(got, want.data.view(torch.uint8))
        exact = torch.stack([part.double().sum(0) for part in x.split(128)])
        size = torch.stack([part.double().abs().sum(0) for part in x.split(128)])
        assert bool(((sums.double() - exact).abs() <= 128 * 2.0 ** -24 * size).all())
    alone = torch.empty(m, depth, dtype=torch.bfloat16, device="cuda")
    _lib.call("dionw_float8_quantize", _lib.elem_code(dtype), x.data_ptr(), m, n, n, tiles,
              alone.data_ptr(), depth, None, 0, None, 0, None, 0, 1, None, _lib.stream_handle(x.device))
    assert torch.equal(2 * alone[:, :n].float(), rows.values())


@pytest.mark.parametrize("rows", [16, 17, 32, 33, 64, 65])
@pytest.mark.parametrize("size", [(4096, 99), (4100, 99), (640, 4200), (14336, 300), (4224, 9000)], ids=str)
def test_float32_rows_on_a_kept_weight(rows, size) -> None:
    """Around the numbers of rows and columns at which the kernel changes, and its shapes."""
    k, n = size
    x, w = _random(rows, k, 5, spread=0.5), _random(n, k, 6, spread=0.3) * k ** -0.5
    bias = torch.randn(n, device="cuda")
    kept = float8_quantize(w, tiles=True)
    _check(float8_linear(x, kept, bias), float8_quantize(x).values(), kept.values(), bias)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 40, 300])
def test_float32_rows_have_the_codes_of_16_bit_ones_and_exact_sums(rows, dtype) -> None:
    """Products that cancel: 448 x 448 and its opposite beside 1 x 1 in each 8 columns. A 16-bit
    row may lose the small ones, the same row in float32 must not."""
    x, w = torch.ones(rows, 256, device="cuda"), torch.ones(64, 256, device="cuda")
    x[:, 0::8], x[:, 1::8] = 448.0, -448.0
    w[:, 0::8], w[:, 1::8] = 448.0, 448.0
    kept = float8_quantize(w, tiles=True)
    half = x.to(dtype)
    assert torch.equal(float8_quantize(half).data.view(torch.uint8), float8_quantize(x).data.view(torch.uint8))
    for weight in (w, kept):
        assert torch.equal(float8_linear(half.float(), weight), torch.full((rows, 64), 192.0, device="cuda"))
        _check(float8_linear(half, weight), half.float(), w)
