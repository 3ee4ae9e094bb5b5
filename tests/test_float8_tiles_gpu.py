"""Products of 8-bit matrices over the sizes where tiles, ranges of the depth and few-row kernels
change, against float64 products of the same quantized values (GPU).

The bounds are those of test_float8_gpu: float32 sums in any order, and for 16-bit outputs the cut
of each 8 columns' products to 13 bits below the exponent of the largest of them.
"""

from __future__ import annotations

import pytest
import torch

from dionw_amd import _lib, float8_linear, float8_matmul, float8_quantize
from tests.test_float8_gpu import SMALLEST, UNIT, _random

pytestmark = pytest.mark.gpu


def _check(got, a, b, bias=None):
    """``got`` against ``a @ b.T + bias``, formed in float64 on the GPU."""
    a, b = a.double(), b.double()
    want, size = a @ b.T, a.abs() @ b.abs().T
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    bound = (a.shape[1] + 1) * 2.0 ** -23 * size
    if got.dtype is not torch.float32:
        most = [torch.nn.functional.pad(t, (0, -t.shape[1] % 8)).abs().view(t.shape[0], -1, 8).amax(2)
                for t in (a, b)]
        bound = bound + 7 * 2.0 ** -13 * (most[0] @ most[1].T)
    bound = bound + UNIT[got.dtype] * (want.abs() + bound) + SMALLEST[got.dtype]
    assert bool(((got.double() - want).abs() <= bound).all())


# 256 x 256 tiles (whole, ragged, an odd and an even number of stages), 128 x 128 ones of two, three
# and more stages, 64 x 64 ones of one and of more than a ring, depths in ranges of each.
SIZES = [(4096, 1024, 4096), (4000, 1152, 4090), (3900, 2300, 4100), (2048, 256, 2048), (1500, 384, 1700),
         (1030, 640, 1290), (64, 128, 4000), (70, 1300, 900), (256, 4096, 4096), (100, 14336, 512),
         (300, 16384, 300), (2304, 8192, 768), (513, 9000, 1025), (17, 30000, 33)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_tiles_and_ranges(size, dtype) -> None:
    m, k, n = size
    a, b = float8_quantize(_random(m, k, 1, spread=0.5)), float8_quantize(_random(n, k, 2, spread=0.5))
    bias = torch.randn(n, device="cuda")
    got = float8_matmul(a, b, bias, dtype=dtype)
    _check(got, a.values(), b.values(), bias)
    assert torch.equal(got, float8_matmul(a, b, bias, dtype=dtype))


def test_depths_are_split_where_tiles_are_few() -> None:
    """Which of the sizes above go through ranges: their workspace is a whole number of outputs."""
    split = {}
    for m, k, n in SIZES:
        size = _lib.library().dionw_float8_gemm_workspace(0, m, n, -(-k // 128) * 128)
        assert size % (4 * m * n) == 0
        split[m, k, n] = size // (4 * m * n)
    assert split[4096, 1024, 4096] == 0 and split[300, 16384, 300] > 1 and split[17, 30000, 33] > 1


def test_scales_land_on_their_rows_and_blocks() -> None:
    """Codes of 1 throughout: an output is the sum over the blocks of 128 x the two rows' scales.
    Every row and block has a power of two of its own between 2^-3 and 2^3, so that the sums are
    exact."""
    gen = torch.Generator().manual_seed(3)
    for m, k, n in ((16, 256, 17), (130, 384, 130), (1500, 384, 1700), (300, 4096, 300), (4096, 1152, 4090)):
        from dionw_amd import Float8Matrix

        def ones(rows):
            data = torch.full((rows, k), 0x38, dtype=torch.uint8).cuda().view(torch.float8_e4m3fn)
            scale = torch.randint(124, 131, (k // 128, -(-rows // 16) * 16), generator=gen, dtype=torch.uint8)
            return Float8Matrix(data, scale.cuda(), k)

        a, b = ones(m), ones(n)
        sa, sb = (2.0 ** (q.scale[:, :r].double() - 127) for q, r in ((a, m), (b, n)))
        want = 128 * (sa.T.contiguous() @ sb)
        assert torch.equal(float8_matmul(a, b, dtype=torch.float32).double(), want)
        got = float8_matmul(a, b, dtype=torch.bfloat16)
        assert torch.equal(got, want.to(torch.bfloat16))


# Few rows: 64, 32 and 16 rows of W a wave; whole and ragged depths; groups of 16 in float32.
FEW = [(1, 256, 16400), (16, 384, 12300), (9, 512, 6000), (3, 768, 9000), (16, 1024, 100), (2, 130, 14000),
       (15, 128, 15), (33, 512, 12300), (64, 640, 5200)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("size", FEW, ids=str)
def test_few_rows(size, dtype) -> None:
    m, k, n = size
    x, w = _random(m, k, 5, dtype, 0.5), _random(n, k, 6, spread=0.3) * k ** -0.5
    bias = torch.randn(n, device="cuda")
    kept = float8_quantize(w, tiles=True)
    got = float8_linear(x, kept, bias)
    _check(got, float8_quantize(x).values(), kept.values(), bias)
    # A row's output does not depend on the rows beside it, nor on where x lies.
    if m <= 16:
        assert torch.equal(float8_linear(x[:1], kept, bias), got[:1])
    moved = torch.empty(m * (k + 3) + 1, dtype=dtype, device="cuda")[1:].view(m, k + 3)[:, :k]
    moved.copy_(x)
    assert torch.equal(float8_linear(moved, kept, bias), got)


def test_few_rows_with_values_that_are_not_finite() -> None:
    kept = float8_quantize(_random(200, 256, 1), tiles=True)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x = _random(5, 256, 2, dtype)
        clean = float8_linear(x, kept)
        x[1, 3], x[3, 200] = float("inf"), float("nan")
        got = float8_linear(x, kept)
        assert got[[1, 3]].isnan().all()
        assert torch.equal(got[[0, 2, 4]], clean[[0, 2, 4]])
