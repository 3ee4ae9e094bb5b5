"""Which tiles and ranges of the depth products of 8-bit matrices run on, and that the tests' sizes
reach each of them."""

from __future__ import annotations

import ctypes

import pytest
import torch

from dionw_amd import _lib, float8_matmul, float8_quantize
from tests import test_float8_gpu, test_float8_tiles_gpu
from tests.test_float8_gpu import _random

# Depths in ranges on 256 x 256 tiles: whole and ragged ones; an odd and an even number of stages
# in a range and in the last one (expanded operands have an even number in all).
CODES = [(1037, 9882, 3662), (3214, 10511, 1185), (3251, 10180, 1153), (3644, 9991, 1030), (1280, 11008, 3328)]
EXPANDED = [(1028, 4880, 3621), (1172, 5033, 3227), (1280, 5504, 3328)]


def _plan(expanded: int, m: int, k: int, n: int) -> tuple[int, int]:
    """(side, ranges) of a product."""
    side, ranges = ctypes.c_int32(), ctypes.c_int32()
    _lib.call("dionw_float8_gemm_plan", expanded, m, n, -(-k // 128) * 128, side, ranges)
    return side.value, ranges.value


@pytest.mark.parametrize("expanded", [0, 1])
def test_the_sizes_reach_every_tile_whole_and_in_ranges(expanded) -> None:
    sizes = test_float8_gpu.PRODUCTS + test_float8_tiles_gpu.SIZES + (EXPANDED if expanded else CODES)
    reached = {(side, ranges > 1) for side, ranges in (_plan(expanded, *size) for size in sizes)}
    assert reached == {(side, split) for side in (64, 128, 256) for split in (False, True)}


@pytest.mark.parametrize("expanded", [0, 1])
def test_ranges_on_large_tiles_are_odd_and_even(expanded) -> None:
    seen = set()
    for m, k, n in EXPANDED if expanded else CODES:
        side, ranges = _plan(expanded, m, k, n)
        assert side == 256 and ranges > 1
        size = _lib.library().dionw_float8_gemm_workspace(expanded, m, n, -(-k // 128) * 128)
        assert size == ranges * m * n * 4
        stages = -(-k // 128) * (1 + expanded)
        per = -(-stages // ranges)
        seen |= {("range", per % 2), ("last", (stages - (ranges - 1) * per) % 2), ("whole", m % 256 == n % 256 == 0)}
    assert len(seen) == (5 if expanded else 6)


def test_a_plan_refuses_what_is_no_product() -> None:
    for bad in ((0, 4, 128), (4, 0, 128), (4, 4, 0), (4, 4, 130), (-1, 4, 128)):
        side, ranges = ctypes.c_int32(), ctypes.c_int32()
        with pytest.raises(ValueError):
            _lib.call("dionw_float8_gemm_plan", 0, *bad, side, ranges)
    with pytest.raises(ValueError):
        _lib.call("dionw_float8_gemm_plan", 0, 4, 4, 128, None, ranges)


@pytest.mark.gpu
@pytest.mark.parametrize(("size", "dtype"), [(s, d) for s in CODES for d in (torch.bfloat16, torch.float16)]
                         + [(s, torch.float32) for s in EXPANDED], ids=str)
def test_ranges_on_large_tiles(size, dtype) -> None:
    m, k, n = size
    a, b = float8_quantize(_random(m, k, 1, spread=0.5)), float8_quantize(_random(n, k, 2, spread=0.5) * k ** -0.5)
    bias = torch.randn(n, device="cuda") if m % 2 else None
    got = float8_matmul(a, b, bias, dtype=dtype)
    test_float8_tiles_gpu._check(got, a.values(), b.values(), bias)
    assert torch.equal(got, float8_matmul(a, b, bias, dtype=dtype))
