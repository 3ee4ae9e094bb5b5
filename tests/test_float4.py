"""4-bit matrices: their format, the oracle, and what is refused before anything is launched (CPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from dionw_amd import (
    Float4Linear,
    Float4Matrix,
    _lib,
    float4_linear,
    float4_matmul,
    float4_quantize,
    float4_quantize_both,
)
from tests import float4_oracle as oracle


def _matrix(rows=4, cols=200, **change):
    depth = -(-cols // 256) * 256
    parts = {"data": torch.zeros(rows, depth // 2, dtype=torch.uint8),
             "scale": torch.zeros(depth // 32, -(-rows // 16) * 16, dtype=torch.uint8), "cols": cols}
    return Float4Matrix(**(parts | change))


def test_a_matrix_checks_its_parts() -> None:
    q = _matrix()
    assert q.shape == (4, 200) and q.device == torch.device("cpu")
    for change in ({"data": torch.zeros(4, 128)}, {"scale": torch.zeros(8, 16)},
                   {"data": torch.zeros(4, 128, dtype=torch.int8)}):
        with pytest.raises(TypeError):
            _matrix(**change)
    byte = {"dtype": torch.uint8}
    with pytest.raises(ValueError):
        Float4Matrix(q.data, q.scale, 257)
    for change in ({"data": torch.zeros(4, 100, **byte)}, {"data": torch.zeros(128, **byte)},
                   {"scale": torch.zeros(7, 16, **byte)}, {"scale": torch.zeros(8, 17, **byte)},
                   {"scale": torch.zeros(8, 0, **byte)}, {"data": torch.zeros(128, 4, **byte).t()},
                   {"scale": torch.zeros(16, 8, **byte).t()}):
        with pytest.raises(ValueError):
            _matrix(**change)


def test_the_oracle_rounds_to_the_nearest_value() -> None:
    """Every value of the format is kept, and nothing in between is nearer to another one."""
    values = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    x = torch.linspace(0, 7, 70001, dtype=torch.float64)[:-1]
    blocks = torch.stack([torch.full_like(x, 7.0), x], 1)  # the first column sets the scale to 1
    got, byte = oracle.quantize(blocks)
    assert (byte == 127).all() and (got[:, 0] == 6).all()
    off = (got[:, 1] - x).abs()
    assert torch.equal(off, (values - x[:, None]).abs().amin(1))
    # Ties go to the code whose last bit is zero.
    ties = torch.tensor([[7, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -2.5]], dtype=torch.float64)
    assert oracle.quantize(ties)[0].tolist() == [[6, 0, 1, 1, 2, 2, 4, 4, -2]]


def test_the_oracle_is_right_on_average_by_chance() -> None:
    """A mean of n roundings of step at most s has a deviation of s / (2 sqrt(n)) at most: six of them."""
    n = 1 << 16
    x = torch.tensor([6.0, 5.1, -3.7, 2.2, 1.3, 0.9, -0.3, 0.01]).repeat(n, 4)
    q, _ = oracle.quantize(x, 1, oracle.noise(5, n, 32))
    assert ((q.mean(0) - x[0].double()).abs() <= 6 * 2 / (2 * n ** 0.5)).all()
    again, _ = oracle.quantize(x, 1, oracle.noise(6, n, 32))
    assert (q != again).double().mean() > 0.2


def test_noise_reaches_past_32_bits() -> None:
    """Pairs 2^32 apart have bits of their own."""
    near, far = oracle.noise(1, 1, 64), oracle.noise(1, 1, 64, first_row=1 << 27)
    assert (near != far).any()


@pytest.mark.parametrize("call", [
    lambda: float4_quantize(torch.ones(4, 8)),
    lambda: float4_quantize_both(torch.ones(4, 8)),
    lambda: float4_quantize(torch.ones(4, 8, dtype=torch.float64)),
    lambda: float4_quantize(torch.ones(8)),
    lambda: float4_quantize(torch.ones(4, 8, dtype=torch.int32)),
    lambda: float4_quantize(torch.ones(4, 8), tiles=True, seed=1),
    lambda: float4_quantize(torch.ones(4, 8), seed=torch.ones(2, dtype=torch.int64)),
    lambda: float4_quantize(torch.ones(4, 8), seed=torch.ones(1)),
    lambda: _matrix().values(),
    lambda: float4_matmul(_matrix(), _matrix()),
    lambda: float4_matmul(_matrix(), _matrix(4, 201)),
    lambda: float4_matmul(_matrix(), _matrix(), dtype=torch.float64),
    lambda: float4_matmul(_matrix(), _matrix(), torch.ones(5)),
    lambda: float4_linear(torch.ones(3, 200), torch.ones(4, 200)),
    lambda: float4_linear(torch.ones(3, 200), _matrix()),
    lambda: float4_linear(torch.ones(3, 200, requires_grad=True), _matrix()),
    lambda: float4_linear(torch.ones(3, 100), torch.ones(4, 200)),
    lambda: float4_linear(torch.ones(3, 200), torch.ones(4, 5, 200)),
    lambda: float4_linear(torch.ones(()), torch.ones(4, 200)),
    lambda: float4_linear(torch.ones(3, 200), torch.ones(4, 200), torch.ones(3)),
    lambda: Float4Linear(8, 4)(torch.ones(2, 8)),
], ids=lambda _: "call")
def test_refusals(call, monkeypatch) -> None:
    monkeypatch.setattr(_lib, "call", lambda name, *args: pytest.fail(f"{name} was launched"))
    with pytest.raises(ValueError):
        call()


def test_the_library_checks_its_arguments() -> None:
    """Rejected before anything is launched: no address here is one of a GPU."""
    def quantize(elem=2, rows=4, cols=200, ld=200, rounding=0, data=16, scale=16, scale_ld=16, data_t=None,
                 scale_t=None, scale_t_ld=0):
        _lib.call("dionw_float4_quantize", elem, 16, rows, cols, ld, rounding, 0, None, data, scale, scale_ld,
                  data_t, scale_t, scale_t_ld, None)

    for bad in ({"elem": 3}, {"rows": -1}, {"ld": 199}, {"data": None}, {"data": 8}, {"scale": None},
                {"scale": 8}, {"scale_ld": 3}, {"scale_ld": 20}, {"data_t": 16}, {"rounding": 3},
                {"rounding": -1}, {"data_t": 16, "scale_t": 16, "scale_t_ld": 199}, {"rows": 1 << 40}):
        with pytest.raises(ValueError):
            quantize(**bad)

    def values(data=16, scale=16, scale_ld=16, rows=4, cols=200, out=16):
        _lib.call("dionw_float4_values", data, scale, scale_ld, rows, cols, out, None)

    for bad in ({"data": None}, {"data": 8}, {"scale": None}, {"scale_ld": 3}, {"rows": -1}, {"out": None},
                {"rows": 1 << 40, "scale_ld": 1 << 40}):
        with pytest.raises(ValueError):
            values(**bad)

    def gemm(m=4, n=4, depth=512, a=16, a_scale=16, a_scale_ld=16, b=16, b_scale_ld=16, elem=1, c=16, ldc=4):
        _lib.call("dionw_float4_gemm", m, n, depth, a, a_scale, a_scale_ld, b, 16, b_scale_ld, None, elem, c,
                  ldc, None, 0, None)

    for bad in ({"m": -1}, {"depth": 128}, {"a": None}, {"a": 8}, {"a_scale": None}, {"a_scale": 20},
                {"a_scale_ld": 3}, {"a_scale_ld": 20}, {"b": None}, {"elem": 3}, {"c": None}, {"ldc": 3},
                {"depth": 1 << 24}, {"n": 1 << 31}):
        with pytest.raises(ValueError):
            gemm(**bad)
    with pytest.raises(ValueError, match="4 GB"):  # 16 blocks' scales at a pitch of 512 MB
        gemm(a_scale_ld=1 << 29)
    # A depth that is split needs its workspace.
    size = _lib.library().dionw_float4_gemm_workspace(64, 64, 1 << 17)
    assert size > 0
    with pytest.raises(ValueError, match="workspace"):
        gemm(m=64, n=64, depth=1 << 17, a_scale_ld=64, b_scale_ld=64, ldc=64)

    def kept(m=1, n=4, k=200, x=16, x_ld=200, w=16, w_scale=16, w_scale_ld=16, y=16, elem=1):
        _lib.call("dionw_float4_linear_kept", elem, x, x_ld, w, w_scale, w_scale_ld, None, m, n, k, y, None, 0,
                  None)

    for bad in ({"elem": 3}, {"m": -1}, {"x": None}, {"x_ld": 199}, {"w": None}, {"w": 8}, {"w_scale": None},
                {"w_scale_ld": 3}, {"y": None}, {"m": 100}, {"n": 1 << 31}):
        with pytest.raises(ValueError):
            kept(**bad)


def test_a_forward_refuses_what_its_gradients_could_not_sum() -> None:
    """Products take rows of less than 8 MB: a layer whose gradients need longer ones says so first."""
    def forward(m, n, k, need_x, need_w):
        _lib.call("dionw_float4_linear_forward", 1, 16, 1 << 62, 1, 16, 1 << 62, None, m, n, k, need_x,
                  need_w, 16, 16, None, 0, None)

    for bad in ((1 << 24, 4, 128, 0, 1), (4, 1 << 24, 128, 1, 0), (4, 4, 1 << 24, 0, 0), (1 << 62, 4, 128, 0, 1)):
        with pytest.raises(ValueError, match="8 MB"):
            forward(*bad)
    with pytest.raises(ValueError, match="scratch"):
        forward(1 << 24, 4, 128, 0, 0)


def test_plans_cover_every_extent() -> None:
    """Every product's ranges hold a stage at least, and the tiles that need two have them."""
    library = _lib.library()
    side, ranges = ctypes.c_int32(), ctypes.c_int32()
    seen = set()
    for m in (1, 17, 64, 100, 130, 1000, 3001, 8192):
        for n in (1, 99, 256, 1408, 14336, 128256):
            for depth in (256, 512, 768, 4096, 14336, 65536):
                assert library.dionw_float4_gemm_plan(m, n, depth, side, ranges) == 0
                stages = depth // 256
                per = -(-stages // ranges.value)
                last = stages - (ranges.value - 1) * per
                assert side.value in (64, 128, 256) and 1 <= ranges.value <= stages and last >= 1
                assert side.value == 64 or last >= 2
                seen.add((side.value, ranges.value > 1))
    assert {(64, False), (64, True), (128, False), (256, False)} <= seen


def test_sizes_follow_the_formats() -> None:
    """Half a byte an element and a byte for each 32, both padded."""
    sizes = (ctypes.c_size_t * 3)()
    _lib.library().dionw_float4_linear_sizes(100, 300, 500, 1, 1, 1, sizes)

    def padded(size):
        return -(-size // 256) * 256

    def matrix(rows, cols):
        depth = -(-cols // 256) * 256
        return padded(rows * depth // 2) + padded(depth // 32 * (-(-rows // 16) * 16))

    assert sizes[0] == matrix(500, 300) + matrix(500, 100)
    assert sizes[1] >= matrix(100, 500) + matrix(300, 500)
    assert sizes[2] >= matrix(100, 300) + matrix(300, 100) + padded(300 * 4)
    _lib.library().dionw_float4_linear_sizes(100, 300, 500, 0, 0, 0, sizes)
    assert sizes[0] == 0


@pytest.mark.parametrize("need_x", [0, 1])
@pytest.mark.parametrize("need_w", [0, 1])
def test_a_forward_of_no_rows_needs_no_room_to_save(need_x, need_w) -> None:
    """An expert that gets no tokens: y is empty, no gradient reads what would be saved, and nothing is launched."""
    sizes = (ctypes.c_size_t * 3)()
    _lib.library().dionw_float4_linear_sizes(0, 50, 130, need_x, need_w, 1, sizes)
    assert need_x or sizes[0] == 0
    _lib.call("dionw_float4_linear_forward", 1, None, 130, 2, 16, 130, None, 0, 50, 130, need_x, need_w, None,
              16 if sizes[0] else None, 16, sizes[1], None)


def test_which_rows_one_launch_serves() -> None:
    """Without scratch: up to 8 rows, and 16 up to the depth from which tiles are faster."""
    scratch = _lib.library().dionw_float4_linear_kept_scratch
    for n in (1, 4096, 4097, 5104, 5105, 16384, 16385, 128256):
        assert scratch(1, n, 1 << 20) == scratch(8, n, 1 << 20) == 0
        deepest = 8192 if n <= 4096 else 2048 if 5104 < n <= 16384 else 4096
        for rows in (9, 16):
            assert scratch(rows, n, deepest) == 0 and scratch(rows, n, deepest + 1) > 0
        assert scratch(17, n, 32) > 0
