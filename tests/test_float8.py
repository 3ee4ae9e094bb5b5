"""Refusals of the 8-bit matrices and the linear layer, and the oracle's rounding (CPU)."""

from __future__ import annotations

import pytest
import torch

from dionw_amd import (
    Float8Linear,
    Float8Matrix,
    _lib,
    float8_linear,
    float8_matmul,
    float8_quantize,
)
from tests import float8_oracle as oracle


def _matrix(rows=4, cols=200):
    depth = -(-cols // 128) * 128
    return Float8Matrix(torch.zeros(rows, depth, dtype=torch.uint8).view(torch.float8_e4m3fn),
                        torch.zeros(depth // 128, 16, dtype=torch.uint8), cols)


def test_the_oracles_rounding_is_to_the_nearest_code() -> None:
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    codes = codes[codes.isfinite()]
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(500, 128, generator=gen, dtype=torch.float64).mul(3).exp()
    values, byte = oracle.quantize(x)
    power = 2.0 ** (byte.double() - 127).t()
    for row in range(0, 500, 50):
        u = x[row] / power[row]
        best = (u[:, None] - codes).abs().amin(1)
        assert torch.equal((values[row] / power[row] - u).abs(), best)
        assert 224 < u.abs().max() <= 448


def test_a_matrix_checks_its_parts() -> None:
    good = _matrix()
    assert good.shape == (4, 200) and not good.values().any()
    data, scale = good.data, good.scale
    for bad in ((data.view(torch.uint8), scale, 200), (data, scale.int(), 200)):
        with pytest.raises(TypeError):
            Float8Matrix(*bad)
    for bad in ((data, scale, 257), (data, scale, 128), (data, scale[:1], 200), (data, scale[:, :3].contiguous(), 200),
                (data[:, ::2], scale, 100), (data.view(-1), scale, 200),
                (torch.zeros(4, 512, dtype=torch.uint8).view(torch.float8_e4m3fn)[:, :256], scale, 200)):
        with pytest.raises(ValueError):
            Float8Matrix(*bad)


@pytest.mark.parametrize("call", [
    lambda: float8_quantize(torch.ones(4, 8)),
    lambda: float8_quantize(torch.ones(4, 8, dtype=torch.float64)),
    lambda: float8_quantize(torch.ones(8)),
    lambda: float8_quantize(torch.ones(4, 8, dtype=torch.int32)),
    lambda: float8_matmul(_matrix(), _matrix()),
    lambda: float8_matmul(_matrix(), _matrix(4, 201)),
    lambda: float8_matmul(_matrix(), _matrix(), dtype=torch.float64),
    lambda: float8_matmul(_matrix(), _matrix(), torch.ones(5)),
    lambda: float8_linear(torch.ones(3, 200), torch.ones(4, 200)),
    lambda: float8_linear(torch.ones(3, 200), _matrix()),
    lambda: float8_linear(torch.ones(3, 200, requires_grad=True), _matrix()),
    lambda: float8_linear(torch.ones(3, 100), torch.ones(4, 200)),
    lambda: float8_linear(torch.ones(3, 200), torch.ones(4, 5, 200)),
    lambda: float8_linear(torch.ones(()), torch.ones(4, 200)),
    lambda: float8_linear(torch.ones(3, 200), torch.ones(4, 200), torch.ones(3)),
    lambda: Float8Linear(8, 4)(torch.ones(2, 8)),
], ids=lambda _: "call")
def test_refusals(call, monkeypatch) -> None:
    monkeypatch.setattr(_lib, "call", lambda name, *args: pytest.fail(f"{name} was launched"))
    with pytest.raises(ValueError):
        call()


def test_the_library_checks_its_arguments() -> None:
    """Rejected before anything is launched: no address here is one of a GPU."""
    def quantize(elem=2, rows=4, cols=200, ld=200, data=16, data_ld=256, scale=16, scale_ld=4, data_t=None):
        _lib.call("dionw_float8_quantize", elem, 16, rows, cols, ld, 0, data, data_ld, scale, scale_ld,
                  data_t, 0, None, 0, 0, None, None)

    for bad in ({"elem": 3}, {"rows": -1}, {"ld": 199}, {"data": None}, {"data": 8}, {"data_ld": 255},
                {"data_ld": 200}, {"scale": None}, {"scale_ld": 3}, {"data_t": 16}):
        with pytest.raises(ValueError):
            quantize(**bad)

    def gemm(m=4, n=4, depth=256, a=16, lda=256, a_scale=16, a_scale_ld=16, b=16, elem=1, c=16, ldc=4,
             expanded=0, ldb=256, b_scale_ld=16):
        _lib.call("dionw_float8_gemm", expanded, m, n, depth, a, lda, a_scale, a_scale_ld, b, ldb, 16,
                  b_scale_ld, None, elem, c, ldc, None, 0, None)

    for bad in ({"m": -1}, {"depth": 200}, {"a": None}, {"a": 8}, {"lda": 128}, {"lda": 264},
                {"a_scale": None}, {"a_scale_ld": 3}, {"a_scale_ld": 20}, {"a_scale": 18}, {"b": None},
                {"elem": 2}, {"elem": 3}, {"expanded": 1}, {"c": None}, {"ldc": 3}, {"lda": 1 << 23}):
        with pytest.raises(ValueError):
            gemm(**bad)
    with pytest.raises(ValueError, match="4 GB"):  # 2 blocks' scales at a pitch of 2 GB
        gemm(a_scale_ld=1 << 31)
    # A depth that is split needs its workspace.
    size = _lib.library().dionw_float8_gemm_workspace(0, 64, 64, 1 << 16)
    assert size > 0
    with pytest.raises(ValueError, match="workspace"):
        gemm(m=64, n=64, depth=1 << 16, lda=1 << 16, ldb=1 << 16, a_scale_ld=64, b_scale_ld=64, ldc=64)

    def expand(data=16, data_ld=256, scale_ld=4, depth=256, out_ld=256):
        _lib.call("dionw_float8_expand", data, data_ld, 16, scale_ld, 4, depth, 16, out_ld, None)

    for bad in ({"data": None}, {"data": 8}, {"data_ld": 128}, {"scale_ld": 3}, {"depth": 130}, {"out_ld": 255}):
        with pytest.raises(ValueError):
            expand(**bad)


def test_a_forward_refuses_what_its_gradients_could_not_sum() -> None:
    """Products take rows of less than 8 MB: a layer whose gradients need longer ones says so first."""
    def forward(m, n, w_elem, need_x, need_w):
        _lib.call("dionw_float8_linear_forward", 1, 16, 128, w_elem, 16, 128, None, m, n, 128, need_x,
                  need_w, 16, 16, None, 0, None)

    for bad in ((1 << 23, 4, 1, 0, 1), (1 << 22, 4, 2, 0, 1), (4, 1 << 23, 1, 1, 0), (1 << 62, 4, 1, 0, 1)):
        with pytest.raises(ValueError, match="8 MB"):
            forward(*bad)
    with pytest.raises(ValueError, match="scratch"):
        forward(1 << 22, 4, 1, 0, 1)
