"""The 8-bit linear layer as evaluation and 16-bit models call it (GPU)."""

from __future__ import annotations

import pytest
import torch

from dionw_amd import Float8Linear, float8_linear
from tests.test_float8_gpu import _random

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
