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
