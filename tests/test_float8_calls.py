"""What the 8-bit linear layer hands to the library, and what it refuses first (CPU).

No GPU is touched: the library's launches are replaced by a spy, so that CPU tensors pass where
GPU ones would.
"""

from __future__ import annotations

import gc
from collections.abc import Callable
from typing import Any

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from dionw_amd import Float8Matrix, _lib, float8_linear

FORWARD = "dionw_float8_linear_forward"
BIAS = 6  # the bias's place among the forward's arguments


@pytest.fixture
def calls(monkeypatch: pytest.MonkeyPatch) -> list[tuple[str, tuple[Any, ...]]]:
    """The library calls made, with the launches taken out."""
    made: list[tuple[str, tuple[Any, ...]]] = []
    monkeypatch.setattr(_lib, "call", lambda name, *args: made.append((name, args)))
    monkeypatch.setattr(_lib, "stream_handle", lambda device=None: 0)
    return made


def _kept(rows: int, cols: int) -> Float8Matrix:
    depth = -(-cols // 128) * 128
    return Float8Matrix(torch.zeros(rows, depth, dtype=torch.uint8).view(torch.float8_e4m3fn),
                        torch.zeros(depth // 128, -(-rows // 16) * 16, dtype=torch.uint8), cols)


class _Copies(TorchDispatchMode):
    """Counts the conversions of tensors of one size."""

    def __init__(self, numel: int) -> None:
        super().__init__()
        self.numel, self.count = numel, 0

    def __torch_dispatch__(self, func: Callable, types: Any, args: Any = (), kwargs: Any = None) -> Any:
        if func is torch.ops.aten._to_copy.default and args[0].numel() == self.numel:
            self.count += 1
        return func(*args, **(kwargs or {}))


def _lives(address: int) -> bool:
    return any(type(o) is torch.Tensor and o.dtype is torch.float32 and o.data_ptr() == address
               for o in gc.get_objects())


@pytest.mark.parametrize("weight", ["float", "kept"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_16_bit_bias_is_converted_once_and_held_during_the_call(weight, dtype, monkeypatch) -> None:
    """The library runs without the interpreter's lock: a temporary that is freed before the call
    may be another thread's by the time the product reads it."""
    held = []

    def spy(name: str, *args: Any) -> None:
        place = BIAS if name == FORWARD else 7
        held.append(_lives(args[place]))

    monkeypatch.setattr(_lib, "call", spy)
    monkeypatch.setattr(_lib, "stream_handle", lambda device=None: 0)
    x, bias = torch.ones(3, 200, dtype=dtype), torch.arange(37).to(dtype)
    w = torch.ones(37, 200) if weight == "float" else _kept(37, 200)
    with _Copies(37) as copies:
        float8_linear(x, w, bias)
    assert held == [True]
    assert copies.count == 1
