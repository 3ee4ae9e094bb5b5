"""What the 8-bit linear layer hands to the library, and what it refuses first (CPU).

No GPU is touched: the library's launches are replaced by a spy, so that CPU tensors pass where
GPU ones would.
"""

from __future__ import annotations

import gc
from collections.abc import Callable, Iterator
from typing import Any

import pytest
import torch
import torch.utils.checkpoint
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from dionw_amd import (
    Float8Linear,
    Float8Matrix,
    _lib,
    float8_linear,
    float8_matmul,
    float8_quantize,
    float8_quantize_both,
)

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


def _float_weight(rows: int, cols: int) -> torch.Tensor:
    return torch.ones(rows, cols)


# Each of the operators as a function of a float x, for a weight [5, 200] made outside of it.
OPERATORS = [
    pytest.param(lambda x, w: float8_linear(x, w), _kept, id="kept"),
    pytest.param(lambda x, w: float8_linear(x, w), _float_weight, id="linear"),
    pytest.param(lambda x, w: float8_matmul(w, w, x[0, :5]), _kept, id="matmul"),
]
QUANTIZERS = [
    pytest.param(lambda x, w: float8_quantize(x).data, _kept, id="quantize"),
    pytest.param(lambda x, w: float8_quantize_both(x)[1].data, _kept, id="quantize both"),
]


@pytest.mark.parametrize(("operator", "weight"), OPERATORS)
def test_forward_mode_duals_are_refused(operator, weight, calls) -> None:
    """Their tangents would be dropped: a derivative of zero."""
    w, x = weight(5, 200), torch.ones(3, 200)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for grad in (torch.enable_grad, torch.no_grad):
            with grad(), pytest.raises(ValueError, match="forward-mode"):
                operator(dual, w)
        assert not calls
        operator(x, w)  # a plain tensor inside a level is served
    assert calls


def test_a_dual_bias_or_weight_is_refused(calls) -> None:
    x, w, bias = torch.ones(3, 200), torch.ones(5, 200), torch.ones(5)
    with forward_ad.dual_level():
        dual = [forward_ad.make_dual(t, torch.ones_like(t)) for t in (w, bias)]
        for call in (lambda: float8_linear(x, dual[0]), lambda: float8_linear(x, w, dual[1]),
                     lambda: float8_linear(x, _kept(5, 200), dual[1])):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
    assert not calls


@pytest.mark.parametrize(("operator", "weight"), OPERATORS + QUANTIZERS)
@pytest.mark.parametrize("recorder", ["make_fx", "make_fx before dispatch", "jit.trace"])
def test_recorders_are_refused(recorder, operator, weight, calls) -> None:
    """A recorded graph would hold the outputs' allocation and no kernel."""
    w, x = weight(5, 200), torch.ones(3, 200)
    with pytest.raises(ValueError, match="record"):
        if recorder == "jit.trace":
            torch.jit.trace(lambda x: operator(x, w), (x,), check_trace=False)
        else:
            make_fx(lambda x: operator(x, w), pre_dispatch="before" in recorder)(x)
    assert not calls


@pytest.mark.parametrize(("operator", "weight"), OPERATORS + QUANTIZERS)
def test_modes_that_record_nothing_are_served(operator, weight, calls) -> None:
    w, x = weight(5, 200), torch.ones(3, 200)
    with torch.device("cpu"), _Copies(-1):
        operator(x, w)
    assert calls


@pytest.mark.parametrize(("operator", "weight"), OPERATORS + QUANTIZERS)
def test_compiled_functions_reach_the_library_every_time(operator, weight, calls) -> None:
    w, x = weight(5, 200), torch.ones(3, 200)
    compiled = torch.compile(lambda x: operator(x + 1, w), backend="eager")
    compiled(x)
    first = len(calls)
    compiled(x)
    assert first and len(calls) == 2 * first


SAVED = slice(10, 14)  # need_x, need_w, y, saved among the forward's arguments


@pytest.mark.parametrize("grad", [torch.no_grad, torch.inference_mode])
def test_a_forward_without_gradients_prepares_none(grad, calls) -> None:
    """Parameters require gradients also where none are recorded: nothing is transposed or kept
    then, and nothing refused that only a gradient could not do."""
    x, layer = torch.ones(30, 200, requires_grad=True), Float8Linear(200, 50)
    with grad():
        y = layer(x)
    ((name, args),) = calls
    need_x, need_w, _, saved = args[SAVED]
    assert name == FORWARD and (need_x, need_w, saved) == (False, False, None)
    assert y.shape == (30, 50) and not y.requires_grad
    calls.clear()
    layer(x)
    ((_, args),) = calls
    need_x, need_w, _, saved = args[SAVED]
    assert need_x and need_w and saved


def test_a_first_pass_of_a_checkpoint_prepares_no_gradients(calls) -> None:
    x, layer = torch.ones(30, 200, requires_grad=True), Float8Linear(200, 50)
    y = torch.utils.checkpoint.checkpoint(layer, x, use_reentrant=True)
    assert y.requires_grad
    y.sum().backward()
    assert [name for name, _ in calls] == [FORWARD, FORWARD, "dionw_float8_linear_backward"]
    assert [bool(args[10] or args[11]) for _, args in calls[:2]] == [False, True]


def test_a_product_refuses_a_bias_whose_gradient_it_would_drop(calls) -> None:
    a, bias = _kept(5, 200), torch.ones(5, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        float8_matmul(a, a, bias)
    assert not calls
    float8_matmul(a, a, bias.detach())
    with torch.no_grad():
        float8_matmul(a, a, bias)
    assert [name for name, _ in calls] == ["dionw_float8_gemm"] * 2


@pytest.fixture
def autocast() -> Iterator[None]:
    """The GPU's autocast to bfloat16, as ``torch.autocast("cuda", torch.bfloat16)`` sets it."""
    before = torch.is_autocast_enabled("cuda"), torch.get_autocast_dtype("cuda")
    torch.set_autocast_dtype("cuda", torch.bfloat16)
    torch.set_autocast_enabled("cuda", True)
    yield
    torch.set_autocast_enabled("cuda", before[0])
    torch.set_autocast_dtype("cuda", before[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_autocast_casts_the_input_as_for_a_linear_layer(dtype, autocast, calls) -> None:
    x, layer = torch.ones(30, 200, dtype=dtype, requires_grad=True), Float8Linear(200, 50)
    y = layer(x)
    assert y.dtype is torch.bfloat16 and calls[0][1][0] == _lib.BF16 and calls[0][1][3] == _lib.F32
    y.sum().backward()
    assert x.grad.dtype is dtype and layer.weight.grad.dtype is layer.bias.grad.dtype is torch.float32
    calls.clear()
    with torch.no_grad():
        assert float8_linear(x, _kept(50, 200), layer.bias).dtype is torch.bfloat16
    assert calls[0][1][0] == _lib.BF16


def test_autocast_leaves_other_types_refused(autocast, calls) -> None:
    for dtype in (torch.float64, torch.int32):
        for w in (torch.ones(5, 200), _kept(5, 200)):
            with pytest.raises(ValueError):
                float8_linear(torch.ones(3, 200, dtype=dtype), w)
    assert not calls
