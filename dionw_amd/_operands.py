"""What the operators on tensors (quantized products, layer norm) share: how they read a tensor, what
they refuse, and how they call the library."""

from __future__ import annotations

from collections.abc import Callable
from typing import Any, Final

import torch
from torch import Tensor
from torch.autograd import forward_ad

from dionw_amd import _lib

DTYPES: Final = (torch.float16, torch.bfloat16, torch.float32)
CODES: Final = {dtype: _lib.elem_code(dtype) for dtype in DTYPES}

# Cheap signs of what check_unrecorded looks for: torch.jit.trace, and function modes, which
# make_fx runs under (as harmless ones do).
tracing = torch._C._is_tracing
function_modes = torch._C._len_torch_function_stack
# Of a process that has a GPU tensor, which is what asks.
_current_device = torch._C._cuda_getDevice


def check_unrecorded(*tensors: Tensor | None) -> None:
    """Kernels run on addresses, which graph recorders and forward-mode derivatives do not see: a
    recorded graph would return the outputs' memory as it was allocated, a tangent would be lost."""
    if torch.jit.is_tracing() or (function_modes() and _recorded_by_fx()):
        raise ValueError("the kernels cannot be recorded by torch.jit.trace or make_fx: the graph "
                         "would lose them")
    if forward_ad._current_level >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError("these operators have no forward-mode derivative: call them on plain "
                         "tensors, or use the backward pass")


def watched() -> bool:
    """Whether check_unrecorded is worth its while."""
    return tracing() or function_modes() or forward_ad._current_level >= 0


def _recorded_by_fx() -> bool:
    from torch.fx.experimental.proxy_tensor import get_proxy_mode  # takes a second to import

    return get_proxy_mode() is not None


def readable(x: Tensor) -> Tensor:
    """A matrix as the kernels read it: rows of adjacent elements that do not overlap."""
    adjacent = x.shape[1] <= 1 or x.stride(1) == 1
    return x if adjacent and (x.shape[0] <= 1 or x.stride(0) >= x.shape[1]) else x.contiguous()


def pitch(x: Tensor) -> int:
    """Elements between the rows of a readable matrix."""
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def once_differentiable(backward: Callable[..., Any]) -> Callable[..., Any]:
    """A backward pass whose gradients may not be differentiated again, whatever they depend on and
    with respect to whatever: where a graph of it is asked for, they raise once one is. (torch's own
    decorator lets them pass as constants where the incoming gradient is one, or where
    ``torch.autograd.grad`` asks for some tensors alone, and costs a call on every pass.)

    What refuses stands between the gradients and the incoming ones and the saved tensors, so that one
    of the latter has to depend on each input: the inputs themselves, or an empty output of the
    forward (``tie``)."""

    def run(ctx: Any, *gradients: Tensor | None) -> Any:
        if not torch.is_grad_enabled():
            return backward(ctx, *gradients)
        with torch.no_grad():
            found = backward(ctx, *gradients)
        places = [i for i, g in enumerate(found) if g is not None]
        tied = [t for t in (*gradients, *ctx.saved_tensors) if t is not None and t.requires_grad]
        refuse = torch._C._functions.DelayedError(
            b"the gradients of dionw_amd's operators are not differentiable a second time",
            len(places) + len(tied))
        refusing = refuse(*[found[i].detach().requires_grad_() for i in places], *tied)
        found = list(found)
        for i, g in zip(places, refusing if isinstance(refusing, tuple) else (refusing,)):
            found[i] = g
        return tuple(found)

    return run


def tie(y: Tensor) -> Tensor:
    """An output of no elements beside y, saved for the backward: it depends on the inputs and keeps
    none of them."""
    return y.new_empty(0)


def check_vector(name: str, v: Tensor | None, n: int, device: torch.device) -> None:
    if v is not None and (v.shape != (n,) or v.dtype not in DTYPES or v.device != device):
        raise ValueError(f"the {name} of {n} outputs is a float vector of that length on {device}, got "
                         f"{v.dtype} {tuple(v.shape)} on {v.device}")


def float_bias(bias: Tensor | None, n: int, device: torch.device) -> Tensor | None:
    """The bias as the products read it: contiguous float32, which the caller holds until the
    library call has returned (a temporary freed before it may be another thread's by then)."""
    check_vector("bias", bias, n, device)
    return None if bias is None else bias.detach().to(torch.float32).contiguous()


def scratch(size: int, device: torch.device) -> Tensor | None:
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def call(device: torch.device, name: str, *args: Any) -> None:
    """``_lib.call`` with ``device`` the current one: a default stream has no device of its own."""
    index = device.index
    if index is None or index == _current_device():
        _lib.call(name, *args)
    else:
        with torch.cuda.device(index):
            _lib.call(name, *args)
