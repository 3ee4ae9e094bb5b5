"""Layer norm: what is refused before anything is launched, and what reaches the library (CPU)."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from dionw_amd import LayerNorm, _lib, float4_layer_norm, layer_norm

OPERATORS = [pytest.param(layer_norm, id="norm"), pytest.param(float4_layer_norm, id="to 4 bits")]


@pytest.fixture
def calls(monkeypatch):
    """The library calls made, with the launches taken out."""
    made = []
    monkeypatch.setattr(_lib, "call", lambda name, *args: made.append((name, args)))
    monkeypatch.setattr(_lib, "stream_handle", lambda device=None: 0)
    return made


@pytest.mark.parametrize("operator", OPERATORS)
@pytest.mark.parametrize("arguments", [
    (torch.ones(4, 8),),
    (torch.ones(()),),
    (torch.ones(4, 0),),
    (torch.ones(4, 8, dtype=torch.float64),),
    (torch.ones(4, 8, dtype=torch.int32),),
    (torch.ones(4, 8), torch.ones(7)),
    (torch.ones(4, 8), torch.ones(4, 8)),
    (torch.ones(4, 8), torch.ones(8, dtype=torch.float64)),
    (torch.ones(4, 8), None, torch.ones(9)),
], ids=lambda _: "call")
def test_refusals(operator, arguments, monkeypatch) -> None:
    monkeypatch.setattr(_lib, "call", lambda name, *args: pytest.fail(f"{name} was launched"))
    with pytest.raises(ValueError):
        operator(*arguments)


def test_the_4_bit_norm_refuses_what_needs_a_gradient(calls) -> None:
    x, g = torch.ones(4, 8), torch.ones(8, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        float4_layer_norm(x, g)
    assert not calls
    with torch.no_grad():
        assert float4_layer_norm(x, g).shape == (4, 8)
    assert [name for name, _ in calls] == ["dionw_layer_norm_float4"]


@pytest.mark.parametrize("operator", OPERATORS)
def test_recorders_and_duals_are_refused(operator, calls) -> None:
    x = torch.ones(3, 200)

    def call(x):
        out = operator(x)
        return out if isinstance(out, torch.Tensor) else out.data

    with pytest.raises(ValueError, match="record"):
        torch.jit.trace(call, (x,), check_trace=False)
    with pytest.raises(ValueError, match="record"):
        make_fx(call)(x)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(ValueError, match="forward-mode"):
            operator(dual)
        assert not calls
        operator(x)
    assert len(calls) == 1


def test_a_forward_without_gradients_keeps_no_statistics(calls) -> None:
    x, norm = torch.ones(30, 200, requires_grad=True), LayerNorm(200)
    norm(x)
    with torch.no_grad():
        norm(x)
    layer_norm(x.detach())
    (_, recorded), *others = calls
    assert recorded[11] and recorded[12]
    assert len(others) == 2 and all(args[11:13] == (None, None) for _, args in others)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_autocast_casts_the_input_as_for_a_layer_norm(dtype, calls) -> None:
    before = torch.is_autocast_enabled("cuda"), torch.get_autocast_dtype("cuda")
    torch.set_autocast_dtype("cuda", torch.bfloat16)
    torch.set_autocast_enabled("cuda", True)
    try:
        x, norm = torch.ones(30, 200, dtype=dtype, requires_grad=True), LayerNorm(200)
        y = norm(x)
    finally:
        torch.set_autocast_enabled("cuda", before[0])
        torch.set_autocast_dtype("cuda", before[1])
    assert y.dtype is torch.float32 and calls[0][1][0] == _lib.F32
    y.sum().backward()
    assert x.grad.dtype is dtype


def test_a_module_takes_its_dimensions_as_one(calls) -> None:
    norm = LayerNorm((4, 5))
    assert norm(torch.ones(3, 2, 4, 5)).shape == (3, 2, 4, 5)
    assert calls[0][1][3:5] == (6, 20)
    for shape in ((3, 5), (4,), (3, 5, 4), (5,)):
        with pytest.raises(ValueError):
            norm(torch.ones(shape))
    assert LayerNorm(5, elementwise_affine=False)(torch.ones(2, 5)).shape == (2, 5)
    assert LayerNorm(5, bias=False)(torch.ones(2, 5)).shape == (2, 5)


def test_the_library_checks_its_arguments() -> None:
    """Rejected before anything is launched: no address here is one of a GPU."""
    def forward(elem=1, x=16, x_ld=200, rows=4, cols=200, w_elem=2, b_elem=2, y=16, mean=16, rstd=16):
        _lib.call("dionw_layer_norm_forward", elem, x, x_ld, rows, cols, w_elem, None, b_elem, None, 1e-5, y,
                  mean, rstd, None)

    for bad in ({"elem": 3}, {"x": None}, {"x_ld": 199}, {"rows": -1}, {"cols": 0}, {"cols": 1 << 31},
                {"w_elem": 3}, {"b_elem": -1}, {"y": None}, {"mean": None}, {"rstd": None}, {"rows": 1 << 26}):
        with pytest.raises(ValueError):
            forward(**bad)
    # A launch takes fewer than 2^32 threads: 16 to 1024 of them take a row.
    for rows, cols in ((1 << 28, 128), (1 << 26, 129), (1 << 26, 1024), (1 << 25, 2048), (1 << 24, 8192),
                       (1 << 22, 8193), (1 << 22, 20000)):
        with pytest.raises(ValueError, match="rows"):
            forward(rows=rows, x_ld=cols, cols=cols)

    def quantized(elem=1, x_ld=200, rows=4, data=16, scale=16, scale_ld=16):
        _lib.call("dionw_layer_norm_float4", elem, 16, x_ld, rows, 200, 2, None, 2, None, 1e-5, data, scale,
                  scale_ld, None)

    for bad in ({"elem": 3}, {"x_ld": 199}, {"data": None}, {"data": 8}, {"scale": None}, {"scale_ld": 3},
                {"rows": 1 << 26, "scale_ld": 1 << 26}):
        with pytest.raises(ValueError):
            quantized(**bad)

    def backward(elem=1, dy=16, dy_ld=200, mean=16, rstd=16, dg=16, scratch=16, size=1 << 30, rows=4, cols=200):
        _lib.call("dionw_layer_norm_backward", elem, 16, cols, dy, dy_ld, rows, cols, 2, None, mean, rstd, 16, dg, 2,
                  None, scratch, size, None)

    for bad in ({"elem": 3}, {"dy": None}, {"dy_ld": 199}, {"mean": None}, {"rstd": None}, {"scratch": None},
                {"scratch": 18}, {"size": 1}, {"rows": 1 << 22, "cols": 8193, "dy_ld": 8193}):
        with pytest.raises(ValueError):
            backward(**bad)


def test_a_second_derivative_is_refused(calls) -> None:
    """Also where the incoming gradient is a constant: the gradient depends on the inputs all the same."""
    x = torch.ones(3, 8, requires_grad=True)
    for loss in (lambda y: y.sum(), lambda y: y.square().sum()):
        (dx,) = torch.autograd.grad(loss(layer_norm(x)), x, create_graph=True)
        with pytest.raises(RuntimeError, match="second time"):
            (dx.sum() + x.sum()).backward()


@pytest.mark.parametrize("trained", ["x", "weight", "both"])
def test_a_second_derivative_is_refused_with_respect_to_any_tensor(trained, calls) -> None:
    """Also where only some tensors' gradients are asked for, an intermediate one's among them."""
    for loss in (lambda y: y.sum(), lambda y: y.square().sum()):
        x = torch.ones(3, 200, requires_grad=trained != "weight")
        w, b = torch.ones(200, requires_grad=trained != "x"), torch.ones(200, requires_grad=True)
        args = [t * 2 if t.requires_grad else t for t in (x, w, b)]
        first = [t for t in args[:2] if t.requires_grad]
        grads = torch.autograd.grad(loss(layer_norm(*args)), first, create_graph=True)
        for asked in [*first, *(t for t in (x, w) if t.requires_grad)]:
            with pytest.raises(RuntimeError, match="second time"):
                torch.autograd.grad(sum(t.sum() for t in (*grads, *first)), asked, retain_graph=True)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.functional.hessian(lambda t: layer_norm(t).square().sum(), torch.ones(3, 200))
