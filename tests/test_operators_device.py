"""The operators on tensors run on the tensors' device, whichever is the current one (CPU: the launches
are taken out, and the devices are names)."""

from __future__ import annotations

import ast
import contextlib
from pathlib import Path

import pytest
import torch

import dionw_amd
from dionw_amd import _lib, _operands

PACKAGE = Path(dionw_amd.__file__).parent


@pytest.fixture
def seen(monkeypatch):
    """What the library is called for, and on which device, the current one being 0."""
    current, made = [0], []

    @contextlib.contextmanager
    def device(index):
        before, current[0] = current[0], index
        yield
        current[0] = before

    monkeypatch.setattr(_operands, "_current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(_lib, "call", lambda name, *args: made.append((name, args, current[0])))
    return made


@pytest.mark.parametrize("index", [0, 1])
def test_a_call_is_made_on_its_device(index, seen) -> None:
    """A default stream belongs to no device of its own: launched there, a kernel runs on the current one."""
    _operands.call(torch.device("cuda", index), "entry", 1, 2)
    _operands.call(torch.device("cuda"), "entry")
    assert seen == [("entry", (1, 2), index), ("entry", (), 0)]


@pytest.mark.parametrize("module", ["float4", "float8", "layer_norm"])
def test_every_launch_goes_that_way(module) -> None:
    """All but the backward passes, which torch runs on their device."""
    tree = ast.parse((PACKAGE / f"{module}.py").read_text())
    launches = {f.name for f in ast.walk(tree) if isinstance(f, ast.FunctionDef)
                for c in ast.walk(f) if isinstance(c, ast.Call) and ast.unparse(c.func) == "_lib.call"}
    assert launches == {"backward"}
