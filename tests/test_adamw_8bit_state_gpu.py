"""The 8-bit AdamW state's entries in ``optimizer.state``: loaded, refused, replaced (GPU)."""

from __future__ import annotations

import copy

import pytest
import torch

from dionw_amd import AdamWState, Dion, EMAConfig, StepGraph
from tests.test_adamw_8bit_gpu import HYPER, _grads, _optimizer, _tensors

pytestmark = pytest.mark.gpu


def _pair(sizes, steps=2, **more):
    """Two optimizers in the same state after ``steps`` steps."""
    params = _tensors(sizes)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    opt, twin = _optimizer(params, **more), _optimizer(twins, **more)
    for k in range(steps):
        _step(opt, params, twin, twins, k)
    return opt, params, twin, twins


def _step(opt, params, twin, twins, seed):
    _grads(params, seed)
    for p, q in zip(params, twins):
        q.grad = p.grad.clone()
    opt.step()
    twin.step()


def _same(opt, params, twin, twins):
    for p, q in zip(params, twins):
        assert torch.equal(p, q)
        assert set(opt.state[p]) == set(twin.state[q])
        for key, value in opt.state[p].items():
            if isinstance(value, torch.Tensor):
                assert value.dtype is twin.state[q][key].dtype
                assert torch.equal(value.float(), twin.state[q][key].float()), key


@pytest.mark.parametrize("key", ["exp_avg", "exp_avg_rms_scale", "adamw_step"])
def test_a_refused_checkpoint_leaves_the_optimizer_as_it_was(key) -> None:
    """One entry of the last tensor has another size: the first tensors' must not be loaded."""
    opt, params, twin, twins = _pair([300, (20, 30), 777])
    broken = copy.deepcopy(opt.state_dict())
    for entry in broken["state"].values():
        for name in entry:
            entry[name] = torch.zeros_like(entry[name])
    broken["state"][2][key] = torch.zeros(5, device="cuda")
    held = [dict(opt.state[p]) for p in params]
    with pytest.raises(ValueError, match=key):
        opt.load_state_dict(broken)
    for param, entry in zip(params, held):
        assert all(opt.state[param][name] is value for name, value in entry.items())
    _same(opt, params, twin, twins)
    _step(opt, params, twin, twins, 9)
    _same(opt, params, twin, twins)


@pytest.mark.parametrize("ema", [False, True])
def test_replaced_entries_are_stepped_on(ema) -> None:
    """An entry that is replaced counts, as it does for float32 state: here by a copy of another
    optimizer's, which the next step must start from."""
    more = {"ema": EMAConfig(decay=0.9)} if ema else {}
    opt, params, twin, twins = _pair([300, (20, 30), 777], **more)
    _grads(params, 50)
    opt.step()  # runs ahead alone
    with torch.no_grad():
        for p, q in zip(params, twins):
            p.copy_(q)
    for p, q in zip(params, twins):
        for key, value in twin.state[q].items():
            opt.state[p][key] = value.clone() if isinstance(value, torch.Tensor) else value
    if ema:
        opt.ema.step_count = twin.ema.step_count
    for k in range(3):
        _step(opt, params, twin, twins, 60 + k)
        _same(opt, params, twin, twins)


@pytest.mark.parametrize("clear", [lambda opt, p: opt.state[p].clear(), lambda opt, p: opt.state.pop(p),
                                   lambda opt, p: opt.state[p].pop("exp_avg")])
def test_cleared_entries_start_again_and_are_saved(clear) -> None:
    opt, params, _, _ = _pair([300, 500])
    kept = {key: value.clone() for key, value in opt.state[params[1]].items()}
    clear(opt, params[0])
    saved = opt.state_dict()["state"]
    assert set(saved[0]) == set(saved[1]) == set(kept)
    assert not saved[0]["exp_avg"].view(torch.uint8).any()
    m, r = opt.adamw_moments(params)
    assert not m[:300].any() and m[300:].any()
    assert all(torch.equal(opt.state[params[1]][key].float(), value.float()) for key, value in kept.items())


def test_a_cleared_state_is_that_of_a_new_optimizer() -> None:
    opt, params, _, _ = _pair([300, 500])
    opt.state.clear()
    opt.initialize_state(params[1])
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    twin = _optimizer(twins)
    assert set(opt.state[params[1]]) == set(twin.state[twins[1]])
    for k in range(2):
        _step(opt, params, twin, twins, 70 + k)
        _same(opt, params, twin, twins)


def test_a_replaced_entry_of_another_size_is_refused() -> None:
    opt, params, _, _ = _pair([300])
    start = params[0].detach().clone()
    opt.state[params[0]]["exp_avg_scale"] = torch.ones(9, device="cuda")
    with pytest.raises(ValueError, match="exp_avg_scale"):
        opt.step()
    assert torch.equal(params[0], start)


def test_replaced_entries_are_not_recorded_in_a_graph() -> None:
    """Taking them up is a copy that a replay would repeat."""
    matrix = torch.nn.Parameter(torch.randn(128, 128, device="cuda") * 0.02)
    vector = torch.nn.Parameter(torch.randn(500, device="cuda"))
    opt = Dion([{"params": [matrix], "dion_route": "matrix"}, {"params": [vector], "dion_route": "adamw"}],
               **HYPER, adamw_state=AdamWState.EIGHT_BIT)
    for p in (matrix, vector):
        p.grad = torch.ones_like(p)
    opt.step()
    opt.state[vector]["adamw_step"] = torch.tensor(5.0, device="cuda")
    with pytest.raises(RuntimeError, match="replaced"), torch.cuda.graph(torch.cuda.CUDAGraph()):
        opt.step()
    torch.cuda.synchronize()
    graph = StepGraph(opt)  # takes them up before it records
    graph.replay()
    graph.replay()
    assert float(opt.state[vector]["adamw_step"]) == 7


def test_a_group_may_name_its_state_by_the_enum(tmp_path) -> None:
    """The group then holds the value, as with the constructor's argument: a checkpoint of either
    loads into the other, and needs no class of this package to be read."""
    params = _tensors([300])
    by_enum = Dion([{"params": params, "dion_route": "adamw", "adamw_state": AdamWState.EIGHT_BIT}], **HYPER)
    twins = _tensors([300])
    by_argument = _optimizer(twins)
    _step(by_enum, params, by_argument, twins, 1)
    _same(by_enum, params, by_argument, twins)
    for source, target in ((by_enum, by_argument), (by_argument, by_enum)):
        torch.save(source.state_dict(), tmp_path / "opt.pt")
        saved = torch.load(tmp_path / "opt.pt", weights_only=True)
        assert saved["param_groups"][0]["adamw_state"] == "8bit"
        target.load_state_dict(saved)
