"""The 8-bit AdamW state's entries in ``optimizer.state``: loaded, refused, replaced (GPU)."""

from __future__ import annotations

import copy

import pytest
import torch

from tests.test_adamw_8bit_gpu import _grads, _optimizer, _tensors

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
