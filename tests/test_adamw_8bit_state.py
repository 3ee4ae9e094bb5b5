"""The 8-bit AdamW state's entries in ``optimizer.state``: loaded, refused, replaced (CPU)."""

from __future__ import annotations

import copy
import io

import pytest
import torch

from dionw_amd._adamw_8bit import AdamWPack, pack_adamw


def _filled(params: list[torch.nn.Parameter], value: int) -> tuple[AdamWPack, dict]:
    """A pack whose every state tensor holds ``value``, and the state that views it."""
    state = {p: {} for p in params}
    (pack,) = pack_adamw(params, state)
    for t in (pack.exp_avg, pack.rms, pack.exp_avg_scale, pack.rms_scale, pack.steps):
        t.fill_(value)
    return pack, state


def _contents(pack: AdamWPack) -> list[torch.Tensor]:
    return [t.clone() for t in (pack.exp_avg, pack.rms, pack.exp_avg_scale, pack.rms_scale, pack.steps)]


@pytest.mark.parametrize("bad", [torch.ones(7), 3.0])
def test_a_refused_state_changes_nothing(bad) -> None:
    params = [torch.nn.Parameter(torch.ones(300)), torch.nn.Parameter(torch.ones(20, 30))]
    pack, state = _filled(params, 2)
    held = [dict(state[p]) for p in params]
    before = _contents(pack)
    _, other = _filled([torch.nn.Parameter(p.detach().clone()) for p in params], 5)
    loaded = dict(zip(params, other.values()))
    loaded[params[1]]["exp_avg_rms_scale"] = bad
    with pytest.raises(ValueError, match="exp_avg_rms_scale"):
        pack.adopt(loaded)
    assert all(torch.equal(a, b) for a, b in zip(_contents(pack), before))
    for param, entry in zip(params, held):
        assert all(state[param][key] is value for key, value in entry.items())


def test_a_pack_knows_when_its_state_was_replaced() -> None:
    params = [torch.nn.Parameter(torch.ones(300)), torch.nn.Parameter(torch.ones(20, 30))]
    pack, state = _filled(params, 3)
    assert pack.holds(state)
    state[params[0]]["ema_shadow"] = torch.zeros(300)  # another's entry
    state[params[0]]["exp_avg"].view(torch.uint8).fill_(1)  # written in place
    assert pack.holds(state)

    def replace(key):
        state[params[1]][key] = state[params[1]][key].clone()

    def drop():
        del state[params[1]]["exp_avg_scale"]

    def clear():
        state[params[0]].clear()

    def renew():
        state[params[1]] = dict(state[params[1]])

    for change in (*(lambda key=key: replace(key) for key in list(state[params[1]])), drop, clear,
                   renew, state.clear):
        change()
        assert not pack.holds(state)
        for param in params:
            state.setdefault(param, {})
        pack.adopt(state)
        assert pack.holds(state)
    # Cleared: from the start again.
    assert not any(t.float().any() for param in params for t in state[param].values())


def test_every_change_of_an_entry_is_noted() -> None:
    param = torch.nn.Parameter(torch.ones(300))
    pack, state = _filled([param], 3)
    new = torch.ones(300, dtype=torch.uint8)

    def ior(entry):
        entry |= {"exp_avg_rms": new}

    for change in (lambda e: e.update(exp_avg_rms=new), ior, lambda e: e.pop("exp_avg_rms"),
                   lambda e: e.popitem(), lambda e: e.__delitem__("exp_avg"), lambda e: e.clear(),
                   lambda e: (e.clear(), e.setdefault("exp_avg_rms", new))):
        change(state[param])
        assert not pack.holds(state)
        pack.adopt(state)
        assert pack.holds(state) and state[param]["exp_avg_rms"] is not new
    state[param].setdefault("exp_avg", new)  # changes nothing
    assert pack.holds(state)
    file = io.BytesIO()
    torch.save(state[param], file)
    file.seek(0)
    for other in (copy.deepcopy(state[param]), torch.load(file, weights_only=False)):
        assert other.keys() == state[param].keys()
        other.clear()
    assert pack.holds(state)
