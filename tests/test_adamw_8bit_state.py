"""The 8-bit AdamW state's entries in ``optimizer.state``: loaded, refused, replaced (CPU)."""

from __future__ import annotations

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
