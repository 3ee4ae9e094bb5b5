"""AdamW state in 8 bits, packed per param group, and its step.

An AdamW group whose ``adamw_state`` is ``"8bit"`` keeps each moment as one
byte per element and one float32 scale (a power of two) per 256 elements:
``exp_avg`` in float8_e4m3fn, and the root of the second moment (``exp_avg_rms``)
as uint8 codes of an unsigned float with 4 exponent bits (bias 8) and 4 fraction
bits. The state of a group's tensors on one device lies in one allocation of
each kind (``AdamWPack``), every tensor at a multiple of 256 elements in
row-major order, and ``optimizer.state[p]`` holds views; so a step passes the
tensors' places instead of six pointers for each. What a caller puts in a view's
place is copied into the pack before the next step reads it, and a view that was
removed starts again from zeros.

The codes are rounded stochastically with bits from a hash of the step, the
tensor's position in its group and the element's index: a run, a resumed run
and every replica of a tensor round alike.
"""

from __future__ import annotations

import ctypes
from collections.abc import Mapping, Sequence
from enum import Enum
from itertools import chain
from operator import attrgetter, is_, itemgetter
from typing import Any, Final

import torch
from torch import Tensor

from dionw_amd import _lib
from dionw_amd._keys import (
    ADAMW_STEP_STATE,
    EXP_AVG_RMS_SCALE_STATE,
    EXP_AVG_RMS_STATE,
    EXP_AVG_SCALE_STATE,
    EXP_AVG_STATE,
    ParamState,
)
from dionw_amd.ema._fusion import ACTIVE_EMA

__all__ = ["AdamWPack", "AdamWState", "adamw_8bit_step", "pack_adamw"]

BLOCK: Final = 256  # elements that share a scale
_FLOAT32: Final = {torch.float32}
_DTYPE, _SHAPE, _GRAD = attrgetter("dtype"), attrgetter("shape"), attrgetter("grad")
_NONE: Final = type(None)
_KEYS: Final = (EXP_AVG_STATE, EXP_AVG_SCALE_STATE, EXP_AVG_RMS_STATE, EXP_AVG_RMS_SCALE_STATE,
                ADAMW_STEP_STATE)
_VIEWS: Final = itemgetter(*_KEYS)
_KEY_SET: Final = frozenset(_KEYS)
_set_item: Final = dict.__setitem__


class AdamWState(Enum):
    """How an AdamW group holds its moments between steps."""

    FLOAT32 = "float32"   # torch's layout: two float32 tensors like the parameter
    EIGHT_BIT = "8bit"    # one byte per element and moment, a scale per 256 elements


def _noting(name: str) -> Any:
    """A dict method that changes an entry, and notes it."""
    change = getattr(dict, name)

    def method(self: AdamWEntry, *args: Any, **kwargs: Any) -> Any:
        self.noted[0] = True
        return change(self, *args, **kwargs)

    return method


class AdamWEntry(dict[str, Any]):
    """A tensor's ``optimizer.state`` entry, which notes that a view may have been replaced or
    removed: a step asks one flag (comparing the views of 65 tensors would take 10 us of its 85)."""

    noted: list[bool] = [False]  # its pack's; this one is that of a copied entry

    def __setitem__(self, key: str, value: Any) -> None:
        if key in _KEY_SET:
            self.noted[0] = True
        _set_item(self, key, value)

    __delitem__, __ior__, update, setdefault, pop, popitem, clear = map(
        _noting, ("__delitem__", "__ior__", "update", "setdefault", "pop", "popitem", "clear"))


class AdamWPack:
    """The 8-bit state of one group's tensors on one device.

    Attributes:
        params: The tensors, ordered as in their group.
        numels, shapes: Their sizes when the state was made.
        first_blocks: Each tensor's first 256-element block.
    """

    def __init__(self, params: Sequence[Tensor]) -> None:
        device = params[0].device
        self.params = list(params)
        self.numels = [p.numel() for p in self.params]
        self.shapes = [p.shape for p in self.params]
        self.first_blocks = []
        blocks = 0
        for numel in self.numels:
            self.first_blocks.append(blocks)
            blocks += -(-numel // BLOCK)
        self.blocks = blocks
        count = len(self.params)
        self.exp_avg = torch.zeros(blocks * BLOCK, dtype=torch.uint8, device=device)
        self.rms = torch.zeros(blocks * BLOCK, dtype=torch.uint8, device=device)
        self.exp_avg_scale = torch.zeros(blocks, device=device)
        self.rms_scale = torch.zeros(blocks, device=device)
        self.steps = torch.zeros(count, device=device)
        self.scalars = torch.zeros(count, 4, device=device)  # rewritten by every step
        # The tensors' state entries, what they held when they were adopted, and whether one of
        # them has noted a change since.
        self.entries: list[AdamWEntry] = []
        self.held: list[Tensor] = []
        self.noted = [False]
        # The whole pack's host tables: a step in which every tensor has a gradient uses them.
        self.every = list(range(count))
        self.tables = self._tables(self.every)

    def _tables(self, places: Sequence[int]) -> tuple[Any, Any, Any]:
        return (_lib.int64_array([self.numels[i] for i in places]),
                _lib.int64_array([self.first_blocks[i] for i in places]),
                (ctypes.c_int32 * max(len(places), 1))(*places))

    def tables_of(self, places: list[int]) -> tuple[Any, Any, Any]:
        """Host tables of sizes, first blocks and ids of the tensors at ``places``."""
        return self.tables if places == self.every else self._tables(places)

    def views(self, place: int) -> dict[str, Tensor]:
        """The state entries of the tensor at ``place``."""
        numel, first = self.numels[place], self.first_blocks[place]
        codes = slice(first * BLOCK, first * BLOCK + numel)
        blocks = slice(first, first + -(-numel // BLOCK))
        shape = self.params[place].shape
        return {
            EXP_AVG_STATE: self.exp_avg[codes].view(torch.float8_e4m3fn).view(shape),
            EXP_AVG_SCALE_STATE: self.exp_avg_scale[blocks],
            EXP_AVG_RMS_STATE: self.rms[codes].view(shape),
            EXP_AVG_RMS_SCALE_STATE: self.rms_scale[blocks],
            ADAMW_STEP_STATE: self.steps[place],
        }

    def check(self, state: Mapping[Tensor, Mapping[str, Any]]) -> None:
        """Refuse a state that ``adopt`` could not take.

        Raises:
            ValueError: If an entry is not a tensor of the parameter's size.
        """
        for place, param in enumerate(self.params):
            entry = state.get(param, {})
            for key, view in self.views(place).items():
                held = entry.get(key)
                if held is not None and (not isinstance(held, Tensor) or held.shape != view.shape):
                    found = tuple(held.shape) if isinstance(held, Tensor) else type(held).__name__
                    raise ValueError(f"the 8-bit AdamW state {key!r} is {found}, the parameter "
                                     f"needs a tensor of shape {tuple(view.shape)}")

    def adopt(self, state: ParamState) -> None:
        """Point the tensors' state entries at the pack, copying in the values they held
        (a loaded checkpoint; torch's loader hands codes over as float32, which holds them
        exactly), zeros where there are none. A refused state changes nothing.

        Raises:
            ValueError: If an entry holds a state of another size.
        """
        self.check(state)
        entries = []
        for place, param in enumerate(self.params):
            entry = state[param]
            if not (isinstance(entry, AdamWEntry) and entry.noted is self.noted):
                entry = state[param] = AdamWEntry(entry)
                entry.noted = self.noted
            entries.append(entry)
            for key, view in self.views(place).items():
                held = entry.get(key)
                if held is None:
                    view.zero_()
                elif held.data_ptr() != view.data_ptr() or held.dtype != view.dtype:
                    view.copy_(held)
                entry[key] = view
        self.entries, self.held = entries, list(chain.from_iterable(map(_VIEWS, entries)))
        self.noted[0] = False

    def holds(self, state: ParamState, *, same_entries: bool = False) -> bool:
        """Whether the tensors' state entries are still the pack's views (values written into
        them are the pack's). Replaced or cleared ones count as they do for float32 state, once
        ``adopt`` has taken them up. ``same_entries``: the caller knows that ``state`` maps the
        tensors to the entries that were adopted."""
        if not same_entries and not all(map(is_, map(state.get, self.params), self.entries)):
            return False
        if self.noted[0]:
            try:
                self.noted[0] = not all(map(is_, chain.from_iterable(map(_VIEWS, self.entries)), self.held))
            except KeyError:
                pass
        return not self.noted[0]

    def moments(self, places: list[int], exp_avg: Tensor, rms: Tensor) -> None:
        """Write the values of the tensors at ``places``, one after another."""
        numels, first_blocks, _ = self.tables_of(places)
        _lib.call("dionw_adamw_8bit_values", numels, first_blocks, len(places), self.blocks,
                  self.exp_avg.data_ptr(), self.exp_avg_scale.data_ptr(), self.rms.data_ptr(),
                  self.rms_scale.data_ptr(), exp_avg.data_ptr(), rms.data_ptr(),
                  _lib.stream_handle(exp_avg.device))


def pack_adamw(params: Sequence[Tensor], state: ParamState) -> list[AdamWPack]:
    """One pack for each device that holds tensors of ``params``."""
    by_device: dict[torch.device, list[Tensor]] = {}
    for param in params:
        by_device.setdefault(param.device, []).append(param)
    packs = [AdamWPack(members) for members in by_device.values()]
    for pack in packs:
        pack.adopt(state)
    return packs


def adamw_8bit_step(group: dict[str, Any], pack: AdamWPack) -> None:
    """One AdamW step of the pack's tensors that have gradients.

    Raises:
        TypeError: For a parameter that is not float32.
        ValueError: For a gradient of another device or size than its parameter.
    """
    device = pack.exp_avg.device
    copies: list[tuple[Tensor, Tensor]] = []
    params, places = pack.params, pack.every
    grads = list(map(_GRAD, params))
    if _NONE in set(map(type, grads)):
        places = [place for place in places if grads[place] is not None]
        params = [params[place] for place in places]
        grads = [grads[place] for place in places]
    if not places:
        return
    dtypes = set(map(_DTYPE, params))
    if dtypes != _FLOAT32:
        raise TypeError(f"the HIP AdamW takes float32 parameters, got {dtypes}")
    shapes = pack.shapes if places is pack.every else [pack.shapes[place] for place in places]
    if (set(map(Tensor.get_device, params)) | set(map(Tensor.get_device, grads))
            != {pack.exp_avg.get_device()}
            or list(map(_SHAPE, grads)) != shapes or list(map(_SHAPE, params)) != shapes):
        raise ValueError("an 8-bit AdamW parameter and its gradient lie on the state's device "
                         "and have the shape that the state was made for")
    if set(map(_DTYPE, grads)) != _FLOAT32 or not all(map(Tensor.is_contiguous, grads)):
        grads = [grad.to(torch.float32).contiguous() for grad in grads]
    targets: Sequence[Tensor] = params
    if not all(map(Tensor.is_contiguous, params)):
        # The state is in row-major order: step row-major copies and write them back.
        targets = [param.data.contiguous() for param in params]
        copies = [(param.data, target) for param, target in zip(params, targets)
                  if not param.is_contiguous()]
    count = len(places)
    ema = ACTIVE_EMA.get()
    shadows = ema.fusable_shadows(params) if ema is not None and not copies else None
    beta1, beta2 = group["betas"]
    numels, first_blocks, ids = pack.tables_of(places)
    _lib.call("dionw_adamw_8bit", _lib.ptr_array(targets), _lib.ptr_array(grads),
              None if shadows is None else _lib.ptr_array(shadows), numels, first_blocks, ids,
              count, pack.blocks, len(pack.params), pack.exp_avg.data_ptr(),
              pack.exp_avg_scale.data_ptr(), pack.rms.data_ptr(), pack.rms_scale.data_ptr(),
              pack.steps.data_ptr(), pack.scalars.data_ptr(), float(group["lr"]), float(beta1),
              float(beta2), float(group["weight_decay"]), float(group["eps"]),
              0.0 if shadows is None else ema.fused_weight(),
              _lib.stream_handle(device))
    if shadows is not None:
        ema.mark_fused(params)
    for original, copy in copies:
        original.copy_(copy)
    if ema is not None:
        ema.stage_written(params)
