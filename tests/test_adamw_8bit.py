"""The 8-bit AdamW state's formats, hash and refusals (CPU)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from dionw_amd import AdamWState, _lib
from dionw_amd._adamw_8bit import AdamWPack, adamw_8bit_step, pack_adamw
from dionw_amd._groups import GroupSpec, refuse_structural_change
from tests import adamw_8bit_oracle as oracle


def test_the_oracles_e4m3_is_torchs() -> None:
    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(oracle.e4m3_values(codes.numpy()), want, equal_nan=True)


def test_u44_codes_are_ordered_and_cover_their_range() -> None:
    values = oracle.u44_values(np.arange(256))
    assert (np.diff(values) > 0).all()
    assert values[0] == 0 and values[1] == 2.0 ** -11 and values[255] == 248


@pytest.mark.parametrize("form", [oracle.E4M3, oracle.U44])
def test_scales_are_the_smallest_that_hold_the_block(form) -> None:
    x = np.exp(np.random.default_rng(0).normal(0, 20, (2000, 1))) * np.ones((1, 256))
    x[0] = form[2]
    x[1] = np.nextafter(form[2], 1e9)
    scale = oracle.block_scales(x, form)
    assert (x[:, 0] <= form[2] * scale).all() and (x[:, 0] > form[2] * scale / 2).all()
    assert scale[0] == 1 and scale[1] == 2


def test_the_hash_is_even_and_its_halves_independent() -> None:
    """Counts of 2^20 draws in 256 bins: chi-square with 255 degrees of freedom, mean 255 and
    standard deviation 22.6; six of them are allowed."""
    for step, place in ((1, 0), (2, 0), (1, 1), (5000, 64)):
        low, high = oracle.noise(step, place, np.arange(1 << 20))
        for bits in (low, high):
            count = np.bincount((bits / 256).astype(int), minlength=256)
            assert abs(((count - 4096) ** 2 / 4096).sum() - 255) < 6 * 22.6
        pairs = np.bincount((low / 4096).astype(int) * 16 + (high / 4096).astype(int), minlength=256)
        assert abs(((pairs - 4096) ** 2 / 4096).sum() - 255) < 6 * 22.6
    a, b = oracle.noise(1, 0, np.arange(1 << 16))[0], oracle.noise(2, 0, np.arange(1 << 16))[0]
    # The correlation of 2^16 independent pairs has a standard deviation of 2^-8.
    assert abs(np.corrcoef(a, b)[0, 1]) < 6 / 256


def test_rounding_is_unbiased() -> None:
    """The mean of 2^18 roundings of a value has a standard deviation of at most half a unit of
    the last place over 2^9; six are allowed."""
    low, high = oracle.noise(3, 2, np.arange(1 << 18))
    for bits, form in ((low, oracle.E4M3), (high, oracle.U44)):
        for value in (1.0, 1.01, 3.3, 0.001 * form[2], 1e-3, 2.0 ** -12):
            x = np.full((1, 1 << 18), value)
            got, _ = oracle.rounded(x, np.ones(1), bits[None], form)
            unit = 2.0 ** (max(np.floor(np.log2(value)), form[1]) - form[0])
            assert abs(got.mean() - value) < 6 * 0.5 * unit / 512


def test_the_pack_lays_tensors_at_whole_blocks() -> None:
    params = [torch.nn.Parameter(torch.ones(s)) for s in ((3, 100), (256,), (0,), (257,))]
    state = {p: {} for p in params}
    (pack,) = pack_adamw(params, state)
    assert pack.first_blocks == [0, 2, 3, 3] and pack.blocks == 5
    for p in params:
        entry = state[p]
        assert entry["exp_avg"].shape == p.shape and entry["exp_avg"].dtype is torch.float8_e4m3fn
        assert entry["exp_avg_rms"].dtype is torch.uint8 and entry["adamw_step"].dim() == 0
        assert entry["exp_avg_scale"].numel() == -(-p.numel() // 256)
    # Loaded values (torch hands codes over as float32) go into the pack, with all 256 codes.
    codes = torch.arange(256, dtype=torch.uint8)
    state[params[1]] = {"exp_avg": codes.view(torch.float8_e4m3fn).float(), "exp_avg_rms": codes.float(),
                        "exp_avg_scale": torch.tensor([0.5]), "adamw_step": torch.tensor(7.0)}
    pack.adopt(state)
    assert torch.equal(pack.rms[512:768], codes) and pack.steps[1] == 7
    kept = pack.exp_avg[512:768]
    nan = (codes & 127) == 127
    assert torch.equal(kept[~nan], codes[~nan]) and ((kept[nan] & 127) == 127).all()
    assert pack.exp_avg_scale[2] == 0.5 and pack.rms_scale[2] == 0


def test_refusals() -> None:
    param = torch.nn.Parameter(torch.ones(8))
    pack = AdamWPack([param])
    group = {"lr": 1e-3, "betas": (0.9, 0.95), "eps": 1e-8, "weight_decay": 0.0}
    adamw_8bit_step(group, pack)  # no gradient: nothing to do
    param.grad = torch.ones(8)
    with pytest.raises(ValueError):  # CPU tensors
        adamw_8bit_step(group, pack)
    with pytest.raises(TypeError):
        half = torch.nn.Parameter(torch.ones(8).half())
        half.grad = torch.ones(8).half()
        adamw_8bit_step(group, AdamWPack([half]))
    with pytest.raises(ValueError):
        pack.adopt({param: {"exp_avg": torch.ones(9)}})
    spec = {"params": [], "dion_route": "adamw", "lr": 1e-3, "weight_decay": 0.0, "fraction": 1.0,
            "num_heads": None, "newton_schulz": "gram", "row_normalization": "normuon",
            "momentum_form": "heavy_ball"}
    assert GroupSpec.of(spec).adamw_state is AdamWState.FLOAT32
    assert GroupSpec.of({**spec, "adamw_state": "8bit"}).adamw_state is AdamWState.EIGHT_BIT
    with pytest.raises(ValueError):
        GroupSpec.of({**spec, "adamw_state": "none"})
    refuse_structural_change([spec], [spec])
    with pytest.raises(ValueError, match="adamw_state"):
        refuse_structural_change([spec], [{**spec, "adamw_state": "8bit"}])


def test_the_library_checks_its_tables() -> None:
    """Rejected before anything is launched: no address here is one of a GPU."""
    def call(numel=8, block0=0, ids=0, count=1, blocks=1, tensors=1, p=16):
        one = _lib.int64_array
        return _lib.call(
            "dionw_adamw_8bit", (_lib.ctypes.c_void_p * 1)(p), (_lib.ctypes.c_void_p * 1)(16), None,
            one([numel]), one([block0]), (_lib.ctypes.c_int32 * 1)(ids), count, blocks, tensors,
            16, 16, 16, 16, 16, 16, 1e-3, 0.9, 0.95, 0.0, 1e-8, 0.0, None)

    for bad in ({"numel": -1}, {"numel": 257}, {"block0": 1}, {"block0": -1}, {"ids": 1}, {"ids": -1},
                {"count": -1}, {"p": None}, {"blocks": -1}):
        with pytest.raises(ValueError):
            call(**bad)
