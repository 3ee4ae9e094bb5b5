"""Quantization to e4m3 with a scale per block of 128, in float64 from its definition (torch on
the CPU; no code of the package)."""

from __future__ import annotations

import torch
from torch import Tensor

TILE = 128


def _powers(exponent: Tensor) -> Tensor:
    return ((exponent.to(torch.int64) + 1023) << 52).view(torch.float64)


def quantize(x: Tensor, rows: int = 1) -> tuple[Tensor, Tensor]:
    """The values of ``x`` rounded to e4m3 in blocks of ``rows`` x 128, and every row's scale
    exponents as kept: bytes [column blocks, rows]."""
    x = x.detach().cpu().double()
    m, n = x.shape
    full = torch.nn.functional.pad(x, (0, -n % TILE, 0, -m % rows))
    v = full.view(full.shape[0] // rows, rows, -1, TILE)
    most = torch.where(v.isfinite(), v, torch.zeros_like(v)).abs().amax((1, 3), keepdim=True)
    mantissa, exponent = torch.frexp(most / 448)
    exponent = torch.where(mantissa == 0.5, exponent - 1, exponent)
    exponent = torch.where(most > 0, exponent, torch.full_like(exponent, -126)).clamp(min=-126)
    scale = _powers(exponent)
    u = torch.where(v.isfinite(), v / scale, torch.zeros_like(v))
    unit = torch.frexp(u)[1] - 1
    unit = _powers(torch.where(u != 0, unit, torch.full_like(unit, -6)).clamp(min=-6) - 3)
    q = torch.where(v.isfinite(), (u / unit).round() * unit * scale, torch.full_like(v, float("nan")))
    byte = (exponent + 127).expand(-1, rows, -1, 1).reshape(full.shape[0], -1)[:m]
    return q.view_as(full)[:m, :n], byte.t()
