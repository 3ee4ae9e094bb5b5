"""Quantization to e2m1 with a scale per block of 32, in float64 from its definition (torch on the
CPU; no code of the package)."""

from __future__ import annotations

import torch
from torch import Tensor

BLOCK = 32
M32 = 0xFFFFFFFF


def _powers(exponent: Tensor) -> Tensor:
    return ((exponent.to(torch.int64) + 1023) << 52).view(torch.float64)


def _mix(x: Tensor) -> Tensor:
    x = x ^ (x >> 16)
    x = (x * 0x9E3779B1) & M32
    x = x ^ (x >> 15)
    x = (x * 0x85EBCA77) & M32
    return x ^ (x >> 16)


def noise(seed: int, rows: int, cols: int, first_row: int = 0) -> Tensor:
    """22 random bits for every element of the rows from ``first_row`` on, int64 [rows, cols]."""
    pairs = (cols + 1) // 2
    p = torch.arange(first_row * pairs, (first_row + rows) * pairs)
    key = _mix(torch.tensor(((seed & M32) + 0x9E3779B1 * (((seed >> 32) & M32) + 1)) & M32))
    h = _mix((p & M32) ^ _mix((key + (p >> 32)) & M32))
    return torch.stack([h >> 10, (h & 0xFFFF) << 6], 1).view(rows, 2 * pairs)[:, :cols]


def quantize(x: Tensor, rows: int = 1, bits: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """The values of ``x`` rounded to e2m1 in blocks of ``rows`` x 32, to nearest or up by ``bits`` of
    2^22, and every row's scale exponents as kept: bytes [column blocks, rows]."""
    x = x.detach().cpu().double()
    m, n = x.shape

    def blocks(t: Tensor) -> Tensor:
        full = torch.nn.functional.pad(t, (0, -n % BLOCK, 0, -m % rows))
        return full.view(full.shape[0] // rows, rows, -1, BLOCK)

    v = blocks(x)
    bad = ~v.isfinite().all(3, keepdim=True).all(1, keepdim=True)
    v = torch.where(bad, torch.zeros_like(v), v)
    most = v.abs().amax((1, 3), keepdim=True)
    mantissa, exponent = torch.frexp(most / (7 if bits is None else 6))
    exponent = torch.where(mantissa == 0.5, exponent - 1, exponent)
    exponent = torch.where(most > 0, exponent, torch.full_like(exponent, -126)).clamp(min=-126)
    scale = _powers(exponent)
    u = v.abs() / scale
    unit = _powers((torch.frexp(u)[1] - 1).clamp(min=0) - 1)
    if bits is None:
        q = ((u / unit).round() * unit).clamp(max=6)
    else:
        u = torch.where(u < 1, (u * 2.0 ** 23).round() / 2.0 ** 23, u)
        q = (u / unit + blocks(bits.double()) / 2.0 ** 22).floor() * unit
    q = torch.where(bad, torch.full_like(v, float("nan")), q * scale * v.sign())
    byte = torch.where(bad, torch.full_like(exponent, 255), exponent + 127)
    byte = byte.expand(-1, rows, -1, 1).reshape(-1, v.shape[2])[:m]
    return q.reshape(-1, v.shape[2] * BLOCK)[:m, :n], byte.t()
