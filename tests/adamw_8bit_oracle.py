"""The 8-bit AdamW step in float64, from its definition (numpy; no code of the package)."""

from __future__ import annotations

import math

import numpy as np

BLOCK = 256
# fraction bits, lowest normal exponent, largest value
E4M3 = (3, -6, 448.0)
U44 = (4, -7, 248.0)


def mix(x: np.ndarray) -> np.ndarray:
    """The hash of 32 bits (uint64 arrays of values below 2^32)."""
    m32 = np.uint64(0xFFFFFFFF)
    x = x ^ (x >> np.uint64(16))
    x = (x * np.uint64(0x9E3779B1)) & m32
    x = x ^ (x >> np.uint64(15))
    x = (x * np.uint64(0x85EBCA77)) & m32
    return x ^ (x >> np.uint64(16))


def noise(step: int, place: int, elements: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """The 16 random bits of m and of r for each element index."""
    m32 = np.uint64(0xFFFFFFFF)
    elements = elements.astype(np.uint64)
    key = mix(np.array([place * 0x9E3779B1 + step & 0xFFFFFFFF], np.uint64))
    bits = mix((elements & m32) ^ mix((key + (elements >> np.uint64(32))) & m32))
    return (bits & np.uint64(0xFFFF)).astype(np.float64), (bits >> np.uint64(16)).astype(np.float64)


def e4m3_values(codes: np.ndarray) -> np.ndarray:
    """float64 values of e4m3 bytes (0x7F and 0xFF are NaN)."""
    c = codes.astype(np.int64)
    field, fraction = (c >> 3) & 15, c & 7
    value = np.where(field == 0, fraction * 2.0 ** -9, (1 + fraction / 8) * 2.0 ** (field - 7.0))
    value = np.where((c & 127) == 127, np.nan, value)
    return np.where(c >= 128, -value, value)


def u44_values(codes: np.ndarray) -> np.ndarray:
    """float64 values of the unsigned bytes (4 exponent bits with bias 8, 4 fraction bits)."""
    c = codes.astype(np.int64)
    field, fraction = c >> 4, c & 15
    return np.where(field == 0, fraction * 2.0 ** -11, (1 + fraction / 16) * 2.0 ** (field - 8.0))


def blocks_of(x: np.ndarray) -> np.ndarray:
    return np.pad(x, (0, -x.size % BLOCK)).reshape(-1, BLOCK)


def block_scales(x: np.ndarray, form: tuple[int, int, float]) -> np.ndarray:
    """The smallest powers of two (at least 2^-126) that bring the blocks' finite largest
    magnitudes to the format's largest value at most."""
    most = np.where(np.isfinite(x), np.abs(x), 0).max(1, initial=0)
    mantissa, exponent = np.frexp(most / form[2])
    exponent = np.where(mantissa == 0.5, exponent - 1, exponent)
    return 2.0 ** np.maximum(np.where(most > 0, exponent, -126), -126).astype(np.float64)


def rounded(x: np.ndarray, scale: np.ndarray, bits: np.ndarray,
            form: tuple[int, int, float]) -> tuple[np.ndarray, np.ndarray]:
    """Magnitudes of blocks rounded by ``bits`` / 2^16, as values, and how far each was from
    being rounded to the neighbour, in units of its last place."""
    u = np.abs(x) / scale[:, None]
    exponent = np.frexp(u)[1] - 1
    unit = 2.0 ** (np.maximum(np.where(u > 0, exponent, form[1]), form[1]) - form[0])
    count = u / unit + bits / 65536
    value = np.floor(count) * unit * scale[:, None]
    return value, np.abs(count - np.round(count))


def update(p, g, m0, r0, step, place, *, lr, beta1, beta2, eps, weight_decay):
    """One step of a tensor from float64 values: new p, m and r before rounding, and the
    rounding's scales and noise by block."""
    m = beta1 * m0 + (1 - beta1) * g
    r = np.sqrt(beta2 * r0 ** 2 + (1 - beta2) * g ** 2)
    p = (p * (1 - lr * weight_decay)
         - lr / (1 - beta1 ** step) * m / (r / math.sqrt(1 - beta2 ** step) + eps))
    bits = noise(step, place, np.arange(g.size))
    return p, m, r, bits
