"""Rotary positions in float64, angles from exact fractions of a turn, with the error that the
kernels' roundings allow for each element (test infrastructure).

Roundings counted, u = half a step of the 16-bit type relative to the value:
* the result rounded once: u |result|, and half the type's smallest step;
* a sine or cosine: the angle in half turns rounded to float32 (2^-24 of at most 1, times pi), two
  float32 steps of the function itself and of its product with the magnitude: 2^-21 in all;
* the two products and their sum: 2^-22 of the sum of absolute values.
"""
from __future__ import annotations

import math
from fractions import Fraction

import torch

from oracle.adapters import floor, half_step

PI = Fraction(3141592653589793238462643383279502884197169399375105820974944592307816406286, 10 ** 75)


def turned(x, positions, frequencies, magnitude, rotary, interleaved, inverse=False):
    """x [rows, heads, dims] on the CPU -> (float64 result, its error)."""
    u, tiny, dtype = half_step(x.dtype), floor(x.dtype), x.dtype
    x = x.double()
    angles = [[float(Fraction(f) * p / (2 * PI) % 1) * 2 * math.pi for f in frequencies] for p in positions.tolist()]
    angle = torch.tensor(angles, dtype=torch.float64).view(len(positions), 1, -1)
    c, s = angle.cos() * magnitude, angle.sin() * magnitude * (-1 if inverse else 1)
    first = torch.arange(0, rotary, 2) if interleaved else torch.arange(rotary // 2)
    other = first + 1 if interleaved else first + rotary // 2
    a, b = x[..., first], x[..., other]
    out, err = x.clone(), torch.zeros_like(x)
    out[..., first], out[..., other] = a * c - b * s, b * c + a * s
    e = (a.abs() + b.abs()) * magnitude * (2.0 ** -21 + 2.0 ** -22)
    err[..., first], err[..., other] = e, e
    turning = torch.zeros(x.shape[-1], dtype=torch.bool)
    turning[:rotary] = True
    return out, torch.where(turning, err + u * (out.abs() + err) + tiny, 0.0)
