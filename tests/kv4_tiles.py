"""Inputs that make every tile of 128 cached positions decisive for decode attention,
with the tolerance they are checked at.

Weights are nearly uniform and V is zero but for one channel per tile: a tile that is
lost, counted twice or taken from another place changes its channel by its whole value.
"""
from __future__ import annotations

import numpy as np

TILE, CHANNELS = 128, 128


def tiles(n: int) -> int:
    return -(-n // TILE)


def signature(n: int, first: int) -> np.ndarray:
    """V [n, 128]: tile first + c (c < 128) is 1 to 2 in channel c (one value a position), the
    rest 0. Stored, a group of them is s = max / 15 and z = 0, with codes 0 and 15: s c
    is within the scale's rounding of what is given."""
    v = np.zeros((n, CHANNELS))
    pos = np.arange(first * TILE, min(n, (first + CHANNELS) * TILE))
    v[pos, pos // TILE - first] = 1 + pos * 37 % 64 / 64
    return v


def attention(q, k, v, s8, drop=None, double=None):
    """q [heads, 128] over k, v [n, 128] in 64 bits, with sum of p * s8 beside it; a tile may
    be left out or counted twice."""
    s = q @ k.T * 128 ** -0.5
    p = np.exp(s - s.max(-1, keepdims=True))
    for tile, w in ((drop, 0.0), (double, 2.0)):
        if tile is not None:
            p[:, tile * TILE:(tile + 1) * TILE] *= w
    p /= p.sum(-1, keepdims=True)
    return p @ v, p @ s8


def tolerance(want, eight, eps):
    """The output's rounding; P s rounded to fp16, 2^-11 of p * 8 s of the channel's group (a code
    is taken as c - 8); the exponent's and the sums' fp32 error, 2^-13 of both."""
    return eps / 2 * np.abs(want) + 2.0 ** -11 * eight + 2.0 ** -13 * (eight + np.abs(want))
