"""The decode attention's tile test itself, on the CPU: with its inputs, the oracle without
one tile, or with one counted twice, is outside its tolerance for every tile."""
from __future__ import annotations

import numpy as np
import pytest

import kv4_tiles
import oracle


@pytest.mark.parametrize("kind,eps", [("f16", 2.0 ** -10), ("bf16", 2.0 ** -7)])
@pytest.mark.parametrize("n,first", [(9000, 0), (140 * 128 + 77, 0), (140 * 128 + 77, 128)])
def test_a_lost_or_doubled_tile_shows(kind, eps, n, first):
    rng = np.random.default_rng(n + first)
    q, k = rng.standard_normal((2, 128)), rng.standard_normal((n, 128)) * 0.1
    v = kv4_tiles.signature(n, first)
    c, s, z = oracle.kv4_quantize(v.astype(np.float32), kind)
    stored = (s[..., None] * c + z[..., None]).reshape(n, 128)
    s8 = np.repeat(8 * s.astype(np.float64), 32, axis=-1)
    want, eight = kv4_tiles.attention(q, k, stored, s8)
    tol = kv4_tiles.tolerance(want, eight, eps)
    last = min(first + 128, kv4_tiles.tiles(n))
    assert last > first
    for t in range(first, last):
        for kw in (dict(drop=t), dict(double=t)):
            got, _ = kv4_tiles.attention(q, k, stored, s8, **kw)
            # outside by four times over in its own channel
            assert np.all(np.abs(got - want)[:, t - first] > 4 * tol[:, t - first]), (t, kw)
