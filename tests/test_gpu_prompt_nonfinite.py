"""Prompt attention with values that are not finite: one touches its own channel and
the queries that see its key, wherever the key falls among the tiles.

Lengths put every key in a masked block of some queries (the diagonal) and an
unmasked one of others; with long mean lengths a CTA has two tiles of queries,
which share a block that is masked for one of them only.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import cpu_randn, to_np

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float16, torch.bfloat16]
INF, NAN = float("inf"), float("nan")


def _status():
    from parallel_serve_b200 import _lib
    return _lib.read_status(torch.device(DEV, 0))


def _cu(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=DEV)


def _inputs(dt, n, rows, seed):
    """Scores stay within a few units, so that every weight is above fp16's smallest."""
    q = cpu_randn((n, 2, 128), seed, 0.5, dt).to(DEV)
    k = cpu_randn((rows, 1, 128), seed + 1, 0.5, dt).to(DEV)
    v = cpu_randn((rows, 1, 128), seed + 2, 1.0, dt).to(DEV)
    return q, k, v


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows", [400, 4200])       # one tile a CTA, and two
@pytest.mark.parametrize("x,y", [(INF, None), (-INF, None), (NAN, None), (INF, -INF), (INF, INF)])
def test_a_value_touches_its_own_channel(dt, rows, x, y):
    from parallel_serve_b200 import ops
    n = 400
    q, k, v = _inputs(dt, n, rows, 201)
    cu = _cu([n])
    want = ops.prompt_attention(q, k, v, cu, cu).view(n, 2, 128)
    for key in (0, 63, 64, 127, 128, 200, 256, 383, 399):
        for ch in (0, 63, 64, 127):
            bad = v.clone()
            bad[key, 0, ch] = x
            expect = want.clone()
            expect[key:, :, ch] = x
            if y is not None and key >= 5:            # an earlier key of the same channel
                bad[key - 5, 0, ch] = y
                expect[key - 5:, :, ch] = y
                expect[key:, :, ch] = x + y
            out = ops.prompt_attention(q, k, bad, cu, cu).view(n, 2, 128)
            assert torch.equal(torch.nan_to_num(out, 0.0), torch.nan_to_num(expect, 0.0)), (key, ch)
            assert torch.equal(out.isnan(), expect.isnan()), (key, ch)
    assert _status() == 0


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows", [700, 4200])
def test_many_values_and_a_history(dt, rows):
    """Infinities and NaNs scattered over keys and channels, keys before the queries."""
    from parallel_serve_b200 import ops
    n, nk = 300, 437
    q, k, v = _inputs(dt, n, rows, 211)
    cu_q, cu_k = _cu([n]), _cu([nk])
    want = ops.prompt_attention(q, k, v, cu_q, cu_k).view(n, 2, 128)
    g = torch.Generator().manual_seed(5)
    bad, seen = v.clone(), torch.zeros(n, 128)
    first = nk - n                                    # the last key that query 0 sees
    for _ in range(60):
        key, ch = int(torch.randint(0, nk, (1,), generator=g)), int(torch.randint(0, 100, (1,), generator=g))
        x = (INF, -INF, NAN)[int(torch.randint(0, 3, (1,), generator=g))]
        bad[key, 0, ch] = x
    bv = bad[:nk, 0].float().cpu()
    special = torch.where(torch.isfinite(bv), torch.zeros(()), bv)
    for i in range(n):
        seen[i] = special[:first + i + 1].sum(0)      # 0, an infinity or NaN
    # a NaN anywhere in a sum of zeros and infinities is that sum
    expect = torch.where(seen.to(DEV)[:, None] == 0, want.float(), seen.to(DEV)[:, None].expand(n, 2, 128))
    out = ops.prompt_attention(q, k, bad, cu_q, cu_k).view(n, 2, 128).float()
    finite = torch.isfinite(expect)
    assert torch.equal(out[finite], expect[finite])
    assert torch.equal(out.isnan(), expect.isnan())
    assert torch.equal(out[~finite & ~expect.isnan()], expect[~finite & ~expect.isnan()])
    assert _status() == 0
