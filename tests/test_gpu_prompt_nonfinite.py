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


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n,pad", [(300, 0), (300, 4200)])
@pytest.mark.parametrize("hidden", [40, 128, 130, 200])
def test_scores_of_minus_infinity(dt, n, pad, hidden):
    """Keys whose score is -inf weigh nothing, and the weights of the others do not
    depend on how far below 0 their scores are: the first `hidden` keys are -inf, the rest lie
    at -120 (2^-173 of what a score of 0 would weigh). A query that sees only keys at -inf
    has no softmax (0 / 0): it is not looked at."""
    import oracle
    from parallel_serve_b200 import ops
    q = cpu_randn((n, 1, 128), 221, 0.1, torch.float32)
    k = cpu_randn((n + pad, 1, 128), 222, 0.1, torch.float32)
    v = cpu_randn((n + pad, 1, 128), 223, 1.0, dt)
    q[..., 0], k[..., 0] = 32.0, -3.75                # -120 of every score, scale 1
    q, k = q.to(dt), k.to(dt)
    k[:hidden, 0, 0] = -INF
    cu = _cu([n])
    out = to_np(ops.prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), cu, cu, scale=1.0))
    kf = k.clone()
    kf[:hidden, 0, 0] = -60.0                         # -1920: weighs 0 in 64 bits, too
    want, size = oracle.grouped_attention(to_np(q), to_np(kf[:n]), to_np(v[:n]), scale=1.0)
    # the output's and P's rounding; scores near 120 in fp32: 173 of log2 p at 2^-24, a few
    # operations, and the reference is a product rounded at the same size: 2^-13 of each term
    eps = torch.finfo(dt).eps
    tol = eps / 2 * np.abs(want) + (eps / 2 + 2.0 ** -13) * size
    rows = slice(hidden, n)
    assert np.all(np.abs(out.reshape(want.shape) - want)[rows] <= tol[rows])
    assert _status() == 0
