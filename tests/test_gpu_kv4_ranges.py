"""The 4-bit cache and its attention over the whole range of the 16-bit types, against
64-bit arithmetic."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import cpu_randn, to_np
from test_gpu_kv4 import DEV, DTYPES, KIND, _filled, _status, _stored

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("e", [-118, -110, -60, 60, 101, 113, 120, 124])
@pytest.mark.parametrize("nh", [3, 9])
def test_queries_of_every_exponent(e, nh):
    """q times 2^e and the scale by 2^-e: the same scores. Tolerance as for queries around
    1 (2^-10 of the terms for the weights' 16 bits, the output's rounding)."""
    import oracle
    from parallel_serve_b200 import ops
    dt, lens = torch.bfloat16, [150]
    pools, table, *_ = _filled(lens, 1, 1, dt, 0, 150, 81)
    q = (cpu_randn((1, nh, 128), 83, 1.0, torch.float32).to(dt).double() * 2.0 ** e).to(dt)
    assert torch.isfinite(q).all()
    pos = torch.tensor([149], dtype=torch.int32, device=DEV)
    scale = 128 ** -0.5 * 2.0 ** -e
    out = ops.kv4_decode_attention(q.to(DEV), pools, pos, max_len=150, scale=scale)
    ks, vs = (_stored(pools, table, lens, 1, 0, part)[0] for part in "kv")
    want, size = oracle.grouped_attention(to_np(q), ks, vs, scale=scale)
    tol = torch.finfo(dt).eps / 2 * np.abs(want) + 2.0 ** -10 * (size + np.abs(vs).max())
    assert np.all(np.abs(to_np(out).reshape(want.shape) - want) <= tol)
    assert _status() == 0


@pytest.mark.parametrize("e", [-117, -105, -70, 70, 104, 112])
@pytest.mark.parametrize("n", [150, 3000])            # one CTA, and several joined
def test_values_of_every_exponent(e, n):
    """V times 2^e: the output is 2^e of what it was (the sums, at most 2^8 x n of the
    values, stay below fp32's 2^128)."""
    import oracle
    from parallel_serve_b200 import KV4Pool, ops
    dt = torch.bfloat16
    k = cpu_randn((n, 1, 128), 91, 1.0, dt)
    v = (cpu_randn((n, 1, 128), 92, 1.0, torch.float32).double() * 2.0 ** e).to(dt)
    pools = (KV4Pool.zeros(1, 1, n, dt, DEV), None)
    ops.kv4_append(k.to(DEV), v.to(DEV), pools, torch.arange(n, dtype=torch.int32, device=DEV),
                   rows=torch.zeros(n, dtype=torch.int32, device=DEV))
    q = cpu_randn((1, 4, 128), 93, 1.0, dt)
    out = ops.kv4_decode_attention(q.to(DEV), pools, torch.tensor([n - 1], dtype=torch.int32, device=DEV),
                                   max_len=n)
    ks, vs = (_stored(pools, None, [n], 1, 0, part)[0] for part in "kv")
    want, size = oracle.grouped_attention(to_np(q), ks, vs)
    tol = torch.finfo(dt).eps / 2 * np.abs(want) + 2.0 ** -10 * (size + np.abs(vs).max())
    assert np.all(np.abs(to_np(out).reshape(want.shape) - want) <= tol)
    assert _status() == 0
