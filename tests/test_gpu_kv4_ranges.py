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


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("ratio", [2.0 ** -4, 2.0 ** -8, 2.0 ** -12, 2.0 ** -16])
@pytest.mark.parametrize("top", [0, 2])
def test_groups_of_different_scales(dt, ratio, top):
    """Three groups' values are `ratio` of the other's, and one key outweighs the rest: a
    group keeps its own accuracy. Many tokens read one sequence, so that a CTA goes through all
    of it. Per group, with 8192 keys of weight p and scale s: the output's rounding;
    P s in fp16, 2^-11 of p * 8 s; the exponent and the sums in fp32, 2^-12 of p (|z| + 8 s)."""
    import oracle
    from parallel_serve_b200 import KV4Pool, ops
    n, nh, M = 8192, 4, 450
    amp = torch.full((4, 32), ratio * 256.0)
    amp[top] = 256.0
    amp = amp.flatten()
    assert dt != torch.float16 or ratio * 256 / 32 >= 2.0 ** -14     # scales are normal numbers
    k = cpu_randn((n, 1, 128), 95, 0.05, torch.float32)
    v = cpu_randn((n, 1, 128), 96, 1.0, torch.float32) * amp
    q = cpu_randn((1, nh, 128), 97, 1.0, torch.float32)
    # one early key whose score is some 9 (2^13) above the others', for every head
    q[..., 0] = 8.0
    k[33, 0, 0] = 9.0 / 8.0 * 128 ** 0.5
    k, v, q = k.to(dt), v.to(dt), q.to(dt)
    pools = (KV4Pool.zeros(1, 1, n, dt, DEV), None)
    ops.kv4_append(k.to(DEV), v.to(DEV), pools, torch.arange(n, dtype=torch.int32, device=DEV),
                   rows=torch.zeros(n, dtype=torch.int32, device=DEV))
    out = ops.kv4_decode_attention(q.to(DEV).expand(M, nh, 128).contiguous(), pools,
                                   torch.full((M,), n - 1, dtype=torch.int32, device=DEV), max_len=n,
                                   rows=torch.zeros(M, dtype=torch.int32, device=DEV))
    ks, vs = (_stored(pools, None, [n], 1, 0, part)[0] for part in "kv")
    want, _ = oracle.grouped_attention(to_np(q), ks, vs)
    meta = np.repeat(to_np(pools[0].v_meta)[0, 0], 32, axis=1)        # [n, 128, (s, z)]
    s8, z = 8 * meta[..., 0], np.abs(meta[..., 1])
    eight, _ = oracle.grouped_attention(to_np(q), ks, s8[:, None])    # sum of p * 8 s
    both, _ = oracle.grouped_attention(to_np(q), ks, (s8 + z)[:, None])
    tol = torch.finfo(dt).eps / 2 * np.abs(want) + 2.0 ** -11 * eight + 2.0 ** -12 * both
    err = np.abs(to_np(out).reshape(M, nh, 128) - want)
    assert np.all(err <= tol), float((err / tol).max())
    assert _status() == 0
