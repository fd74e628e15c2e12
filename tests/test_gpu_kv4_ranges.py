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


def _codes(x, dt):
    """Codes, scale and zero of a row [128] as kv4_append stores them."""
    import oracle
    from parallel_serve_b200 import KV4Pool, ops
    pool = KV4Pool.zeros(1, 1, 8, dt, DEV)
    x = x.to(dt).view(1, 1, 128).to(DEV)
    ops.kv4_append(x, x, (pool, None), torch.zeros(1, dtype=torch.int32, device=DEV))
    meta = to_np(pool.k_meta)[0, 0, 0]
    ident = np.stack([np.ones(4), np.zeros(4)], -1)                   # s = 1, z = 0: the codes
    c = oracle.kv4_unpack(pool.k_codes.cpu().numpy()[0, 0, 0], ident).reshape(4, 32)
    assert torch.equal(pool.k_codes, pool.v_codes) and torch.equal(pool.k_meta, pool.v_meta)
    return c, meta[:, 0], meta[:, 1]


def _exact(x, dt):
    """The format's definition in 64 bits (the inputs here leave no quotient within 2^-20
    of a half, which the test checks)."""
    g = to_np(x.to(dt)).reshape(4, 32)
    z = to_np(torch.from_numpy(g.min(-1)).to(dt))
    s = to_np(torch.from_numpy((g.max(-1) - z) / 15).to(dt))
    y = (g - z[:, None]) / np.where(s == 0, 1, s)[:, None]
    return np.clip(np.rint(y), 0, 15), s, z, np.abs(y - np.floor(y) - 0.5).min()


def test_groups_wider_than_fp32():
    """bf16 groups whose largest and smallest value are more than fp32's range apart."""
    dt, top = torch.bfloat16, torch.finfo(torch.bfloat16).max
    x = torch.linspace(-1, 1, 32).double().repeat(4, 1) * top
    x[1] *= 0.8
    x[2] = x[2].flip(0) * 0.6
    x[3, 1:] *= 0.01                                   # one value far below the others
    c, s, z = _codes(x, dt)
    want, ws, wz, margin = _exact(x.flatten(), dt)
    assert margin > 2.0 ** -20
    assert np.array_equal(z, wz) and np.array_equal(s, ws) and np.array_equal(c, want)
    assert _status() == 0


@pytest.mark.parametrize("e", [-130, -126, -124, -122, -115, -101, -90])
def test_groups_of_tiny_values(e):
    """bf16 groups whose step is near fp32's smallest normal number: the codes of a
    division, ties included (fp32 holds these quotients' operands exactly)."""
    import oracle
    dt = torch.bfloat16
    g = torch.Generator().manual_seed(3)
    for _ in range(8):
        x = (torch.randn(128, generator=g).to(dt).double() * 2.0 ** e).to(dt)
        c, s, z = _codes(x, dt)
        wc, ws, wz = oracle.kv4_quantize(to_np(x).astype(np.float32), KIND[dt])
        assert np.array_equal(s, ws) and np.array_equal(z, wz) and np.array_equal(c, wc)
        # halves of the step on purpose: 15 steps, then odd multiples of half a step
        step = 2.0 ** e
        y = torch.arange(32).double().repeat(4) * step / 2
        y[31::32] = 15 * step
        c, s, z = _codes(y, dt)
        wc, ws, wz = oracle.kv4_quantize(to_np(y.to(dt)).astype(np.float32), KIND[dt])
        assert np.array_equal(s, ws) and np.array_equal(z, wz) and np.array_equal(c, wc)
    assert _status() == 0


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("scale", [-0.1, 0.0, 3.0])
def test_scales_of_either_sign(dt, scale):
    """Scores reach some 100 at scale 3: |log2 p| <= 256 at 2^-24, 2^-13 of each term in place
    of the 2^-14 of scores around 1."""
    import oracle
    from parallel_serve_b200 import ops
    lens = [300]
    pools, table, *_ = _filled(lens, 1, 1, dt, 0, 300, 85)
    q = cpu_randn((1, 4, 128), 86, 1.0, dt)
    pos = torch.tensor([299], dtype=torch.int32, device=DEV)
    out = ops.kv4_decode_attention(q.to(DEV), pools, pos, max_len=300, scale=scale)
    ks, vs = (_stored(pools, table, lens, 1, 0, part)[0] for part in "kv")
    want, size = oracle.grouped_attention(to_np(q), ks, vs, scale=scale)
    tol = torch.finfo(dt).eps / 2 * np.abs(want) + (2.0 ** -10 + 2.0 ** -13) * (size + np.abs(vs).max())
    assert np.all(np.abs(to_np(out).reshape(want.shape) - want) <= tol)
    for bad in (float("nan"), float("inf"), -2.5e38):
        with pytest.raises(ValueError):
            ops.kv4_decode_attention(q.to(DEV), pools, pos, max_len=300, scale=bad)
    assert _status() == 0
