"""The 4-bit KV cache on the GPU: write (with head norms and rotation), read-back
and decode attention, against the oracle's 64-bit arithmetic.

Tolerances come from the arithmetic. T is the 16-bit type, eps = finfo(T).eps:
* q and k in 16 bits: one rounding, eps/2 of the value, plus fp32's error of a
  few 2^-24 of the row's largest value (2^-18 is allowed).
* codes from 16-bit inputs: equal bit for bit (the format is defined in fp32).
* attention: the output's rounding, eps/2 |o|; P s rounded to fp16, 2^-11 of each
  term s c <= |v| + |z|; the exponent's fp32 error, |log2 p| <= 64 at 2^-24 with a
  few operations, below 2^-14. Together eps/2 |o| + 2^-10 sum p (|v| + max|z|).
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import cpu_randn, to_np

pytestmark = pytest.mark.gpu
DEV = "cuda"
KIND = {torch.float16: "f16", torch.bfloat16: "bf16"}
DTYPES = [torch.float16, torch.bfloat16]


def _tables(n, rotary):
    from parallel_serve_b200 import ops
    return ops.rope_tables(n, rotary, device=DEV)


def _weights(seed, dt):
    return (1 + cpu_randn((2, 128), seed, 0.2, torch.float32)).to(dt)


def _status():
    from parallel_serve_b200 import _lib
    return _lib.read_status(torch.device(DEV, 0))


def _assert16(got, want, dt, scale=None):
    got, eps = to_np(got), torch.finfo(dt).eps
    top = np.abs(want).max(-1, keepdims=True) if scale is None else scale
    assert np.all(np.abs(got - want) <= eps / 2 * np.abs(want) + 2.0 ** -18 * top)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,nh,nkv", [(1, 1, 1), (3, 4, 2), (7, 32, 8), (65, 40, 40), (2, 5, 5)])
@pytest.mark.parametrize("rotary,inter,norm", [(128, False, True), (128, True, True),
                                               (64, False, False), (96, False, True),
                                               (16, True, False), (0, False, True)])
def test_qk_norm_rope(dt, M, nh, nkv, rotary, inter, norm):
    import oracle
    from parallel_serve_b200 import ops
    qkv = cpu_randn((M, nh + 2 * nkv, 128), M + nh, 1.5, dt)
    pos = torch.randint(0, 500, (M,), generator=torch.Generator().manual_seed(M)).int()
    c0 = M // 2
    wq, wk = (_weights(1, dt), _weights(2, dt)) if norm else (None, None)
    cos, sin = _tables(500, rotary) if rotary else (None, None)
    d = qkv.to(DEV)
    q, k = ops.qk_norm_rope(d[:, :nh], d[:, nh:nh + nkv], pos.to(DEV),
                            q_weight=None if wq is None else wq.to(DEV),
                            k_weight=None if wk is None else wk.to(DEV), eps=1e-5, rope_cos=cos,
                            rope_sin=sin, interleaved=inter, split_point=c0)
    model = (np.arange(M) >= c0).astype(int)
    x = to_np(qkv)
    c, s = (None, None) if cos is None else (to_np(cos), to_np(sin))
    for got, rows, w in ((q, x[:, :nh], wq), (k, x[:, nh:nh + nkv], wk)):
        want = oracle.norm_rope(rows, None if w is None else to_np(w)[model], 1e-5, c, s,
                                pos.numpy(), inter)
        _assert16(got, want, dt)
    assert _status() == 0


def test_qk_norm_rope_in_place_counts_and_zero_tokens():
    from parallel_serve_b200 import ops
    M, nh, nkv, dt = 9, 8, 2, torch.bfloat16
    qkv = cpu_randn((M, nh + 2 * nkv, 128), 5, 1.0, dt).to(DEV)
    pos = torch.arange(M, dtype=torch.int32, device=DEV)
    w = _weights(3, dt).to(DEV)
    cos, sin = _tables(16, 128)
    kw = dict(q_weight=w, k_weight=w, rope_cos=cos, rope_sin=sin)
    q, k = ops.qk_norm_rope(qkv[:, :nh], qkv[:, nh:nh + nkv], pos, split_point=4, **kw)
    buf = qkv.clone()
    counts = torch.tensor([4, 5], dtype=torch.int32, device=DEV)
    a, b = buf[:, :nh], buf[:, nh:nh + nkv]
    ops.qk_norm_rope(a, b, pos, counts=counts, q_out=a, k_out=b, **kw)
    assert torch.equal(a, q) and torch.equal(b, k) and torch.equal(buf[:, nh + nkv:], qkv[:, nh + nkv:])
    q0, k0 = ops.qk_norm_rope(qkv[:0, :nh], qkv[:0, nh:nh + nkv], pos[:0], **kw)
    assert q0.shape == (0, nh, 128) and k0.shape == (0, nkv, 128)
    # a position outside the tables: flagged, its rows untouched, the others written
    bad = pos.clone()
    bad[3] = 16
    bad[7] = -1
    qo, ko = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    ops.qk_norm_rope(qkv[:, :nh], qkv[:, nh:nh + nkv], bad, split_point=4, q_out=qo, k_out=ko, **kw)
    assert _status() == 4
    for got, want in ((qo, q), (ko, k)):
        assert (got[[3, 7]] == 7).all()
        keep = [0, 1, 2, 4, 5, 6, 8]
        assert torch.equal(got[keep], want[keep])


def _pools(lens0, lens1, nkv, dt, page, cap, seed=0):
    """Empty pools for two models (None without sequences) and the block table."""
    from parallel_serve_b200 import KV4Pool
    n = (len(lens0), len(lens1))
    if not page:
        return tuple(KV4Pool.zeros(k, nkv, cap, dt, DEV) if k else None for k in n), None
    per = -(-cap // page)
    table = torch.full((sum(n), per), -1, dtype=torch.int32)
    pools, base = [], 0
    g = torch.Generator().manual_seed(seed)
    for m, lens in enumerate((lens0, lens1)):
        need = [-(-x // page) for x in lens]
        ids = torch.randperm(sum(need), generator=g).int()
        at = 0
        for i, k in enumerate(need):
            table[base + i, :k] = ids[at:at + k]
            at += k
        base += len(lens)
        pools.append(KV4Pool.zeros(at, nkv, page, dt, DEV) if at else None)
    return tuple(pools), table.to(DEV)


def _filled(lens, n0, nkv, dt, page, cap, seed, scale=1.0, offset=0.0):
    """Pools holding random sequences, written through kv4_append, and the stored
    values [len, nkv, 128] of every sequence."""
    from parallel_serve_b200 import ops
    pools, table = _pools(lens[:n0], lens[n0:], nkv, dt, page, cap, seed)
    T = sum(lens)
    k = (cpu_randn((T, nkv, 128), seed, scale, torch.float32) + offset).to(dt).to(DEV)
    v = (cpu_randn((T, nkv, 128), seed + 1, scale, torch.float32) - offset).to(dt).to(DEV)
    pos = torch.cat([torch.arange(x) for x in lens]).int().to(DEV)
    home = torch.cat([torch.full((x,), i if table is not None or i < n0 else i - n0)
                      for i, x in enumerate(lens)]).int().to(DEV)
    ops.kv4_append(k, v, pools, pos, rows=home, block_table=table, split_point=sum(lens[:n0]))
    return pools, table, k, v, pos, home


def _stored(pools, table, lens, n0, page, part):
    import oracle
    out = []
    for i, n in enumerate(lens):
        p = pools[0 if i < n0 else 1]
        codes, meta = (p.k_codes, p.k_meta) if part == "k" else (p.v_codes, p.v_meta)
        if table is None:
            s = i if i < n0 else i - n0
            codes, meta = codes[s, :, :n], meta[s, :, :n]
        else:
            t = table[i, :-(-n // page)].long()
            codes, meta = (x[t].transpose(0, 1).flatten(1, 2)[:, :n] for x in (codes, meta))
        out.append(oracle.kv4_unpack(codes.cpu().numpy(), to_np(meta)).swapaxes(0, 1))
    return out


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("page", [0, 8, 64])
@pytest.mark.parametrize("nkv,scale,offset", [(1, 1.0, 0.0), (3, 1e-3, 0.0), (8, 300.0, 5000.0)])
def test_append_stores_the_format_bit_for_bit(dt, page, nkv, scale, offset):
    import oracle
    lens, n0, cap = [1, 17, 40, 9], 2, 48
    pools, table, k, v, pos, home = _filled(lens, n0, nkv, dt, page, cap, 11, scale, offset)
    base = 0
    for i, n in enumerate(lens):
        p = pools[0 if i < n0 else 1]
        for part, x in (("k", k), ("v", v)):
            c, s, z = oracle.kv4_quantize(to_np(x[base:base + n]).astype(np.float32), KIND[dt])
            codes, meta = (p.k_codes, p.k_meta) if part == "k" else (p.v_codes, p.v_meta)
            if page:
                t = table[i].long()
                at = torch.arange(n, device=DEV)
                codes, meta = (y[t[at // page], :, at % page] for y in (codes, meta))
            else:
                sl = i if i < n0 else i - n0
                codes, meta = (y[sl, :, :n].transpose(0, 1) for y in (codes, meta))
            assert np.array_equal(codes.cpu().numpy(), oracle.kv4_pack(c))
            assert np.array_equal(to_np(meta), np.stack([s, z], -1).astype(np.float64))
        base += n
    assert _status() == 0


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("page", [0, 16])
def test_append_with_norm_and_rotation(dt, page):
    """k is quantised from the fp32 result: its read-back is within half a step
    (plus the grid's own rounding: z by eps/2, 15 s by eps/2 of itself) of the
    64-bit value, and q is the same as without a cache."""
    import oracle
    from parallel_serve_b200 import ops
    lens, n0, nh, nkv, cap = [5, 33, 2], 1, 8, 4, 40
    T = sum(lens)
    pools, table = _pools(lens[:n0], lens[n0:], nkv, dt, page, cap)
    qkv = cpu_randn((T, nh + 2 * nkv, 128), 21, 1.0, dt)
    pos = torch.cat([torch.arange(x) for x in lens]).int()
    home = torch.cat([torch.full((x,), i if page or i < n0 else i - n0)
                      for i, x in enumerate(lens)]).int()
    wq, wk = _weights(4, dt), _weights(5, dt)
    cos, sin = _tables(cap, 128)
    d = qkv.to(DEV)
    kw = dict(q_weight=wq.to(DEV), k_weight=wk.to(DEV), rope_cos=cos, rope_sin=sin,
              split_point=sum(lens[:n0]))
    q = ops.kv4_append(d[:, nh:nh + nkv], d[:, nh + nkv:], pools, pos.to(DEV), q=d[:, :nh],
                       rows=home.to(DEV), block_table=table, **kw)
    q2, _ = ops.qk_norm_rope(d[:, :nh], d[:, nh:nh + nkv], pos.to(DEV), **kw)
    assert torch.equal(q, q2)
    model = (np.arange(T) >= sum(lens[:n0])).astype(int)
    x = to_np(qkv)
    want = oracle.norm_rope(x[:, nh:nh + nkv], to_np(wk)[model], 1e-6, to_np(cos), to_np(sin),
                            pos.numpy())
    seqs = torch.tensor([[0 if i < n0 else 1, i if page or i < n0 else i - n0, 0]
                         for i in range(len(lens))], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=DEV)
    k, v = ops.kv4_gather(pools, seqs, cu, T, block_table=table)
    eps = torch.finfo(dt).eps
    for got, ref in ((k, want), (v, x[:, nh + nkv:])):
        g = ref.reshape(T, nkv, 4, 32)
        lo, hi = g.min(-1, keepdims=True), g.max(-1, keepdims=True)
        bound = (hi - lo) / 30 * (1 + 16 * eps) + eps * (np.abs(lo) + (hi - lo)) + eps / 2 * np.abs(g) + 1e-6
        assert np.all(np.abs(to_np(got).reshape(g.shape) - g) <= bound)
    for part, got in (("k", k), ("v", v)):
        _assert16(got, np.concatenate(_stored(pools, table, lens, n0, page, part)), dt)
    assert _status() == 0


ROTATIONS = [(128, False), (128, True), (64, False), (96, False), (48, True), (0, False)]


@pytest.mark.parametrize("rotary,inter", ROTATIONS)
@pytest.mark.parametrize("nh,nkv", [(1, 1), (40, 8), (13, 13), (96, 32)])
def test_many_tokens_are_as_few(rotary, inter, nh, nkv):
    """Rows do not depend on how many tokens a call has, nor on being done in place."""
    from parallel_serve_b200 import ops
    dt, M, c0 = torch.float16, 701, 300
    x = cpu_randn((M, nh + nkv, 128), nh + rotary, 1.0, dt).to(DEV)
    pos = torch.randint(0, 900, (M,), generator=torch.Generator().manual_seed(9)).int().to(DEV)
    kw = dict(q_weight=_weights(6, dt).to(DEV), k_weight=_weights(7, dt).to(DEV), interleaved=inter)
    if rotary:
        kw["rope_cos"], kw["rope_sin"] = _tables(900, rotary)
    q, k = ops.qk_norm_rope(x[:, :nh], x[:, nh:], pos, split_point=c0, **kw)
    for a in range(0, M, 67):
        b = min(M, a + 67)
        qs, ks = ops.qk_norm_rope(x[a:b, :nh], x[a:b, nh:], pos[a:b],
                                  split_point=min(max(c0 - a, 0), b - a), **kw)
        assert torch.equal(qs, q[a:b]) and torch.equal(ks, k[a:b])
    ops.qk_norm_rope(x[:, :nh], x[:, nh:], pos, split_point=c0, q_out=x[:, :nh], k_out=x[:, nh:], **kw)
    assert torch.equal(x[:, :nh], q) and torch.equal(x[:, nh:], k) and _status() == 0


@pytest.mark.parametrize("M", [5, 700])
@pytest.mark.parametrize("shift,extra", [(8, 0), (0, 8), (8, 8), (16, 16)])
def test_output_rows_of_any_alignment(M, shift, extra):
    """Rows at 16-byte and at 32-byte boundaries give the same, and nothing beside them is written."""
    from parallel_serve_b200 import ops
    dt, nh, nkv = torch.bfloat16, 6, 3
    x = cpu_randn((M, nh + nkv, 128), 77, 1.0, dt).to(DEV)
    pos = torch.arange(M, dtype=torch.int32, device=DEV)
    cos, sin = _tables(M, 128)
    want = ops.qk_norm_rope(x[:, :nh], x[:, nh:], pos, rope_cos=cos, rope_sin=sin)
    bufs, outs = [], []
    for h in (nh, nkv):
        stride = h * 128 + extra
        bufs.append(torch.full((shift + M * stride + 64,), 9.0, dtype=dt, device=DEV))
        outs.append(bufs[-1].as_strided((M, h, 128), (stride, 128, 1), shift))
    ops.qk_norm_rope(x[:, :nh], x[:, nh:], pos, rope_cos=cos, rope_sin=sin, q_out=outs[0],
                     k_out=outs[1])
    for buf, out, w in zip(bufs, outs, want):
        assert torch.equal(out, w)
        out.fill_(9.0)
        assert (buf == 9).all()
    assert _status() == 0


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("page", [0, 8])
@pytest.mark.parametrize("nh,nkv,rotary,inter", [(0, 1, 0, False), (5, 5, 96, False), (40, 8, 128, False),
                                                 (32, 32, 64, True)])
def test_a_long_append_is_as_short_ones(dt, page, nh, nkv, rotary, inter):
    from parallel_serve_b200 import ops
    lens, n0, cap = [400, 300, 29], 2, 400
    T = sum(lens)
    x = cpu_randn((T, nh + 2 * nkv, 128), T + nh, 1.0, dt).to(DEV)
    pos = torch.cat([torch.arange(n) for n in lens]).int().to(DEV)
    home = torch.cat([torch.full((n,), i if page or i < n0 else i - n0)
                      for i, n in enumerate(lens)]).int().to(DEV)
    kw = dict(k_weight=_weights(8, dt).to(DEV), interleaved=inter)
    if rotary:
        kw["rope_cos"], kw["rope_sin"] = _tables(cap, rotary)
    split = sum(lens[:n0])
    got = []
    for step in (T, 41):
        pools, table = _pools(lens[:n0], lens[n0:], nkv, dt, page, cap)
        qs = []
        for a in range(0, T, step):
            b = min(T, a + step)
            qs.append(ops.kv4_append(x[a:b, nh:nh + nkv], x[a:b, nh + nkv:], pools, pos[a:b],
                                     q=x[a:b, :nh] if nh else None, rows=home[a:b], block_table=table,
                                     split_point=min(max(split - a, 0), b - a), **kw))
        got.append((pools, torch.cat(qs) if nh else None))
    for one, many in zip(*(g[0] for g in got)):
        for a, b in zip(one, many):
            assert torch.equal(a, b)
    assert nh == 0 or torch.equal(got[0][1], got[1][1])
    assert _status() == 0


def test_gather_windows_and_untouched_rows():
    from parallel_serve_b200 import ops
    dt, lens, n0, nkv = torch.float16, [30, 12, 50], 2, 2
    for page in (0, 16):
        pools, table, k, v, _, _ = _filled(lens, n0, nkv, dt, page, 64, 3)
        full_k = torch.from_numpy(np.concatenate(_stored(pools, table, lens, n0, page, "k")))
        # windows: positions 7..29 of sequence 0, none of sequence 1, 40..49 of sequence 2
        seqs = torch.tensor([[0, 0, 7], [0, 1, 3], [1, 2 if page else 0, 40]], dtype=torch.int32,
                            device=DEV)
        cu = torch.tensor([0, 23, 23, 33], dtype=torch.int32, device=DEV)
        out = tuple(torch.full((40, nkv, 128), 9.0, dtype=dt, device=DEV) for _ in range(2))
        ops.kv4_gather(pools, seqs, cu, 40, block_table=table, out=out)
        want = torch.cat([full_k[7:30], full_k[42 + 40:42 + 50]]).to(dt)
        assert torch.equal(out[0][:33].cpu(), want)
        assert (out[0][33:] == 9).all() and (out[1][33:] == 9).all()
        assert _status() == 0
        # out of range: beyond the capacity, an unknown slot, a bad model
        seqs = torch.tensor([[0, 0, 60], [0, 9, 0], [2, 0, 0], [1, 2 if page else 0, 0]],
                            dtype=torch.int32, device=DEV)
        cu = torch.tensor([0, 10, 12, 14, 20], dtype=torch.int32, device=DEV)
        out[0].fill_(9.0)
        ops.kv4_gather(pools, seqs, cu, 40, block_table=table, out=out)
        assert _status() == 4
        assert (out[0][10:14] == 9).all() and torch.equal(out[0][14:20].cpu(), full_k[42:48].to(dt))


@pytest.mark.parametrize("dt", DTYPES)
def test_special_values(dt):
    """Constant groups, huge values, NaN and infinities in a group."""
    from parallel_serve_b200 import KV4Pool, ops
    x = torch.zeros(1, 1, 128, dtype=dt)
    x[0, 0, :32] = 2.5
    top = torch.finfo(dt).max
    x[0, 0, 32:48], x[0, 0, 48:64] = top, -top
    x[0, 0, 64:96] = torch.arange(32).to(dt)
    x[0, 0, 70] = float("inf")
    x[0, 0, 96:128] = torch.arange(32).to(dt)
    x[0, 0, 100] = float("nan")
    pool = KV4Pool.zeros(1, 1, 8, dt, DEV)
    pos = torch.tensor([3], dtype=torch.int32, device=DEV)
    ops.kv4_append(x.to(DEV), x.to(DEV), (pool, None), pos)
    seqs = torch.tensor([[0, 0, 3]], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    for y in ops.kv4_gather((pool, None), seqs, cu, 1):
        y = y.cpu().float()[0, 0]
        assert (y[:32] == 2.5).all()
        # (max - min) / 15 rounds to 16 bits: 15 s is within eps/2 of the range
        assert torch.allclose(y[32:64], x[0, 0, 32:64].float(), rtol=2 * torch.finfo(dt).eps)
        assert torch.isnan(y[64:]).all()
    assert _status() == 0


def test_append_refuses_bad_indices_on_the_device():
    from parallel_serve_b200 import ops
    dt, nkv = torch.float16, 2
    k = cpu_randn((5, nkv, 128), 1).to(DEV)
    for page in (0, 8):
        pools, table = _pools([16, 16], [16], nkv, dt, page, 16)
        if page:
            table[1, 1] = 99                     # a page that the pool does not have
        before = [t.clone() for p in pools for t in p]
        pos = torch.tensor([16, -1, 9, 3, 2], dtype=torch.int32, device=DEV)
        rows = torch.tensor([0, 0, 1 if page else 7, -1, 50], dtype=torch.int32, device=DEV)
        q = torch.full_like(k, 5.0)
        ops.kv4_append(k, k, pools, pos, q=k, q_out=q, rows=rows, block_table=table)
        assert _status() == 4
        assert (q == 5).all()
        assert all(torch.equal(a, b) for a, b in zip(before, [t for p in pools for t in p]))


def _check_attention(out, q, ks, vs, lens, dt, zmax):
    import oracle
    eps = torch.finfo(dt).eps
    nh = q.shape[1]
    got = to_np(out).reshape(len(lens), nh, 128)
    for j, n in enumerate(lens):
        want, size = oracle.grouped_attention(to_np(q[j:j + 1]), ks[j], vs[j])
        tol = eps / 2 * np.abs(want[0]) + 2.0 ** -10 * (size[0] + zmax)
        assert np.all(np.abs(got[j] - want[0]) <= tol), (j, n, np.abs(got[j] - want[0]).max())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("page", [0, 8, 16, 256])
@pytest.mark.parametrize("nh,nkv", [(1, 1), (8, 2), (5, 1), (8, 8), (12, 1), (32, 2)])
def test_decode_attention(dt, page, nh, nkv):
    from parallel_serve_b200 import ops
    lens, n0, cap = [1, 2, 31, 32, 33, 127, 128, 129, 255, 300, 511], 5, 512
    pools, table, *_ = _filled(lens, n0, nkv, dt, page, cap, 31)
    q = cpu_randn((len(lens), nh, 128), 33, 1.0, dt)
    pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device=DEV)
    out = ops.kv4_decode_attention(q.to(DEV), pools, pos, max_len=cap, block_table=table,
                                   split_point=n0)
    ks = _stored(pools, table, lens, n0, page, "k")
    vs = _stored(pools, table, lens, n0, page, "v")
    assert _status() == 0
    _check_attention(out, q, ks, vs, lens, dt, max(np.abs(x).max() for x in vs))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("lens,n0", [([5000], 1), ([5000], 0), ([3, 9000, 700], 2)])
@pytest.mark.parametrize("scale", [1.0, 2e-3])
def test_decode_attention_split_over_ctas(dt, lens, n0, scale):
    """Long sequences are cut over CTAs; strided q, device counts, slots in another
    order; small scales keep their accuracy."""
    from parallel_serve_b200 import ops
    nh, nkv = 8, 2
    pools, table, *_ = _filled(lens, n0, nkv, dt, 0, 9100, 41, scale, 3 * scale)
    wide = cpu_randn((len(lens), nh + 3, 128), 43, 1.0, dt).to(DEV)
    q = wide[:, 1:1 + nh]
    pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device=DEV)
    counts = torch.tensor([n0, len(lens) - n0], dtype=torch.int32, device=DEV)
    out = ops.kv4_decode_attention(q, pools, pos, max_len=9100, counts=counts)
    ks = _stored(pools, table, lens, n0, 0, "k")
    vs = _stored(pools, table, lens, n0, 0, "v")
    assert _status() == 0
    _check_attention(out, q, ks, vs, lens, dt, max(np.abs(x).max() for x in vs))
    again = ops.kv4_decode_attention(q, pools, pos, max_len=9100, counts=counts)
    assert torch.equal(out, again)               # no dependence on which CTA ends last


def test_decode_attention_many_tokens_and_shared_rows():
    """More tokens than prefix-sum entries; many tokens read one sequence."""
    from parallel_serve_b200 import ops
    dt, nh, nkv, M = torch.bfloat16, 4, 2, 2500
    pools, table, *_ = _filled([200, 50], 1, nkv, dt, 16, 208, 51)
    g = torch.Generator().manual_seed(9)
    n0 = 1300
    pos = torch.cat([torch.randint(0, 200, (n0,), generator=g),
                     torch.randint(0, 50, (M - n0,), generator=g)]).int()
    rows = torch.cat([torch.zeros(n0), torch.ones(M - n0)]).int()
    q = cpu_randn((M, nh, 128), 53, 1.0, dt)
    out = ops.kv4_decode_attention(q.to(DEV), pools, pos.to(DEV), max_len=208, rows=rows.to(DEV),
                                   block_table=table, split_point=n0)
    ks = _stored(pools, table, [200, 50], 1, 16, "k")
    vs = _stored(pools, table, [200, 50], 1, 16, "v")
    pick = list(range(0, M, 37)) + [M - 1]
    lens = [int(pos[j]) + 1 for j in pick]
    _check_attention(out[pick], q[pick], [ks[int(rows[j])][:n] for j, n in zip(pick, lens)],
                     [vs[int(rows[j])][:n] for j, n in zip(pick, lens)], lens, dt,
                     max(np.abs(x).max() for x in vs))
    assert _status() == 0


@pytest.mark.parametrize("page", [0, 16])
def test_stale_rows_and_bad_tokens(page):
    """What lies behind a sequence's last position never counts, NaN and infinity
    included; a token out of range leaves its output as it was."""
    from parallel_serve_b200 import ops
    dt, nh, nkv, lens, n0 = torch.float16, 8, 2, [40, 129, 7, 260], 2
    pools, table, *_ = _filled(lens, n0, nkv, dt, page, 272, 61)
    q = cpu_randn((4, nh, 128), 63, 1.0, dt).to(DEV)
    pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device=DEV)
    kw = dict(max_len=272, block_table=table, split_point=n0)
    want = ops.kv4_decode_attention(q, pools, pos, **kw)
    for i, n in enumerate(lens):
        p = pools[0 if i < n0 else 1]
        for at in range(n, 272):
            row, col = (i if i < n0 else i - n0, at)
            if page:
                row, col = int(table[i, at // page]), at % page
                if row < 0:
                    break
            for meta, codes in ((p.k_meta, p.k_codes), (p.v_meta, p.v_codes)):
                meta[row, :, col, :, 0] = float("inf")
                meta[row, :, col, :, 1] = float("nan")
                codes[row, :, col] = 255
    assert torch.equal(ops.kv4_decode_attention(q, pools, pos, **kw), want)
    assert _status() == 0
    bad = pos.clone()
    bad[0], bad[2] = -1, 272
    out = torch.full_like(want, 3.0)
    ops.kv4_decode_attention(q, pools, bad, out=out, **kw)
    assert _status() == 4
    assert (out[[0, 2]] == 3).all() and torch.equal(out[[1, 3]], want[[1, 3]])
    if page:
        table[3, 1] = 10 ** 6
        out.fill_(3.0)
        ops.kv4_decode_attention(q, pools, pos, out=out, **kw)
        assert _status() == 4
        assert (out[3] == 3).all() and torch.equal(out[:3], want[:3])


def test_nan_in_a_visible_row_shows():
    from parallel_serve_b200 import ops
    dt, nh, nkv, lens = torch.bfloat16, 4, 1, [70, 70, 70]
    pools, table, *_ = _filled(lens, 3, nkv, dt, 0, 128, 71)
    q = cpu_randn((3, nh, 128), 73, 1.0, dt).to(DEV)
    pos = torch.full((3,), 69, dtype=torch.int32, device=DEV)
    want = ops.kv4_decode_attention(q, pools, pos, max_len=128)
    pools[0].k_meta[0, 0, 5, 2] = torch.tensor([0.0, float("nan")])
    pools[0].v_meta[1, 0, 66, 1] = torch.tensor([0.0, float("nan")])
    out = ops.kv4_decode_attention(q, pools, pos, max_len=128).view(3, nh, 128)
    assert torch.isnan(out[0]).all()
    assert torch.isnan(out[1, :, 32:64]).all() and torch.isfinite(out[1, :, :32]).all()
    assert torch.isfinite(out[1, :, 64:]).all()
    assert torch.equal(out[2].flatten(), want[2])


def test_large_and_tiny_queries():
    """q of any exponent, zeros included, keeps its precision."""
    from parallel_serve_b200 import ops
    for dt, f in ((torch.bfloat16, 1e-12), (torch.bfloat16, 1.0), (torch.float16, 20.0),
                  (torch.bfloat16, 0.0)):
        lens, nh, nkv = [150], 3, 1
        pools, table, *_ = _filled(lens, 1, nkv, dt, 0, 150, 81)
        q = (cpu_randn((1, nh, 128), 83, 1.0, torch.float32) * f).to(dt)
        pos = torch.tensor([149], dtype=torch.int32, device=DEV)
        scale = 128 ** -0.5 if f in (0.0, 1.0) else 128 ** -0.5 / f
        out = ops.kv4_decode_attention(q.to(DEV), pools, pos, max_len=150, scale=scale)
        ks = _stored(pools, table, lens, 1, 0, "k")
        vs = _stored(pools, table, lens, 1, 0, "v")
        import oracle
        want, size = oracle.grouped_attention(to_np(q), ks[0], vs[0], scale=scale)
        tol = torch.finfo(dt).eps / 2 * np.abs(want) + 2.0 ** -10 * (size + np.abs(vs[0]).max())
        assert np.all(np.abs(to_np(out).reshape(want.shape) - want) <= tol)


def test_step_in_a_graph_and_on_another_stream():
    """append -> attention as a decode step uses them: captured, replayed with new
    lengths, and eagerly on a side stream, with equal results."""
    from parallel_serve_b200 import ops
    dt, nh, nkv, lens, n0 = torch.bfloat16, 16, 4, [300, 5, 1000, 64], 2
    pools, table, *_ = _filled([n + 2 for n in lens], n0, nkv, dt, 16, 1024, 91)
    qkv = cpu_randn((4, nh + 2 * nkv, 128), 93, 1.0, dt).to(DEV)
    cos, sin = _tables(1024, 128)
    pos = torch.tensor(lens, dtype=torch.int32, device=DEV)

    def step():
        q = ops.kv4_append(qkv[:, nh:nh + nkv], qkv[:, nh + nkv:], pools, pos, q=qkv[:, :nh],
                           rope_cos=cos, rope_sin=sin, block_table=table, split_point=n0)
        return ops.kv4_decode_attention(q, pools, pos, max_len=1024, block_table=table,
                                        split_point=n0)
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    pos.add_(1)
    want1 = step()
    got.zero_()
    for _ in range(3):
        graph.replay()
    assert torch.equal(got, want1)
    pos.sub_(1)
    graph.replay()
    assert torch.equal(got, want)
    assert _status() == 0


def test_two_streams_and_two_graphs_at_once():
    """Calls that overlap have workspaces of their own: long sequences, whose pieces
    several CTAs join, on two streams and in two graphs replayed side by side."""
    from parallel_serve_b200 import ops
    dt, nkv, nh, cap = torch.float16, 2, 8, 8192
    sides, todo = [torch.cuda.Stream() for _ in range(2)], []
    for i, (lens, page) in enumerate((([8000, 3, 5000], 16), ([7000], 0))):
        pools, table, _, _, _, _ = _filled(lens, 1, nkv, dt, page, cap, 51 + i)
        pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device=DEV)
        q = cpu_randn((len(lens), nh, 128), 61 + i, 1.0, dt).to(DEV)

        def call(q=q, pools=pools, pos=pos, table=table):
            return ops.kv4_decode_attention(q, pools, pos, max_len=cap, block_table=table,
                                            split_point=1)
        todo.append((call, call()))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(sides):
            with torch.cuda.stream(s):
                outs[i].append(todo[i][0]())
    torch.cuda.synchronize()
    graphs = []
    for call, _ in todo:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for _ in range(20):
        for (g, _), s in zip(graphs, sides):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for i, (_, want) in enumerate(todo):
        assert all(torch.equal(o, want) for o in outs[i]) and torch.equal(graphs[i][1], want)
    assert _status() == 0


def test_registered_operators_run_together():
    """norm + rotation, cache write, decode and prompt attention through torch.ops: what
    a prompt and the step after it do."""
    from parallel_serve_b200 import KV4Pool, ops
    P = torch.ops.parallel_serve
    dt, nh, nkv, T = torch.bfloat16, 8, 2, 37
    qkv = cpu_randn((T, nh + 2 * nkv, 128), 101, 1.0, dt).to(DEV)
    w = _weights(6, dt).to(DEV)
    cos, sin = _tables(64, 128)
    pos = torch.arange(T, dtype=torch.int32, device=DEV)
    counts = torch.tensor([T, 0], dtype=torch.int32, device=DEV)
    q, k = P.qk_norm_rope(qkv[:, :nh], qkv[:, nh:nh + nkv], pos, w, w, cos, sin, counts, 1e-6, False)
    v = qkv[:, nh + nkv:]
    pool = KV4Pool.zeros(1, nkv, 64, dt, DEV)
    rows = torch.zeros(T, dtype=torch.int32, device=DEV)
    P.kv4_append(k, v, list(pool), [], pos, counts, rows, None)
    cu = torch.tensor([0, T], dtype=torch.int32, device=DEV)
    seqs = torch.zeros(1, 3, dtype=torch.int32, device=DEV)
    k4, v4 = ops.kv4_gather((pool, None), seqs, cu, T)
    prompt = P.prompt_attention(q, k4, v4, cu, cu)
    step = P.kv4_decode_attention(q, list(pool), [], pos, counts, 64, rows, None)
    # the same attention twice: over the read-back rows on the tensor core, over the
    # codes row by row. They differ by their own roundings (eps/2 of P and of the
    # output, and the read-back's eps/2 of k and v; scores here stay below 2^4).
    eps = torch.finfo(dt).eps
    _, size = __import__("oracle").grouped_attention(to_np(q), to_np(k4), to_np(v4))
    err = np.abs(to_np(prompt) - to_np(step)).reshape(size.shape)
    assert np.all(err <= eps * np.abs(to_np(step)).reshape(size.shape) + (2 + 2 ** 4) * eps * size)
    assert _status() == 0


def test_wrappers_refuse():
    from parallel_serve_b200 import KV4Pool, ops
    dt = torch.float16
    q = torch.zeros(2, 4, 128, dtype=dt, device=DEV)
    k = torch.zeros(2, 2, 128, dtype=dt, device=DEV)
    i = torch.zeros(2, dtype=torch.int32, device=DEV)
    pool = KV4Pool.zeros(2, 2, 16, dt, DEV)
    cos, sin = _tables(16, 128)
    tab = torch.zeros(2, 1, dtype=torch.int32, device=DEV)
    seqs = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    for call in (
            lambda: ops.qk_norm_rope(q, k[:1], i),
            lambda: ops.qk_norm_rope(q[..., :64], k, i),
            lambda: ops.qk_norm_rope(q.transpose(0, 1), k, i),
            lambda: ops.qk_norm_rope(q, k.bfloat16(), i),
            lambda: ops.qk_norm_rope(q, k, i.long()),
            lambda: ops.qk_norm_rope(q, k, i[:1]),
            lambda: ops.qk_norm_rope(q, k, i, rope_cos=cos),
            lambda: ops.qk_norm_rope(q, k, i, rope_cos=cos[:, :5], rope_sin=sin[:, :5]),
            lambda: ops.qk_norm_rope(q, k, i, q_weight=torch.ones(128, dtype=dt, device=DEV)),
            lambda: ops.qk_norm_rope(q, k, i, split_point=3),
            lambda: ops.qk_norm_rope(q, k, i, q_out=k),
            lambda: ops.kv4_append(k, k, (None, None), i),
            lambda: ops.kv4_append(k, k, (pool,), i),
            lambda: ops.kv4_append(k[:, :1], k[:, :1], (pool, None), i),
            lambda: ops.kv4_append(k, k[:1], (pool, None), i),
            lambda: ops.kv4_append(k.bfloat16(), k.bfloat16(), (pool, None), i),
            lambda: ops.kv4_append(k, k, (pool, KV4Pool.zeros(2, 2, 8, dt, DEV)), i),
            lambda: ops.kv4_append(k, k, (pool, None), i, q_out=q),
            lambda: ops.kv4_append(k, k, (pool, None), i, rows=i[:1]),
            lambda: ops.kv4_append(k, k, (pool, None), i, block_table=tab[:1]),
            lambda: ops.kv4_append(k, k, (pool, None), i, block_table=i),
            lambda: ops.kv4_append(k, k, (KV4Pool.zeros(2, 2, 12, dt, DEV), None), i, block_table=tab),
            lambda: ops.kv4_append(k, k, (KV4Pool(pool[0], pool[1], pool[2], pool[3][..., :1]), None), i),
            lambda: ops.kv4_gather((pool, None), seqs[:, :2], cu, 2),
            lambda: ops.kv4_gather((pool, None), seqs, cu[:2], 2),
            lambda: ops.kv4_gather((pool, None), seqs, cu, -1),
            lambda: ops.kv4_gather((pool, None), seqs, cu, 2, out=(k, q)),
            lambda: ops.kv4_decode_attention(q[:, :3], (pool, None), i, max_len=16),
            lambda: ops.kv4_decode_attention(q, (pool, None), i, max_len=17),
            lambda: ops.kv4_decode_attention(q, (pool, None), i, max_len=0),
            lambda: ops.kv4_decode_attention(q, (pool, None), i, max_len=16, out=q),
            lambda: ops.kv4_decode_attention(q, (pool, None), i.cpu(), max_len=16),
            lambda: ops.prompt_attention(q, k, k[:1], cu),
            lambda: ops.prompt_attention(q[:, :3], k, k, cu),
            lambda: ops.prompt_attention(q, k, k, cu, cu[:2]),
            lambda: ops.prompt_attention(q, k[:1], k[:1], cu),
            lambda: ops.prompt_attention(q, k, k, cu, scale=0.0),
            lambda: ops.prompt_attention(q, k, k, cu, out=k)):
        with pytest.raises((ValueError, TypeError)):
            call()
    from parallel_serve_b200 import _lib
    with pytest.raises(_lib.PSError):
        ops.kv4_decode_attention(q, (pool, None), i, max_len=16,
                                 workspace=torch.zeros(64, dtype=torch.uint8, device=DEV))
    assert _status() == 0
