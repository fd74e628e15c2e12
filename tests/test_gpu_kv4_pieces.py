"""Decode attention over sequences cut into many pieces: every tile of 128 positions is
checked (``kv4_tiles``), also where one item spans every CTA of the launch."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv4_tiles
from conftest import cpu_randn, to_np
from test_gpu_kv4 import DEV, _pools, _status, _stored

pytestmark = pytest.mark.gpu


def _append(pools, table, lens, n0, k, v):
    from parallel_serve_b200 import ops
    pos = torch.cat([torch.arange(x) for x in lens]).int().to(DEV)
    home = torch.cat([torch.full((x,), i if table is not None or i < n0 else i - n0)
                      for i, x in enumerate(lens)]).int().to(DEV)
    ops.kv4_append(k, v, pools, pos, rows=home, block_table=table, split_point=sum(lens[:n0]))


# One sequence of 444 tiles with one KV head: on 148 SMs a piece for each of 444 CTAs; 300
# tiles with two: 150 pieces of 2 tiles an item. Then ragged batches, items of 1 to 71 tiles.
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page", [0, 16, 64])
@pytest.mark.parametrize("lens,n0,nh,nkv", [([444 * 128 - 5], 1, 8, 1), ([300 * 128], 0, 6, 2),
                                            ([3, 9000, 700], 2, 8, 2), ([5000, 128, 129], 1, 6, 3)])
def test_every_tile_counts_once(dt, page, lens, n0, nh, nkv):
    from parallel_serve_b200 import ops
    T, cap, eps = sum(lens), -(-max(lens) // 64) * 64, torch.finfo(dt).eps
    pools, table = _pools(lens[:n0], lens[n0:], nkv, dt, page, cap)
    k = cpu_randn((T, nkv, 128), 131, 0.1, dt).to(DEV)
    q = cpu_randn((len(lens), nh, 128), 132, 1.0, dt)
    pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device=DEV)
    ks = None
    for first in range(0, kv4_tiles.tiles(max(lens)), 128):
        v = np.concatenate([kv4_tiles.signature(n, first) if first * 128 < n else np.zeros((n, 128))
                            for n in lens])
        v = torch.from_numpy(v).to(dt)[:, None].expand(T, nkv, 128).contiguous().to(DEV)
        _append(pools, table, lens, n0, k, v)
        out = ops.kv4_decode_attention(q.to(DEV), pools, pos, max_len=cap, block_table=table,
                                       split_point=n0)
        again = ops.kv4_decode_attention(q.to(DEV), pools, pos, max_len=cap, block_table=table,
                                         split_point=n0)
        assert torch.equal(out, again)
        ks = ks or _stored(pools, table, lens, n0, page, "k")
        vs = _stored(pools, table, lens, n0, page, "v")
        got, G = to_np(out).reshape(len(lens), nh, 128), nh // nkv
        for j in range(len(lens)):
            for h in range(nkv):
                # z = 0 and codes 0 or 15: the scale is a fifteenth of the group's largest value
                s = vs[j][:, h].reshape(-1, 4, 32).max(-1) / 15
                want, eight = kv4_tiles.attention(to_np(q)[j, h * G:(h + 1) * G], ks[j][:, h], vs[j][:, h],
                                                  np.repeat(8 * s, 32, axis=-1))
                err = np.abs(got[j, h * G:(h + 1) * G] - want)
                assert np.all(err <= kv4_tiles.tolerance(want, eight, eps)), (first, j, h)
    assert _status() == 0


@pytest.mark.parametrize("page", [0, 16, 4096])
def test_rows_beyond_32_bits(page):
    """Pools of 2^27 rows (8 GB of codes each for K and V): the sequence lies at their end."""
    from parallel_serve_b200 import KV4Pool, ops
    dt, n, nh = torch.float16, 3000, 4
    # the pool's address space without 21 GB of it: K and V are the same tensors
    rows = 1 << 27
    shape = (rows // page, 1, page) if page else (64, 1, rows // 64)
    codes = torch.zeros(*shape, 64, dtype=torch.uint8, device=DEV)
    meta = torch.zeros(*shape, 4, 2, dtype=dt, device=DEV)
    pools = (KV4Pool(codes, meta, codes, meta), None)
    x = cpu_randn((n, 1, 128), 151, 1.0, dt).to(DEV)
    last, table = shape[0] - 1, None
    base = 0 if page else shape[2] - n                # contiguous: the slot's last positions
    if page:
        per = -(-n // page)
        table = torch.arange(last, last - per, -1, dtype=torch.int32, device=DEV).view(1, per)
    home = torch.full((n,), 0 if page else last, dtype=torch.int32, device=DEV)
    pos = torch.arange(n, dtype=torch.int32, device=DEV) + base
    ops.kv4_append(x, x, pools, pos, rows=home, block_table=table)
    small = (KV4Pool.zeros(1, 1, n, dt, DEV), None)
    ops.kv4_append(x, x, small, pos - base, rows=torch.zeros_like(home))
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    seqs = torch.tensor([[0, 0 if page else last, base]], dtype=torch.int32, device=DEV)
    got = ops.kv4_gather(pools, seqs, cu, n, block_table=table)
    want = ops.kv4_gather(small, torch.zeros(1, 3, dtype=torch.int32, device=DEV), cu, n)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert int(codes.view(-1, 64)[:1 << 26].count_nonzero()) == 0
    if page:                                          # 2^21 positions of one slot are too many to attend over here
        q = cpu_randn((1, nh, 128), 152, 1.0, dt).to(DEV)
        at = torch.tensor([n - 1], dtype=torch.int32, device=DEV)
        out = ops.kv4_decode_attention(q, pools, at, max_len=n, block_table=table)
        same = ops.kv4_decode_attention(q, small, at, max_len=n)
        # the same pieces of the same values: bit for bit
        assert torch.equal(out, same)
    assert _status() == 0
