"""Prompts through the 4-bit cache in chunks of different sizes: the chunk boundary falls inside
a block of 128 keys, and the keys before it come from the cache.

Chunks change the shapes of the products and the attention's tiles, so results are
equal up to rounding, not bit for bit: a rounding of k or v may move a code by one.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import cpu_randn, rel_err, to_np
from test_gpu_kv4 import DEV, DTYPES, _status
from test_gpu_kv4_decoder import FF, H, N_LAYERS, NH, TOL, V, _decoder, _State

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [None, 16])
def test_prompts_in_chunks_of_any_size(page):
    """Every chunk size agrees with the oracle over its own cache. Layer 0 sees the same
    embeddings whatever the chunk: its k and v differ by their 16-bit rounding (one
    last place, so 2 eps of the pair that a rotation mixes) and hence by at most one
    quantisation step plus the rounding of (s, z). The logits differ by no more than the
    oracle's own do between the two caches, plus each side's distance from it."""
    import oracle
    ids, lens, L_cap = [0, 1, 0, 1], [150, 33, 200, 129], 208
    g = torch.Generator().manual_seed(28)
    prompts = [torch.randint(0, V, (n,), generator=g).tolist() for n in lens]
    cos, sin = oracle.rope_tables(L_cap)
    runs = []
    for chunk in (7, 32, 100, 256):
        dec, P = _decoder(ids, L_cap, page, chunk)
        dec.prefill(prompts)
        torch.cuda.synchronize()
        dec.check_status()
        st = _State(dec, max(lens))
        _, logits = oracle.prefill(prompts, np.array(ids), P, st, NH, cos, sin, 1e-5)
        assert rel_err(to_np(dec.logits), logits) < TOL, chunk
        st.check()
        kv = [[to_np(t) for t in dec.read_kv(0, m, max(lens))] for m in range(2)]
        runs.append((chunk, to_np(dec.logits), logits, kv))
    eps = torch.finfo(torch.float16).eps
    for chunk, got, logits, kv in runs[1:]:
        first = runs[0]
        assert rel_err(got, first[1]) <= 2 * TOL + rel_err(logits, first[2]), chunk
        for m in range(2):
            slot_lens = [n for n, i in zip(lens, ids) if i == m]
            for a, b in zip(kv[m], first[3][m]):
                for slot, n in enumerate(slot_lens):
                    x, y = (t[slot, :, :n].reshape(NH, n, 4, 32) for t in (a, b))
                    span = y.max(-1, keepdims=True) - y.min(-1, keepdims=True)
                    # a step of either grid, k's or v's rounding, (s, z) of either
                    top = np.abs(b[slot, :, :n]).max(-1).reshape(NH, n, 1, 1)
                    assert np.all(np.abs(x - y) <= span / 15 * 1.05 + 4 * eps * top), (chunk, m)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("chunk", [7, 32, 100, 256])
def test_attention_in_chunks(dt, chunk):
    """The same keys and values, read back from the cache: queries in chunks, each behind
    the keys before it, against all at once (both within their tolerance of the 64-bit result)."""
    import oracle
    from parallel_serve_b200 import KV4Pool, ops
    n, nh, nkv = 417, 4, 2
    qkv = [cpu_randn((n, h, 128), 141 + i, 1.0, dt).to(DEV) for i, h in enumerate((nh, nkv, nkv))]
    pool = (KV4Pool.zeros(1, nkv, n, dt, DEV), None)
    zeros = torch.zeros(n, dtype=torch.int32, device=DEV)
    ops.kv4_append(qkv[1], qkv[2], pool, torch.arange(n, dtype=torch.int32, device=DEV), rows=zeros)
    parts, q = [], qkv[0]
    for a in range(0, n, chunk):
        b = min(n, a + chunk)
        cu_q, cu_k = (torch.tensor([0, x], dtype=torch.int32, device=DEV) for x in (b - a, b))
        k, v = ops.kv4_gather(pool, torch.zeros(1, 3, dtype=torch.int32, device=DEV), cu_k, b)
        parts.append(ops.prompt_attention(q[a:b], k, v, cu_q, cu_k))
    want, size = oracle.grouped_attention(to_np(q), to_np(k), to_np(v))
    eps = torch.finfo(dt).eps
    tol = eps / 2 * np.abs(want) + (eps / 2 + 2.0 ** -14) * size
    assert np.all(np.abs(to_np(torch.cat(parts)).reshape(want.shape) - want) <= tol)
    assert _status() == 0
