"""Host side of the 4-bit cache, head norm and prompt attention entry points: what the
C ABI refuses before any CUDA call, the descriptor's layout, the oracle's format, and
the decoder's prefill bookkeeping. No GPU."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from parallel_serve_b200 import _lib, ops

BAD, P = _lib.PS_ERR_INVALID_ARGUMENT, 0x10000            # a non-null, aligned address


def cache(rows=(2, 1), n_kv=2, L_cap=64, table=0, page=0, max_pages=0, table_rows=0, codes=P):
    one = [codes, P, P, P]
    return ops._CACHE.pack(*(one if rows[0] else [0] * 4), rows[0],
                           *(one if rows[1] else [0] * 4), rows[1], table, n_kv, L_cap, page,
                           max_pages, table_rows)


def test_descriptor_matches_the_header(tmp_path):
    import os
    import subprocess

    from conftest import ROOT
    src = tmp_path / "x.c"
    src.write_text('#include "parallel_serve.h"\n#include <stdio.h>\nint main(void) { printf("%zu %zu '
                   '%zu %zu\\n", sizeof(ps_kv4_cache_t), offsetof(ps_kv4_cache_t, pool[1].rows), '
                   'offsetof(ps_kv4_cache_t, block_table), offsetof(ps_kv4_cache_t, table_rows)); }\n')
    exe = tmp_path / "x"
    subprocess.check_call(["gcc", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    size, rows1, table, last = map(int, subprocess.check_output([str(exe)]).split())
    b = ops._CACHE.pack(*[0] * 9, 7, 0x1122, *[0] * 4, 9)
    assert len(b) == size == ops._CACHE.size
    assert b[rows1] == 7 and b[table:table + 2] == b"\x22\x11" and b[last] == 9


def norm_rope(q=P, qs=1024, k=P, ks=256, qo=P, qos=1024, ko=P, kos=256, qw=None, kw=None, rc=P, rs=P,
              n=16, rot=128, pos=P, counts=None, split=0, M=4, nh=8, nkv=2, dt=0):
    return _lib.lib.ps_qk_norm_rope(q, qs, k, ks, qo, qos, ko, kos, qw, kw, 1e-6, rc, rs, n, rot, 0,
                                    pos, counts, split, M, nh, nkv, dt, None, None)


@pytest.mark.parametrize("kw", [dict(M=-1), dict(nkv=0), dict(dt=2), dict(split=5), dict(split=-1),
                                dict(rs=None), dict(rot=24), dict(rot=0), dict(rot=144), dict(n=0),
                                dict(qo=None), dict(q=None), dict(k=None), dict(pos=None),
                                dict(ks=128), dict(ks=260), dict(qs=1016), dict(q=P + 8),
                                dict(qos=1000), dict(ko=None), dict(kos=200), dict(ko=P + 2),
                                dict(nh=0), dict(qw=P + 4), dict(rc=P + 4)])
def test_qk_norm_rope_refuses(kw):
    assert norm_rope(**kw) == BAD


def append(c=None, q=None, qs=0, k=P, ks=256, v=P, vs=256, qo=None, qos=0, pos=P, rows=None, split=0,
           M=4, nh=0, dt=0, rc=None, rs=None):
    return _lib.lib.ps_kv4_append(q, qs, k, ks, v, vs, qo, qos, cache() if c is None else c, None,
                                  None, 1e-6, rc, rs, 16, 128, 0, pos, rows, None, split, M, nh, dt,
                                  None, None)


BAD_CACHES = [dict(n_kv=0), dict(rows=(0, 0)), dict(L_cap=0), dict(codes=0), dict(codes=P + 8),
              dict(rows=(-1, 1)), dict(table=P, page=12, max_pages=4, table_rows=8),
              dict(table=P, page=4, max_pages=4, table_rows=8),
              dict(table=P, page=8192, max_pages=4, table_rows=8),
              dict(table=P, page=16, max_pages=0, table_rows=8),
              dict(table=P, page=16, max_pages=4, table_rows=0),
              dict(table=P, page=4096, max_pages=1 << 19, table_rows=8)]


@pytest.mark.parametrize("c", BAD_CACHES)
def test_every_cache_call_refuses_a_bad_cache(c):
    c = cache(**c)
    assert append(c) == BAD
    assert _lib.lib.ps_kv4_gather(c, P, P, 1, 4, P, P, 0, None, None) == BAD
    assert attend(c) == BAD


@pytest.mark.parametrize("kw", [dict(M=-1), dict(dt=3), dict(v=None), dict(vs=100), dict(v=P + 4),
                                dict(q=P, qs=256, nh=2), dict(qo=P, qos=256), dict(split=9),
                                dict(rc=P), dict(q=P, qs=256, qo=P, qos=256, nh=0)])
def test_append_refuses(kw):
    assert append(**kw) == BAD
    assert append(c=cache(table=P, page=16, max_pages=4, table_rows=3)) == BAD   # a row per token


@pytest.mark.parametrize("kw", [dict(n=-1), dict(total=-1), dict(dt=2), dict(seqs=None), dict(cu=None),
                                dict(k=None), dict(v=P + 8)])
def test_gather_refuses(kw):
    a = dict(seqs=P, cu=P, n=1, total=4, k=P, v=P, dt=0) | kw
    assert _lib.lib.ps_kv4_gather(cache(), a["seqs"], a["cu"], a["n"], a["total"], a["k"], a["v"],
                                  a["dt"], None, None) == BAD


def attend(c=None, q=P, qs=1024, out=P, pos=P, split=0, M=4, nh=8, max_len=64, dt=0):
    return _lib.lib.ps_kv4_decode_attention(q, qs, cache() if c is None else c, out, pos, None, None,
                                            split, M, nh, max_len, 0.1, dt, None, 0, None, None)


@pytest.mark.parametrize("kw", [dict(M=-1), dict(nh=7), dict(nh=0), dict(max_len=0), dict(max_len=65),
                                dict(dt=2), dict(split=5), dict(q=None), dict(out=None), dict(pos=None),
                                dict(qs=1000), dict(qs=1028), dict(q=P + 8)])
def test_decode_attention_refuses(kw):
    assert attend(**kw) == BAD


def prompt(q=P, qs=256, k=P, ks=128, v=P, vs=128, o=P, os=256, cq=P, ck=P, n=1, Tq=8, Tk=8, nh=2, nkv=1,
           scale=0.1, dt=0):
    return _lib.lib.ps_prompt_attention(q, qs, k, ks, v, vs, o, os, cq, ck, n, Tq, Tk, nh, nkv, scale,
                                        dt, None, None)


@pytest.mark.parametrize("kw", [dict(n=-1), dict(Tq=-1), dict(Tk=-1), dict(nh=3, nkv=2), dict(nkv=0),
                                dict(dt=4), dict(scale=0.0), dict(scale=-1.0),
                                dict(scale=float("inf")), dict(scale=float("nan")), dict(q=None),
                                dict(o=None), dict(cq=None), dict(ck=None), dict(k=None),
                                dict(v=None), dict(q=P + 8), dict(v=P + 2), dict(qs=128),
                                dict(os=250), dict(ks=64), dict(vs=132)])
def test_prompt_attention_refuses(kw):
    assert prompt(**kw) == BAD


def test_nothing_to_do_is_no_error():
    assert norm_rope(M=0) == 0 and append(M=0) == 0 and attend(M=0) == 0
    assert prompt(Tq=0) == 0 and prompt(n=0) == 0
    assert _lib.lib.ps_kv4_gather(cache(), P, P, 0, 4, P, P, 0, None, None) == 0
    assert _lib.lib.ps_kv4_decode_attention_workspace_bytes(0, 8, 2, 64) == 0
    assert _lib.lib.ps_kv4_decode_attention_workspace_bytes(4, 7, 2, 64) == 0


def test_wrappers_refuse_host_tensors():
    t, i = torch.zeros(2, 1, 128, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    from parallel_serve_b200 import KV4Pool
    pool = KV4Pool.zeros(2, 1, 8, device="cpu")
    assert KV4Pool.bytes_per_position(32) == 32 * 160
    for call in (lambda: ops.qk_norm_rope(t, t, i), lambda: ops.kv4_append(t, t, (pool, None), i),
                 lambda: ops.kv4_gather((pool, None), i.view(-1)[:0].view(0, 3), i, 0),
                 lambda: ops.kv4_decode_attention(t, (pool, None), i, max_len=8),
                 lambda: ops.prompt_attention(t, t, t, i)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        KV4Pool.zeros(1, 1, 8, torch.float32, "cpu")


def test_oracle_format_round_trip():
    import oracle
    rng = np.random.default_rng(0)
    x = rng.standard_normal((5, 3, 128)).astype(np.float32) * 3 + 1
    for kind, eps in (("f16", 2.0 ** -10), ("bf16", 2.0 ** -7)):
        c, s, z = oracle.kv4_quantize(x, kind)
        v = oracle.kv4_unpack(oracle.kv4_pack(c), np.stack([s, z], -1))
        g, r = x.reshape(5, 3, 4, 32), v.reshape(5, 3, 4, 32)
        bound = s[..., None] / 2 + eps * (np.abs(z)[..., None] + 15 * s[..., None])
        assert np.all(np.abs(r - g) <= bound)


def test_oracle_attention_against_a_softmax():
    import oracle
    rng = np.random.default_rng(1)
    q, k, v = rng.standard_normal((3, 4, 128)), rng.standard_normal((5, 2, 128)), rng.standard_normal((5, 2, 128))
    out, size = oracle.grouped_attention(q, k, v)
    for i in range(3):
        for h in range(4):
            p = np.exp(k[:3 + i, h // 2] @ q[i, h] / np.sqrt(128))
            assert np.allclose(out[i, h], p @ v[:3 + i, h // 2] / p.sum())
    assert np.all(size >= np.abs(out) - 1e-12)
    assert np.all(oracle.grouped_attention(q, k[:1], v[:1])[0][:2] == 0)   # queries without keys


def test_chunk_sequences_of_the_prefill():
    from parallel_serve_b200.decoder import TwoModelDecoder, prefill_layout
    dec = TwoModelDecoder.__new__(TwoModelDecoder)
    dec.device = torch.device("cpu")
    prompts = [list(range(300)), list(range(5)), list(range(130))]
    lens, seen = {0: 300, 1: 5, 2: 130}, {0: 0, 1: 0, 2: 0}
    for ch in prefill_layout(prompts, [0, 2, 1], 2, 200, paged=True):
        seqs, cu_q, cu_k, total = dec._chunk_sequences(ch["qblocks"])
        assert cu_q[0] == 0 and int(cu_q[-1]) == len(ch["tok"]) and int(cu_k[-1]) == total
        for (model, row, first), n, nk in zip(seqs.tolist(), cu_q.diff().tolist(), cu_k.diff().tolist()):
            who = [0, 2, 1][row]
            assert first == 0 and model == (0 if row < 2 else 1)
            seen[who] += n
            assert nk == seen[who]
    assert seen == lens
