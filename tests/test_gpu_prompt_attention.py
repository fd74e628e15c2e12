"""Packed causal prompt attention on the GPU against the oracle in 64 bits.

Tolerance: the output's rounding, eps/2 |o|; P rounded to the 16-bit type, eps/2
of each term, so eps/2 sum p |v|; the exponent's fp32 error, |log2 p| <= 64 at
2^-24 with a few operations (2^-15 of each term). Together
eps/2 |o| + (eps/2 + 2^-14) sum p |v|.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import cpu_randn, to_np

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float16, torch.bfloat16]


def _status():
    from parallel_serve_b200 import _lib
    return _lib.read_status(torch.device(DEV, 0))


def _cu(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=DEV)


def _check(out, q, k, v, lens, klens, dt, scale=None, heads=None):
    import oracle
    eps = torch.finfo(dt).eps
    got = to_np(out).reshape(q.shape[0], -1, 128)
    a = b = 0
    G = q.shape[1] // k.shape[1]
    pick = range(q.shape[1]) if heads is None else heads
    for n, nk in zip(lens, klens):
        for h in pick:
            kv = slice(h // G, h // G + 1)
            want, size = oracle.grouped_attention(to_np(q[a:a + n, h:h + 1]),
                                                  to_np(k[b:b + nk, kv]), to_np(v[b:b + nk, kv]),
                                                  scale=scale)
            tol = eps / 2 * np.abs(want) + (eps / 2 + 2.0 ** -14) * size + 1e-30
            err = np.abs(got[a:a + n, h:h + 1] - want)
            assert np.all(err <= tol), (n, nk, h, float((err - tol).max()))
        a, b = a + n, b + nk


def _run(lens, klens, nh, nkv, dt, seed, scale=None, heads=None, amp=1.0):
    from parallel_serve_b200 import ops
    q = cpu_randn((sum(lens), nh, 128), seed, amp, dt)
    k = cpu_randn((sum(klens), nkv, 128), seed + 1, amp, dt)
    v = cpu_randn((sum(klens), nkv, 128), seed + 2, 1.0, dt)
    out = ops.prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), _cu(lens), _cu(klens), scale=scale)
    assert _status() == 0
    _check(out, q, k, v, lens, klens, dt, scale, heads)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("lens", [[1], [2, 1, 1], [127], [128], [129], [256], [257, 3], [300, 0, 513],
                                  [64, 64, 64, 64, 1]])
def test_prompts_alone(dt, lens):
    _run(lens, lens, 2, 1, dt, 100 + sum(lens))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("nh,nkv", [(1, 1), (4, 4), (5, 1), (8, 2)])
def test_histories_and_heads(dt, nh, nkv):
    lens = [5, 130, 1, 260]
    _run(lens, [n + h for n, h in zip(lens, [300, 0, 129, 77])], nh, nkv, dt, 7)


@pytest.mark.parametrize("dt", DTYPES)
def test_long_and_steep(dt):
    _run([1100], [1100], 2, 2, dt, 11, heads=[1])
    # scores far apart: the maximum moves again and again
    _run([700], [900], 2, 1, dt, 13, scale=2.0, amp=2.0)
    _run([40], [40], 2, 1, dt, 17, scale=1e-4)


@pytest.mark.parametrize("dt", DTYPES)
def test_rows_that_see_nothing(dt):
    """Fewer keys than queries: the first queries see none and return 0."""
    _run([300, 20, 7], [10, 20, 0], 2, 1, dt, 23)


def test_strides_and_untouched_rows():
    from parallel_serve_b200 import ops
    dt, nh, nkv, lens = torch.bfloat16, 4, 2, [70, 200]
    T = 290
    qkv = cpu_randn((T, nh + 2 * nkv + 1, 128), 29, 1.0, dt)
    d = qkv.to(DEV)
    out = torch.full((T, nh + 1, 128), 5.0, dtype=dt, device=DEV)
    got = ops.prompt_attention(d[:, :nh], d[:, nh:nh + nkv], d[:, nh + nkv:nh + 2 * nkv], _cu(lens),
                               out=out[:, :nh])
    assert got.data_ptr() == out.data_ptr() and _status() == 0
    assert (out[270:] == 5).all() and (out[:, nh] == 5).all()
    _check(out[:270, :nh].reshape(270, -1), qkv[:270, :nh], qkv[:270, nh:nh + nkv],
           qkv[:270, nh + nkv:nh + 2 * nkv], lens, lens, dt)
    none = ops.prompt_attention(d[:0, :nh], d[:0, nh:nh + nkv], d[:0, nh:nh + nkv], _cu([0]))
    assert none.shape == (0, nh * 128)
    zero = ops.prompt_attention(d[:9, :nh], d[:0, nh:nh + nkv], d[:0, nh:nh + nkv], _cu([9]),
                                _cu([0]))
    assert (zero == 0).all() and _status() == 0


def test_masked_places_never_count():
    """NaN and infinities in other sequences, behind the last one, and in keys that a
    query does not see."""
    from parallel_serve_b200 import ops
    dt, nh, nkv, lens = torch.float16, 2, 1, [40, 150, 30]
    T = sum(lens) + 64
    q, k, v = (cpu_randn((T, n, 128), 31 + i, 1.0, dt).to(DEV) for i, n in enumerate((nh, nkv, nkv)))
    want = ops.prompt_attention(q, k, v, _cu(lens))
    for t in (q, k, v):
        t[sum(lens):] = float("nan")
    for a, b in ((40, 190),):                     # the middle sequence
        for t, x in ((q, float("nan")), (k, float("nan")), (v, float("inf"))):
            t[a:b] = x
    k[20:40] = float("nan")                       # keys that queries 0..19 do not see
    v[20:40] = float("inf")
    out = ops.prompt_attention(q, k, v, _cu(lens))
    assert torch.equal(out[:20], want[:20]) and torch.equal(out[190:220], want[190:220])
    assert torch.isnan(out[40:190]).all()
    assert torch.isnan(out[21:40].float()).any(-1).all()
    assert _status() == 0


def test_bad_ranges_are_skipped():
    from parallel_serve_b200 import ops
    dt, nh, nkv = torch.float16, 2, 1
    q, k, v = (cpu_randn((100, n, 128), 41 + i, 1.0, dt).to(DEV) for i, n in enumerate((nh, nkv, nkv)))
    out = torch.full((100, nh * 128), 3.0, dtype=dt, device=DEV)
    good = ops.prompt_attention(q, k, v, _cu([50]), _cu([60]))
    cu_q = torch.tensor([0, 50, 100], dtype=torch.int32, device=DEV)
    cu_k = torch.tensor([0, 60, 101], dtype=torch.int32, device=DEV)
    ops.prompt_attention(q, k, v, cu_q, cu_k, out=out)
    assert _status() == 4
    assert torch.equal(out[:50], good[:50]) and (out[50:] == 3).all()


def test_graph_replay_follows_the_lengths():
    from parallel_serve_b200 import ops
    dt, nh, nkv = torch.bfloat16, 4, 2
    q, k, v = (cpu_randn((600, n, 128), 51 + i, 1.0, dt).to(DEV) for i, n in enumerate((nh, nkv, nkv)))
    cu = _cu([100, 300, 200])
    out = torch.zeros(600, nh * 128, dtype=dt, device=DEV)
    ops.prompt_attention(q, k, v, cu, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.prompt_attention(q, k, v, cu, out=out)
    cu.copy_(_cu([257, 3, 340]))
    graph.replay()
    want = ops.prompt_attention(q, k, v, cu)
    assert torch.equal(out, want) and _status() == 0


@pytest.mark.parametrize("dt", DTYPES)
def test_non_finite_values_reach_their_queries_only(dt):
    from parallel_serve_b200 import ops
    nh, nkv, lens = 2, 1, [400]
    q, k, v = (cpu_randn((400, n, 128), 61 + i, 1.0, dt).to(DEV) for i, n in enumerate((nh, nkv, nkv)))
    want = ops.prompt_attention(q, k, v, _cu(lens))
    for key in (0, 127, 128, 200, 256, 399):
        bad = v.clone()
        bad[key, 0, 77] = float("nan") if key & 1 else float("inf")
        out = ops.prompt_attention(q, k, bad, _cu(lens))
        assert torch.equal(out[:key], want[:key]), key
        assert not torch.isfinite(out.view(400, nh, 128)[key:, :, 77]).any()
    assert _status() == 0


# Long mean lengths (4096 keys and more) take CTAs of two tiles.

@pytest.mark.parametrize("dt", DTYPES)
def test_long_histories(dt):
    lens = [5, 130, 1, 300]
    _run(lens, [n + h for n, h in zip(lens, [5000, 4100, 3900, 4096])], 4, 2, dt, 71, heads=[0, 3])
    _run([257, 0], [4099, 4200], 2, 1, dt, 73, scale=1.0)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("lens,klens", [([1], [1]), ([128], [128]), ([129], [129]), ([256], [256]),
                                        ([300, 0, 513], [300, 0, 513]), ([300, 20, 7], [10, 20, 0]),
                                        ([40, 300, 100], [40, 290, 229])])
def test_two_tiles_of_short_sequences(dt, lens, klens):
    """Rows of NaN behind the last key make the mean length long."""
    from parallel_serve_b200 import ops
    nh, nkv, T = 2, 1, 4096 * len(lens) + 64
    q = cpu_randn((sum(lens), nh, 128), 81, 1.0, dt)
    k, v = (torch.full((T, nkv, 128), float("nan"), dtype=dt) for _ in range(2))
    k[:sum(klens)] = cpu_randn((sum(klens), nkv, 128), 82, 1.0, dt)
    v[:sum(klens)] = cpu_randn((sum(klens), nkv, 128), 83, 1.0, dt)
    out = ops.prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), _cu(lens), _cu(klens))
    assert _status() == 0
    _check(out, q, k[:sum(klens)], v[:sum(klens)], lens, klens, dt)


def test_two_tiles_and_non_finite_values():
    from parallel_serve_b200 import ops
    dt, nh, nkv, n = torch.float16, 2, 1, 400
    q, k, v = (cpu_randn((m, h, 128), 91 + i, 1.0, dt).to(DEV)
               for i, (m, h) in enumerate(((n, nh), (4200, nkv), (4200, nkv))))
    cu = _cu([n])
    want = ops.prompt_attention(q, k, v, cu, cu)
    for key in (0, 127, 128, 200, 256, 399):
        bad = v.clone()
        bad[key, 0, 77] = float("nan") if key & 1 else float("inf")
        out = ops.prompt_attention(q, k, bad, cu, cu)
        assert torch.equal(out[:key], want[:key]), key
        assert not torch.isfinite(out.view(n, nh, 128)[key:, :, 77]).any()
        bad = k.clone()
        bad[key, 0, 5] = float("nan")
        out = ops.prompt_attention(q, bad, v, cu, cu)
        assert torch.equal(out[:key], want[:key]), key
        assert torch.isnan(out[key:]).all()
    assert _status() == 0


@pytest.mark.parametrize("keys", [600, 4200])
@pytest.mark.parametrize("shift,extra", [(0, 8), (8, 0), (8, 8), (16, 16)])
def test_output_rows_of_any_alignment(shift, extra, keys):
    """Rows at 16-byte and at 32-byte boundaries give the same, and nothing beside them is written."""
    from parallel_serve_b200 import ops
    dt, nh, nkv, n = torch.bfloat16, 2, 1, 300
    q, k, v = (cpu_randn((m, h, 128), 111 + i, 1.0, dt).to(DEV)
               for i, (m, h) in enumerate(((n, nh), (keys, nkv), (keys, nkv))))
    cu_q, cu_k = _cu([n]), _cu([keys])
    want = ops.prompt_attention(q, k, v, cu_q, cu_k)
    stride = nh * 128 + extra
    buf = torch.full((shift + n * stride + 64,), 9.0, dtype=dt, device=DEV)
    out = buf[shift:].as_strided((n, nh * 128), (stride, 1), shift)
    ops.prompt_attention(q, k, v, cu_q, cu_k, out=out)
    assert torch.equal(out, want) and _status() == 0
    out.fill_(9.0)
    assert (buf == 9).all()
