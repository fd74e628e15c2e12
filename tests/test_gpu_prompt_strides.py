"""Prompt attention on rows far apart: token strides whose offsets pass 32 bits."""
from __future__ import annotations

import pytest
import torch

from conftest import cpu_randn

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("keys", [700, 4200])         # one tile a CTA, and two
def test_offsets_beyond_32_bits(keys):
    from parallel_serve_b200 import _lib, ops
    dt, nh, nkv, n = torch.bfloat16, 2, 1, 600
    stride = 1 << 22                                  # 600 tokens: 2.5e9 elements
    buf = torch.empty(n * stride, dtype=dt, device=DEV)
    q = buf.as_strided((n, nh, 128), (stride, 128, 1))
    out = buf.as_strided((n, nh * 128), (stride, 1), 1024)
    q.copy_(cpu_randn((n, nh, 128), 161, 1.0, dt))
    k, v = (cpu_randn((keys, nkv, 128), 162 + i, 1.0, dt).to(DEV) for i in range(2))
    cu_q, cu_k = (torch.tensor([0, m], dtype=torch.int32, device=DEV) for m in (n, keys))
    ops.prompt_attention(q, k, v, cu_q, cu_k, out=out)
    want = ops.prompt_attention(q.contiguous(), k, v, cu_q, cu_k)
    assert torch.equal(out, want)
    far = buf.as_strided((n, nkv, 128), (stride, 128, 1), 2048), buf.as_strided((n, nkv, 128), (stride, 128, 1), 4096)
    far[0].copy_(k[:n])
    far[1].copy_(v[:n])
    got = ops.prompt_attention(q, *far, cu_q)
    assert torch.equal(got, ops.prompt_attention(q.contiguous(), k[:n].contiguous(), v[:n].contiguous(), cu_q))
    assert _lib.read_status(torch.device(DEV, 0)) == 0
