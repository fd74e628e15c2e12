"""Arguments that the 4-bit cache, prompt attention and decoder entry points refuse on the
host, before anything is launched. No GPU."""
from __future__ import annotations

import pytest
import torch

from parallel_serve_b200 import _lib, ops
from test_kv4_host import BAD, P, cache, prompt


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 2.5e38, -2.5e38])
def test_scales_that_are_not_finite_in_fp32(scale):
    """times log2 e, as the kernels take them."""
    assert _lib.lib.ps_kv4_decode_attention(P, 1024, cache(), P, P, None, None, 0, 0, 8, 64, scale, 0,
                                            None, 0, None, None) == BAD
    assert prompt(scale=scale) == BAD


def test_scales_of_a_decode_call():
    """Any finite scale, negative ones and 0 included, is a softmax."""
    for scale in (0.1, 0.0, -3.0, 1e38):
        assert _lib.lib.ps_kv4_decode_attention(P, 1024, cache(), P, P, None, None, 0, 0, 8, 64, scale,
                                                0, None, 0, None, None) == 0


def test_a_captured_stream_of_another_device_gets_its_own_workspace(monkeypatch):
    """Whether a call is captured is asked of its tensors' device, not of the current one."""
    now = [0]

    class Device:
        def __init__(self, idx):
            self.idx = idx

        def __enter__(self):
            self.was, now[0] = now[0], self.idx

        def __exit__(self, *a):
            now[0] = self.was
    shared = torch.zeros(1)
    monkeypatch.setattr(ops, "_current_device", lambda: now[0])
    monkeypatch.setattr(ops, "_raw_stream", lambda idx: 7)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now[0] == 1)
    monkeypatch.setattr(_lib, "stream_workspace", lambda idx, stream, nbytes, tag: shared)
    like = torch.zeros(1)
    assert ops._counter_workspace(like, 0, 5000, "x", 4096) is shared
    ws = ops._counter_workspace(like, 1, 5000, "x", 4096)
    assert ws is not shared and ws.numel() == 5000 and bool((ws[:4096] == 0).all()) and now == [0]


def _decoder(page_size=None):
    """A decoder's bookkeeping alone: 2 sequences of model 0 and 1 of model 1, 64 positions."""
    from parallel_serve_b200.decoder import TwoModelDecoder
    from parallel_serve_b200.paged_kv import BlockTable, PageAllocator
    dec = TwoModelDecoder.__new__(TwoModelDecoder)
    dec.device, dec.dt, dec.nh, dec.kv_bits = torch.device("cpu"), torch.float16, 2, 4
    dec.counts_host, dec.L_cap, dec.page_size, dec.block_table = (2, 1), 64, page_size, None
    if page_size:
        dec.block_table = BlockTable([0, 0, 1], (PageAllocator(8), PageAllocator(4)), 64 // page_size,
                                     page_size)
    return dec


def test_a_history_needs_its_room():
    """Positions beyond the capacity, pages that are not reserved and sequences that the model does
    not have were left out of the cache in silence."""
    dec, kv = _decoder(), lambda n, L: (torch.zeros(n, 2, L, 128),) * 2
    for n, L in ((2, 65), (1, 4), (3, 4)):
        with pytest.raises(ValueError):
            dec.write_kv(0, 0, *kv(n, L))
    with pytest.raises(ValueError):
        dec.write_kv(0, 0, kv(2, 4)[0], kv(2, 5)[0])
    with pytest.raises(ValueError):
        dec.read_kv(0, 1, 65)
    dec = _decoder(16)
    with pytest.raises(ValueError):
        dec.write_kv(0, 0, *kv(2, 4))
    with pytest.raises(ValueError):
        dec.read_kv(0, 1, 4)
    dec.block_table.ensure(range(3), 20)             # reserved on the host, not yet on the device
    seqs, cu = dec._kv4_sequences(0, 32)
    assert seqs.tolist() == [[0, 0, 0], [0, 1, 0]] and cu.tolist() == [0, 32, 64]
    assert torch.equal(dec.block_table.device, torch.from_numpy(dec.block_table.host))
    with pytest.raises(ValueError):
        dec._kv4_sequences(1, 33)
    dec.write_kv(0, 0, *kv(2, 0))                    # no positions: nothing to do


@pytest.mark.parametrize("page_size", [4, 12, 8192])
def test_page_sizes_of_a_4_bit_decoder(page_size):
    """Refused where it is made, not at the first step, and before anything is allocated."""
    from parallel_serve_b200.decoder import DecoderConfig, TwoModelDecoder
    cfg = DecoderConfig(n_layers=1, hidden=256, n_heads=2, ffn=256, vocab=256)
    with pytest.raises(ValueError, match="power of two"):
        TwoModelDecoder(cfg, [0, 1], 64, kv_bits=4, page_size=page_size)


def test_gather_takes_two_pools():
    from parallel_serve_b200 import KV4Pool
    pool = KV4Pool.zeros(2, 1, 8, device="cpu")
    none = KV4Pool.zeros(0, 1, 8, device="cpu")
    seqs, cu = torch.zeros(1, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for pools in ((), (None,), (none,), (pool,), (pool, None, None), (None, None)):
        with pytest.raises(ValueError):
            ops.kv4_gather(pools, seqs, cu, 0)
