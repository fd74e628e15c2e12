"""The decode loop with its KV cache in 4 bits, against the oracle reading the same
cache: prefill (any chunking, paged or not), decode steps, graph replay, history
in and out. The cache itself is checked against what the oracle would store: half a
quantisation step, and the 16-bit GEMM's error beside it."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import rel_err, to_np
from test_gpu_prefill import _weights

pytestmark = pytest.mark.gpu
TOL = 1e-2
N_LAYERS, H, NH, FF, V = 2, 256, 2, 512, 384


class _Stored:
    """One model's cache as the decoder holds it; what the oracle writes is kept apart."""

    def __init__(self, values):
        self.values, self.written = values, {}

    def __setitem__(self, key, row):
        self.written[key[0], int(key[2])] = row

    def __getitem__(self, key):
        return self.values[key]


class _State:
    def __init__(self, dec, L):
        both = [[dec.read_kv(li, m, L) for m in range(2)] for li in range(N_LAYERS)]
        self.k = [[_Stored(to_np(kv[0])) for kv in layer] for layer in both]
        self.v = [[_Stored(to_np(kv[1])) for kv in layer] for layer in both]

    def check(self):
        for part in (self.k, self.v):
            for layer in part:
                for st in layer:
                    for (slot, pos), row in st.written.items():
                        g = row.reshape(NH, 4, 32)
                        step = (g.max(-1) - g.min(-1))[..., None] / 15
                        got = st.values[slot, :, pos].reshape(g.shape)
                        assert np.all(np.abs(got - g) <= 0.51 * step + TOL * np.abs(g).mean())


def _decoder(ids, L_cap, page, chunk=256):
    from parallel_serve_b200.decoder import DecoderConfig, TwoModelDecoder
    cfg = DecoderConfig(n_layers=N_LAYERS, hidden=H, n_heads=NH, ffn=FF, vocab=V)
    w = _weights(N_LAYERS, H, FF, V, 7)
    dec = TwoModelDecoder(cfg, ids, L_cap, weights=w, page_size=page, prefill_chunk=chunk, kv_bits=4)
    P = dict(layers=[{k: to_np(v) for k, v in L.items()} for L in w["layers"]], emb=to_np(w["emb"]),
             ln_f=to_np(w["ln_f"]), W_lm=to_np(w["W_lm"]))
    return dec, P


@pytest.mark.parametrize("page,chunk", [(None, 8), (None, 256), (16, 13), (8, 256)])
def test_prefill_and_decode(page, chunk):
    import oracle
    ids, lens, L_cap = [0, 1, 1, 0, 1, 0], [5, 9, 1, 21, 7, 3], 40
    g = torch.Generator().manual_seed(8)
    prompts = [torch.randint(0, V, (n,), generator=g).tolist() for n in lens]
    dec, P = _decoder(ids, L_cap, page, chunk)
    dec.prefill(prompts)
    torch.cuda.synchronize()
    dec.check_status()
    cos, sin = oracle.rope_tables(dec.L_cap)
    mids = np.array(ids)
    st = _State(dec, max(lens))
    nxt, logits = oracle.prefill(prompts, mids, P, st, NH, cos, sin, 1e-5)
    assert rel_err(to_np(dec.logits), logits) < TOL
    st.check()
    seq = np.array(lens)
    for _ in range(3):
        tokens = dec.tokens.cpu().numpy().astype(np.int64)
        dec.step_device("fused")
        torch.cuda.synchronize()
        st = _State(dec, int(seq.max()) + 1)
        _, logits = oracle.decode_step(tokens, mids, P, st, seq, NH, cos, sin, 1e-5)
        assert rel_err(to_np(dec.logits), logits) < TOL
        st.check()
    dec.check_status()


def test_chunking_does_not_change_the_result():
    ids, L_cap = [0, 1, 0], 64
    g = torch.Generator().manual_seed(18)
    prompts = [torch.randint(0, V, (n,), generator=g).tolist() for n in (33, 12, 50)]
    logits = []
    for page, chunk in ((None, 256), (16, 256)):
        dec, _ = _decoder(ids, L_cap, page, chunk)
        dec.prefill(prompts)
        logits.append(dec.logits.clone())
    assert torch.equal(logits[0], logits[1])     # pages only move the rows


def test_graph_serial_mode_and_history():
    ids, L_cap = [0, 1, 1, 0], 48
    dec, _ = _decoder(ids, L_cap, 16)
    gen = torch.Generator().manual_seed(3)
    hist = [[torch.randn(2, NH, 17, 128, generator=gen).to(torch.float16) for _ in range(2)]
            for _ in range(2 * N_LAYERS)]
    tokens = torch.tensor([5, 17, 29, 101])

    def reset():
        dec.set_state(tokens, [17] * 4)
        for li in range(N_LAYERS):
            for m in range(2):
                dec.write_kv(li, m, *hist[2 * li + m])
    reset()
    for li in range(N_LAYERS):
        for m in range(2):
            for got, want in zip(dec.read_kv(li, m, 17), hist[2 * li + m]):
                g = want.double().view(2, NH, 17, 4, 32)
                step = (g.amax(-1) - g.amin(-1))[..., None] / 15
                err = (got.cpu().double().view(g.shape) - g).abs()
                assert bool((err <= 0.505 * step + 1e-3 * g.abs()).all())
    dec.step_device("fused")
    want = dec.logits.clone()
    reset()
    dec.step_device("serial")
    assert rel_err(to_np(dec.logits), to_np(want)) < 1e-3
    reset()
    dec.reserve(4)
    dec.capture("fused")
    reset()
    dec.replay("fused")
    torch.cuda.synchronize()
    assert torch.equal(dec.logits, want)
    dec.check_status()
    assert dec.launches_per_step() == 3 + 6 * N_LAYERS + 1 + 1


def test_long_random_history_runs():
    dec, _ = _decoder([0, 1] * 4, 2048, None)
    dec.fill_kv_random(1500)
    dec.set_state(torch.arange(8), [1500] * 8)
    dec.step_device("fused")
    torch.cuda.synchronize()
    dec.check_status()
    assert torch.isfinite(dec.logits).all()
