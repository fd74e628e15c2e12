"""The 4-bit cache under tensor parallelism on one GPU: two ranks' decoders as host threads on
one stream, the all-reduce replaced by a sum of both partials that the host enqueues once
both are (no kernel waits for another)."""
from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

from conftest import rel_err, to_np
from test_gpu_prefill import _weights

pytestmark = pytest.mark.gpu
TOL = 1e-2
N_LAYERS, H, NH, FF, V, WORLD = 2, 512, 4, 512, 384, 2


class _Group:
    """What both ranks share."""

    def __init__(self):
        self.barrier = threading.Barrier(WORLD, timeout=120)
        self.slots, self.logits = {}, {}


class _Rank:
    def __init__(self, shared, rank):
        self.shared, self.rank = shared, rank


class _Sum:
    """NvlinkAllReduce's interface."""

    def __init__(self, group, max_elems, device, dtype, algo=0):
        self.g, self.rank = group.shared, group.rank
        for slot in range(2):
            self.g.slots[self.rank, slot] = torch.zeros(max_elems, dtype=dtype, device=device)

    def slot_ptr(self, slot):
        return self.g.slots[self.rank, slot].data_ptr()

    def __call__(self, slot, count, out, residual=None, *, out_sumsq=None):
        self.g.barrier.wait()                        # both partials are enqueued
        total = sum(self.g.slots[r, slot][:count].float() for r in range(WORLD)).view(out.shape)
        total = total if residual is None else total + residual.float()
        out.copy_(total)
        if out_sumsq is not None:
            out_sumsq.copy_(out.float().square().view(*out_sumsq.shape, 256).sum(-1))
        self.g.barrier.wait()                        # both sums are

    def pick(self, logits, perm, next_tokens, tokens_out=None, seq_len=None):
        self.g.logits[self.rank] = logits
        self.g.barrier.wait()
        best = torch.cat([self.g.logits[r] for r in range(WORLD)], 1).argmax(1).int()
        next_tokens.index_copy_(0, perm.long(), best)
        if tokens_out is not None:
            tokens_out.copy_(next_tokens)
        if seq_len is not None:
            seq_len.add_(1)
        self.g.barrier.wait()

    def close(self):
        pass


def _together(fn, ranks):
    """fn(rank) of both ranks at once, their results."""
    out, errors = [None] * WORLD, []

    def work(r):
        try:
            out[r] = fn(r)
        except BaseException as ex:                  # noqa: BLE001 (raised below)
            errors.append(ex)
            ranks[0].shared.barrier.abort()
    threads = [threading.Thread(target=work, args=(r,)) for r in range(WORLD)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if errors:
        raise next((e for e in errors if not isinstance(e, threading.BrokenBarrierError)), errors[0])
    return out


class _Stored:
    """Both ranks' cache of one model, heads side by side."""

    def __init__(self, values):
        self.values, self.written = values, {}

    def __setitem__(self, key, row):
        self.written[key[0], int(key[2])] = row

    def __getitem__(self, key):
        return self.values[key]


class _State:
    def __init__(self, decs, L):
        both = [[[to_np(torch.cat(t, 1)) for t in zip(*(d.read_kv(li, m, L) for d in decs))]
                 for m in range(2)] for li in range(N_LAYERS)]
        self.k = [[_Stored(kv[0]) for kv in layer] for layer in both]
        self.v = [[_Stored(kv[1]) for kv in layer] for layer in both]

    def check(self):
        for part in (self.k, self.v):
            for layer in part:
                for st in layer:
                    for (slot, pos), row in st.written.items():
                        g = row.reshape(NH, 4, 32)
                        step = (g.max(-1) - g.min(-1))[..., None] / 15
                        got = st.values[slot, :, pos].reshape(g.shape)
                        assert np.all(np.abs(got - g) <= 0.51 * step + TOL * np.abs(g).mean())


@pytest.mark.parametrize("page,chunk", [(None, 8), (16, 256)])
def test_two_ranks_prefill_and_decode(monkeypatch, page, chunk):
    import torch.distributed as dist

    import oracle
    import parallel_serve_b200.tp as tp
    from parallel_serve_b200.decoder import DecoderConfig, TwoModelDecoder
    shared = _Group()
    ranks = [_Rank(shared, r) for r in range(WORLD)]
    monkeypatch.setattr(dist, "get_world_size", lambda g: WORLD)
    monkeypatch.setattr(dist, "get_rank", lambda g: g.rank)
    monkeypatch.setattr(tp, "NvlinkAllReduce", _Sum)
    cfg = DecoderConfig(n_layers=N_LAYERS, hidden=H, n_heads=NH, ffn=FF, vocab=V)
    w = _weights(N_LAYERS, H, FF, V, 9)
    P = dict(layers=[{k: to_np(v) for k, v in L.items()} for L in w["layers"]], emb=to_np(w["emb"]),
             ln_f=to_np(w["ln_f"]), W_lm=to_np(w["W_lm"]))
    ids, lens, L_cap = [0, 1, 1, 0], [5, 19, 1, 21], 40
    g = torch.Generator().manual_seed(38)
    prompts = [torch.randint(0, V, (n,), generator=g).tolist() for n in lens]
    decs = [TwoModelDecoder(cfg, ids, L_cap, weights=w, page_size=page, prefill_chunk=chunk, kv_bits=4,
                            tp_group=r) for r in ranks]
    _together(lambda r: decs[r].prefill(prompts), ranks)
    torch.cuda.synchronize()
    cos, sin = oracle.rope_tables(decs[0].L_cap)
    mids = np.array(ids)

    def logits():
        return to_np(torch.cat([d.logits for d in decs], 1))
    st = _State(decs, max(lens))
    _, want = oracle.prefill(prompts, mids, P, st, NH, cos, sin, 1e-5)
    assert rel_err(logits(), want) < TOL
    st.check()
    seq = np.array(lens)
    for _ in range(3):
        tokens = decs[0].tokens.cpu().numpy().astype(np.int64)
        assert np.array_equal(tokens, decs[1].tokens.cpu().numpy())
        _together(lambda r: decs[r].step_device("fused"), ranks)
        torch.cuda.synchronize()
        st = _State(decs, int(seq.max()) + 1)
        _, want = oracle.decode_step(tokens, mids, P, st, seq, NH, cos, sin, 1e-5)
        assert rel_err(logits(), want) < TOL
        st.check()
    decs[0].check_status()
