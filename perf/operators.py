"""Timed cases of the 4-bit KV cache operators and of the prompt attention.

Each case is one pass through one operator: in its plain form (elementary torch
operations in 32 bits) or, with ``own`` set, through the package's entry points.

The 4-bit cache format: a row is the 128 channels of one (position, kv head), in
4 groups of 32 channels. A group stores zero z = T(min) and scale
s = T((max - z) / 15) in the model's 16-bit type T, and codes
c = clamp(rint((x - z) / s), 0, 15); it stands for s * c + z. A row's 64 code
bytes are 16 words of 8 codes (low nibble first); word w of group g is stored at
4 * w + g, so that a row is the 4 x 4 transpose of its natural word order.
"""
import math
import random

import numpy as np
import torch

own = False

D, GROUP = 128, 32
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one decode step's q and k of 64 sequences, 32 heads on 8: launch latency
        dict(name="norm_rope_step", op="norm_rope", tokens=64, heads=32, kv_heads=8, rotary=128,
             interleaved=False, norm=True, dtype="bf16"),
        # a prompt chunk of 16384 tokens, interleaved pairs over half of the head
        dict(name="norm_rope_prompt", op="norm_rope", tokens=16384, heads=32, kv_heads=8, rotary=64,
             interleaved=True, norm=True, dtype="fp16"),
        # the cache write of one decode step of the 64-sequence, 32-head workload, rows read back
        dict(name="kv4_write_read_step", op="write_read", seqs=64, longest=1, history=2048, heads=32,
             kv_heads=32, page=0, norm=True, dtype="fp16"),
        # ragged prompts into 16-position pages, read back whole
        dict(name="kv4_write_read_ragged", op="write_read", seqs=13, longest=1777, history=0, heads=32,
             kv_heads=8, page=16, norm=False, dtype="bf16"),
        # a large prefill of a 32-head model
        dict(name="kv4_write_read_prompts", op="write_read", seqs=16, longest=2048, history=0, heads=32,
             kv_heads=32, page=0, norm=False, dtype="fp16"),
        # one sequence, one token: latency
        dict(name="kv4_decode_single", op="decode", seqs=1, longest=1023, heads=32, kv_heads=8, page=0,
             dtype="bf16"),
        # the 64-sequence, 2048-position, 32-head workload with its cache in 4 bits
        dict(name="kv4_decode_b64", op="decode", seqs=64, longest=2048, heads=32, kv_heads=32, page=0,
             dtype="fp16"),
        # ragged paged batch with grouped heads
        dict(name="kv4_decode_ragged", op="decode", seqs=96, longest=16411, heads=40, kv_heads=8, page=16,
             dtype="bf16"),
        # few long contexts
        dict(name="kv4_decode_long", op="decode", seqs=4, longest=131072, heads=32, kv_heads=8, page=64,
             dtype="bf16"),
        # a few short prompts arriving together
        dict(name="prompt_short", op="prompt", seqs=7, longest=173, history=0, heads=32, kv_heads=8,
             dtype="bf16"),
        # ragged prompts, some with history before them
        dict(name="prompt_ragged", op="prompt", seqs=9, longest=4099, history=777, heads=32, kv_heads=32,
             dtype="fp16"),
        # one long prompt with grouped heads
        dict(name="prompt_long", op="prompt", seqs=1, longest=16384, history=0, heads=32, kv_heads=8,
             dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rope", "write_read", "decode", "prompt"])
    kv = rng.choice([1, 2, 4, 8, 8, 10])
    heads = kv * rng.choice([1, 2, 4, 5, 8])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "norm_rope":
        return dict(op=op, tokens=_log(rng, 1, 8000), heads=heads, kv_heads=kv,
                    rotary=rng.choice([32, 64, 96, 128, 128]), interleaved=rng.random() < 0.5,
                    norm=rng.random() < 0.7, dtype=dtype)
    page = rng.choice([0, 8, 16, 32, 128])
    if op == "write_read":
        longest = rng.choice([1, _log(rng, 2, 1500)])
        return dict(op=op, seqs=_log(rng, 1, 12 if longest > 1 else 200), longest=longest,
                    history=_log(rng, 1, 900) - 1, heads=heads, kv_heads=kv, page=page,
                    norm=longest == 1 and rng.random() < 0.5, dtype=dtype)
    if op == "decode":
        longest = _log(rng, 1, 40000)
        return dict(op=op, seqs=_log(rng, 1, max(2, min(150, 400000 // longest))), longest=longest,
                    heads=heads, kv_heads=kv, page=page, dtype=dtype)
    longest = _log(rng, 1, 6000)
    return dict(op=op, seqs=_log(rng, 1, max(2, min(40, 12000 // longest))), longest=longest,
                history=rng.choice([0, 0, _log(rng, 1, 1500)]), heads=heads, kv_heads=kv, dtype=dtype)


def _lens(case):
    """The case's sequence lengths: the longest first, the others spread below it
    (equal lengths where the longest is a power of two: a padded workload)."""
    n, longest = case["seqs"], case["longest"]
    if longest & (longest - 1) == 0:
        return [longest] * n
    rng = random.Random(1000 * longest + n)
    return [longest] + [max(1, int(longest * rng.random())) for _ in range(n - 1)]


def _histories(case, n):
    """Cached positions before each sequence's new ones."""
    h = case.get("history", 0)
    if not h or h & (h - 1) == 0:
        return [h] * n
    rng = random.Random(77 * h + n)
    return [int(h * rng.random()) for _ in range(n)]


def _pairs(lens, hist):
    return sum(n * h + n * (n + 1) // 2 for n, h in zip(lens, hist))


def work(case):
    h, kv = case["heads"], case["kv_heads"]
    if case["op"] == "norm_rope":
        t, r = case["tokens"], case["rotary"]
        rows = t * (h + kv)
        return {"bytes": rows * D * 4 + t * (4 + r * 4), "flops": rows * (4 * D + 3 * r)}
    lens = _lens(case)
    t = sum(lens)
    if case["op"] == "write_read":
        q = t * h * D * 4
        kvb = t * kv * (2 * D * 2 + 2 * 80 + 2 * 80 + 2 * D * 2)  # read, written, read back, returned
        return {"bytes": q + kvb + t * (4 + D * 4), "flops": t * kv * D * 2 * 8 + t * (h + kv) * D * 7}
    if case["op"] == "decode":
        return {"bytes": t * kv * 160 + case["seqs"] * h * D * 4, "flops": t * h * D * 4}
    hist = _histories(case, case["seqs"])
    keys = t + sum(hist)
    return {"bytes": t * h * D * 4 + keys * kv * D * 4, "flops": 4 * D * h * _pairs(lens, hist)}


# ---------------------------------------------------------------- the 4-bit format
def _quantise(x, dt):
    """x [..., 128] -> codes [..., 4, 32] (uint8), scale and zero [..., 4] of type dt."""
    g = x.reshape(*x.shape[:-1], D // GROUP, GROUP)
    z = g.amin(-1).to(dt)
    s = ((g.amax(-1) - z.float()) / torch.full((), 15.0, device=x.device)).to(dt)
    step = torch.where(s == 0, 1.0, s.float()).unsqueeze(-1)
    c = ((g - z.float().unsqueeze(-1)) / step).round().clamp(0, 15).to(torch.uint8)
    return c, s, z


def _pack(c):
    """codes [..., 4, 32] -> bytes [..., 64]."""
    b = c[..., 0::2] | (c[..., 1::2] << 4)                      # [..., 4 groups, 16 bytes]
    b = b.reshape(*b.shape[:-1], 4, 4)                          # [..., group, word, byte]
    return b.transpose(-2, -3).reshape(*b.shape[:-3], 64)


def _unpack(b):
    """bytes [..., 64] -> codes [..., 4, 32]."""
    b = b.reshape(*b.shape[:-1], 4, 4, 4).transpose(-2, -3)     # [..., group, word, byte]
    c = torch.stack([b & 15, b >> 4], -1)
    return c.reshape(*c.shape[:-4], 4, 32)


def _values(codes, meta, real=torch.float32):
    """Bytes [..., 64] and meta [..., 4, 2] -> the values they stand for, [..., 128]."""
    m = meta.to(real)
    v = _unpack(codes).to(real) * m[..., 0:1] + m[..., 1:2]
    return v.reshape(*v.shape[:-2], D)


def _fill(pool, part, gen, dt):
    """Fill one K or V pool with the quantised form of N(0, 1) rows, a slot at a time."""
    codes, meta = pool[part + "_codes"], pool[part + "_meta"]
    step = max(1, (1 << 26) // (codes[0].numel() * 2))
    for i in range(0, codes.shape[0], step):
        x = torch.randn(*codes[i:i + step].shape[:-1], D, generator=gen, device=codes.device)
        c, s, z = _quantise(x, dt)
        codes[i:i + step] = _pack(c)
        meta[i:i + step] = torch.stack([s, z], -1)


def _new_pool(rows, kv, length, dt, dev):
    p = {}
    for part in ("k", "v"):
        p[part + "_codes"] = torch.zeros(rows, kv, length, 64, dtype=torch.uint8, device=dev)
        p[part + "_meta"] = torch.zeros(rows, kv, length, 4, 2, dtype=dt, device=dev)
    return p


def _cache(case, total, gen, dt, dev):
    """Two models' pools for sequences of `total` positions each (the first half of
    the sequences belong to model 0) and the block table when the case has pages."""
    n, kv, page = len(total), case["kv_heads"], case["page"]
    n0 = n - n // 2
    cap = max(total)
    if not page:
        return n0, [_new_pool(m, kv, cap, dt, dev) if m else None for m in (n0, n - n0)], None
    pages = -(-cap // page)
    table = torch.full((n, pages), -1, dtype=torch.int32)
    pools = []
    for a, b in ((0, n0), (n0, n)):
        need = [-(-t // page) for t in total[a:b]]
        ids = torch.randperm(sum(need), generator=torch.Generator().manual_seed(n * 31 + cap))
        at = 0
        for i, k in enumerate(need):
            table[a + i, :k] = ids[at:at + k].to(torch.int32)
            at += k
        pools.append(_new_pool(at, kv, page, dt, dev) if at else None)
    return n0, pools, table.to(dev)


def _tables(n, rotary, dev):
    inv = 10000.0 ** (-2.0 * torch.arange(rotary // 2, dtype=torch.float64, device=dev) / rotary)
    ang = torch.arange(n, dtype=torch.float64, device=dev)[:, None] * inv
    return ang.cos().float().contiguous(), ang.sin().float().contiguous()


def _cum(lens, dev):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=dev)


def prepare(case, seed):
    dev, dt = torch.device("cuda"), DT[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)
    h, kv = case["heads"], case["kv_heads"]

    def rnd(*shape):
        return torch.randn(*shape, generator=gen, device=dev).to(dt)

    def weights():
        # RMSNorm weights of the two models
        return (1 + 0.2 * torch.randn(2, D, generator=gen, device=dev)).to(dt)

    st = dict(op=case["op"], heads=h, kv=kv, dt=dt)
    if case["op"] == "norm_rope":
        t = case["tokens"]
        qkv = rnd(t, h + 2 * kv, D)
        st.update(qkv=qkv, q=qkv[:, :h], k=qkv[:, h:h + kv], interleaved=case["interleaved"],
                  n0=t - t // 2, pos=torch.randint(0, 32768, (t,), generator=gen, device=dev).int())
        st["cos"], st["sin"] = _tables(32768, case["rotary"], dev)
        st["wq"], st["wk"] = (weights(), weights()) if case["norm"] else (None, None)
        return st
    lens = _lens(case)
    n, t = len(lens), sum(lens)
    if case["op"] == "prompt":
        hist = _histories(case, n)
        qkv = rnd(t, h, D)
        klens = [a + b for a, b in zip(lens, hist)]
        st.update(q=qkv, k=rnd(sum(klens), kv, D), v=rnd(sum(klens), kv, D), lens=lens, klens=klens,
                  cu_q=_cum(lens, dev), cu_k=_cum(klens, dev))
        return st
    hist = _histories(case, n)
    total = [a + b for a, b in zip(lens, hist)]
    n0, pools, table = _cache(case, total, gen, dt, dev)
    st.update(n0=n0, pools=pools, table=table, page=case["page"])
    slots = [i if i < n0 else i - n0 for i in range(n)]
    if case["op"] == "decode":
        for pool in pools:
            for part in ("k", "v"):
                if pool is not None:
                    _fill(pool, part, gen, dt)
        st.update(q=rnd(n, h, D), lens=total, longest=max(total),
                  pos=torch.tensor([x - 1 for x in total], dtype=torch.int32, device=dev))
    else:
        qkv = rnd(t, h + 2 * kv, D)
        seq = torch.repeat_interleave(torch.arange(n), torch.tensor(lens))
        off = torch.arange(t) - torch.tensor([0] + list(np.cumsum(lens))[:-1])[seq]
        home = seq if table is not None else torch.tensor(slots)[seq]
        st.update(q=qkv[:, :h], k=qkv[:, h:h + kv], v=qkv[:, h + kv:], qkv=qkv,
                  pos=(off + torch.tensor(hist)[seq]).int().to(dev), home=home.int().to(dev),
                  split=sum(lens[:n0]), cu=_cum(lens, dev), total=t)
        st["seqs"] = torch.tensor([[0 if i < n0 else 1, i if table is not None else slots[i], hist[i]]
                                   for i in range(n)], dtype=torch.int32, device=dev)
        st["cos"], st["sin"] = _tables(max(total), D, dev)
        st["wq"], st["wk"] = (weights(), weights()) if case["norm"] else (None, None)
    st["kv4"] = tuple(None if p is None else (p["k_codes"], p["k_meta"], p["v_codes"], p["v_meta"])
                      for p in pools)
    return st


# ---------------------------------------------------------------- plain forms
def _norm(x, w, n0, eps):
    x = x.float()
    if w is None:
        return x
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    w = w.float()
    return torch.cat([x[:n0] * w[0], x[n0:] * w[1]])


def _rope(x, cos, sin, pos, interleaved):
    c, s = cos[pos.long()].unsqueeze(1), sin[pos.long()].unsqueeze(1)
    half = c.shape[-1]
    r = x[..., :2 * half]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :half], r[..., half:])
    a, b = a * c - b * s, b * c + a * s
    r = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([r, x[..., 2 * half:]], -1)


def _addresses(st, rows, pos, m):
    """Row and column of each token's cache entry in model m's pool."""
    if st["table"] is None:
        return rows.long(), pos.long()
    return st["table"][rows.long(), (pos // st["page"]).long()].long(), (pos % st["page"]).long()


def _plain_write_read(st):
    dt, n0 = st["dt"], st["split"]
    q = _rope(_norm(st["q"], st["wq"], n0, 1e-6), st["cos"], st["sin"], st["pos"], False).to(dt)
    k = _rope(_norm(st["k"], st["wk"], n0, 1e-6), st["cos"], st["sin"], st["pos"], False)
    out = []
    for part, x in (("k", k), ("v", st["v"].float())):
        c, s, z = _quantise(x, dt)
        codes, meta, back = _pack(c), torch.stack([s, z], -1), []
        for m, sl in ((0, slice(0, n0)), (1, slice(n0, st["total"]))):
            pool = st["pools"][m]
            if pool is None:
                continue
            row, col = _addresses(st, st["home"][sl], st["pos"][sl], m)
            pool[part + "_codes"][row, :, col] = codes[sl]
            pool[part + "_meta"][row, :, col] = meta[sl]
            back.append(_values(pool[part + "_codes"][row, :, col], pool[part + "_meta"][row, :, col]))
        out.append(torch.cat(back).to(dt))
    return {"q": q, "k": out[0], "v": out[1]}


def _visible(st, m, part, real):
    """Model m's cached rows of its sequences, [seqs, kv, longest, 128]."""
    pool, sl = st["pools"][m], (slice(0, st["n0"]) if m == 0 else slice(st["n0"], None))
    codes, meta = pool[part + "_codes"], pool[part + "_meta"]
    if st["table"] is not None:
        t = st["table"][sl].long().clamp_min(0)
        codes, meta = (x[t].transpose(1, 2).flatten(2, 3) for x in (codes, meta))
    return _values(codes, meta, real)


def _plain_decode(st):
    out = []
    for m, sl in ((0, slice(0, st["n0"])), (1, slice(st["n0"], None))):
        if st["pools"][m] is None:
            continue
        q, pos = st["q"][sl].float(), st["pos"][sl]
        q = q.reshape(q.shape[0], st["kv"], -1, D)
        k = _visible(st, m, "k", torch.float32)
        s = q @ k.transpose(-1, -2) / math.sqrt(D)
        del k
        hidden = torch.arange(s.shape[-1], device=s.device) > pos[:, None]
        s = s.masked_fill(hidden[:, None, None], -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = (p @ _visible(st, m, "v", torch.float32)) / p.sum(-1, keepdim=True)
        out.append(o.reshape(q.shape[0], -1).to(st["dt"]))
    return torch.cat(out)


def _plain_prompt(st):
    out, a, b = [], 0, 0
    group = st["heads"] // st["kv"]
    for n, nk in zip(st["lens"], st["klens"]):
        q = st["q"][a:a + n].float().reshape(n, st["kv"], group, D).permute(1, 2, 0, 3)
        k, v = (st[x][b:b + nk].float().permute(1, 0, 2) for x in ("k", "v"))
        i = torch.arange(n, device=q.device)[:, None] + (nk - n)
        hidden = torch.arange(nk, device=q.device)[None] > i
        # as many kv heads together as keep the score matrix within a few GB
        step = max(1, (1 << 30) // (group * n * nk))
        heads = []
        for j in range(0, st["kv"], step):
            s = q[j:j + step] @ k[j:j + step].unsqueeze(1).transpose(-1, -2) / math.sqrt(D)
            s = s.masked_fill_(hidden, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            heads.append(p @ v[j:j + step].unsqueeze(1) / p.sum(-1, keepdim=True))
        out.append(torch.cat(heads).permute(2, 0, 1, 3).reshape(n, -1))
        a, b = a + n, b + nk
    return torch.cat(out).to(st["dt"])


def run(st):
    if own:
        return _own(st)
    if st["op"] == "norm_rope":
        return [_rope(_norm(st[x], st["w" + x], st["n0"], 1e-6), st["cos"], st["sin"], st["pos"],
                      st["interleaved"]).to(st["dt"]) for x in ("q", "k")]
    return {"write_read": _plain_write_read, "decode": _plain_decode, "prompt": _plain_prompt}[st["op"]](st)


def _own(st):
    from parallel_serve_b200 import ops
    if st["op"] == "norm_rope":
        return list(ops.qk_norm_rope(st["q"], st["k"], st["pos"], q_weight=st["wq"], k_weight=st["wk"],
                                     eps=1e-6, rope_cos=st["cos"], rope_sin=st["sin"],
                                     interleaved=st["interleaved"], split_point=st["n0"]))
    if st["op"] == "write_read":
        q = ops.kv4_append(st["k"], st["v"], st["kv4"], st["pos"], q=st["q"], q_weight=st["wq"],
                           k_weight=st["wk"], eps=1e-6, rope_cos=st["cos"], rope_sin=st["sin"],
                           rows=st["home"], block_table=st["table"], split_point=st["split"])
        k, v = ops.kv4_gather(st["kv4"], st["seqs"], st["cu"], st["total"], block_table=st["table"])
        return {"q": q, "k": k, "v": v}
    if st["op"] == "decode":
        return ops.kv4_decode_attention(st["q"], st["kv4"], st["pos"], max_len=st["longest"],
                                        block_table=st["table"], split_point=st["n0"])
    return ops.prompt_attention(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"])


# ---------------------------------------------------------------- 64 bits
def _exact_rows(x, weight, n0, cos, sin, pos, interleaved):
    """Norm and rotation of [tokens, heads, 128] in 64 bits, pairs as complex numbers."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y ** 2).sum(-1, keepdim=True) / D + 1e-6)
        model = (torch.arange(y.shape[0], device=y.device) >= n0).long()
        y = y * weight.double()[model][:, None]
    turn = torch.complex(cos.double(), sin.double())[pos.long()][:, None]
    half = turn.shape[-1]
    idx = torch.arange(2 * half, device=y.device)
    first, second = (idx[0::2], idx[1::2]) if interleaved else (idx[:half], idx[half:])
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
    y = y.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_stored(x, dt):
    """What a 4-bit row stands for, from its definition, in 64 bits."""
    y = x.double().unflatten(-1, (4, 32))
    zero = y.min(-1, keepdim=True).values.to(dt).double()
    scale = ((y.max(-1, keepdim=True).values - zero) / 15).to(dt).double()
    code = torch.clamp(torch.round((y - zero) / torch.where(scale > 0, scale, 1.0)), 0, 15)
    return (scale * code + zero).flatten(-2)


def _exact_cache(st, m, part, seq):
    """Sequence `seq`'s cached rows, [kv, length, 128], byte by byte from the format."""
    pool, n = st["pools"][m], st["lens"][seq]
    codes, meta = pool[part + "_codes"], pool[part + "_meta"]
    if st["table"] is None:
        s = seq - (st["n0"] if m else 0)
        codes, meta = codes[s, :, :n], meta[s, :, :n]
    else:
        at = torch.arange(n, device=codes.device)
        page = st["table"][seq].long()[at // st["page"]]
        codes, meta = (x[page, :, at % st["page"]].transpose(0, 1) for x in (codes, meta))
    channel = torch.arange(D, device=codes.device)
    group, within = channel // 32, channel % 32
    byte = (within // 8) * 16 + group * 4 + (within % 8) // 2
    c = (codes[..., byte].long() >> (4 * (channel % 2))) & 15
    return meta[..., group, 0].double() * c + meta[..., group, 1].double()


def _exact_attention(q, k, v, first):
    """q [heads, n, 128] against k, v [kv, m, 128]; query i sees keys up to first + i."""
    out = []
    group = q.shape[0] // k.shape[0]
    for h in range(q.shape[0]):
        rows = []
        for a in range(0, q.shape[1], 8192):
            s = (q[h, a:a + 8192] @ k[h // group].T) / math.sqrt(D)
            i = torch.arange(a, a + s.shape[0], device=s.device)[:, None] + first
            s = torch.where(torch.arange(s.shape[1], device=s.device) <= i, s, -math.inf)
            rows.append(torch.softmax(s, -1) @ v[h // group])
        out.append(torch.cat(rows))
    return torch.stack(out, 1).flatten(1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm_rope":
        return [_exact_rows(st[x], st["w" + x], st["n0"], st["cos"], st["sin"], st["pos"],
                            st["interleaved"]) for x in ("q", "k")]
    if case["op"] == "write_read":
        q, k = (_exact_rows(st[x], st["w" + x], st["split"], st["cos"], st["sin"], st["pos"], False)
                for x in ("q", "k"))
        return {"q": q, "k": _exact_stored(k, st["dt"]), "v": _exact_stored(st["v"], st["dt"])}
    if case["op"] == "decode":
        out = []
        for j, n in enumerate(st["lens"]):
            m = 0 if j < st["n0"] else 1
            out.append(_exact_attention(st["q"][j].double()[:, None], _exact_cache(st, m, "k", j),
                                        _exact_cache(st, m, "v", j), n - 1))
        return torch.cat(out)
    out, a, b = [], 0, 0
    for n, nk in zip(st["lens"], st["klens"]):
        out.append(_exact_attention(st["q"][a:a + n].double().transpose(0, 1),
                                    st["k"][b:b + nk].double().transpose(0, 1),
                                    st["v"][b:b + nk].double().transpose(0, 1), nk - n))
        a, b = a + n, b + nk
    return torch.cat(out)
