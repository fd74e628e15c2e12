"""numpy restatement of the 4-bit KV cache, head norms and rotation, and the two
attentions around them (test infrastructure only). The reference has none of
these; they are written from their definitions, in 64 bits except where the
stored format itself is defined by 32-bit arithmetic."""
from __future__ import annotations

import numpy as np

from .ref_ops import round16

__all__ = ["kv4_quantize", "kv4_pack", "kv4_unpack", "norm_rope", "grouped_attention"]


def kv4_quantize(x: np.ndarray, kind: str):
    """x [..., 128] (any finite float32 values) -> codes uint8 [..., 4, 32], scale and
    zero [..., 4] (values of the 16-bit type ``kind``, as float32). The steps round
    as the format says: differences and quotients in fp32, (s, z) to 16 bits. A
    difference beyond fp32 is taken of halves, which rounds the same."""
    g = np.asarray(x, np.float32).reshape(*x.shape[:-1], 4, 32)
    top = np.float32(65504.0 if kind == "f16" else 3.3895313892515355e38)
    z = round16(np.clip(g.min(-1), -top, top), kind).astype(np.float32)
    with np.errstate(over="ignore"):
        half = np.where(np.isinf(g.max(-1) - z), np.float32(0.5), np.float32(1))
    s = (g.max(-1) * half - z * half) / np.float32(15) / half
    s = round16(np.clip(s, -top, top), kind).astype(np.float32)
    step, half = np.where(s == 0, np.float32(1), s)[..., None], half[..., None]
    y = (g * half - z[..., None] * half) / (step * half)
    return np.clip(np.rint(y), 0, 15).astype(np.uint8), s, z


def kv4_pack(codes: np.ndarray) -> np.ndarray:
    """codes [..., 4, 32] -> bytes [..., 64]: channel by channel from the layout."""
    out = np.zeros((*codes.shape[:-2], 64), np.uint8)
    for ch in range(128):
        g, i = divmod(ch, 32)
        word = 4 * (i // 8) + g
        out[..., 4 * word + (i % 8) // 2] |= codes[..., g, i] << (4 * (i % 2))
    return out


def kv4_unpack(codes: np.ndarray, meta: np.ndarray) -> np.ndarray:
    """bytes [..., 64] and meta [..., 4, 2] (scale, zero) -> values [..., 128], float64."""
    out = np.zeros((*codes.shape[:-1], 128), np.float64)
    meta = np.asarray(meta, np.float64)
    for ch in range(128):
        g, i = divmod(ch, 32)
        c = (codes[..., 4 * (4 * (i // 8) + g) + (i % 8) // 2] >> (4 * (i % 2))) & 15
        out[..., ch] = meta[..., g, 0] * c + meta[..., g, 1]
    return out


def norm_rope(x, w=None, eps=1e-6, cos=None, sin=None, pos=None, interleaved=False):
    """x [tokens, heads, 128]; w [tokens, 128] (each token's model's weight) or None;
    cos / sin [positions, rotary / 2]."""
    y = np.array(x, np.float64)
    if w is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)[:, None]
    if cos is not None:
        c, s = cos[pos][:, None].astype(np.float64), sin[pos][:, None].astype(np.float64)
        n = c.shape[-1]
        i = np.arange(n)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        ya, yb = y[..., a].copy(), y[..., b].copy()
        y[..., a] = ya * c - yb * s
        y[..., b] = yb * c + ya * s
    return y


def grouped_attention(q, k, v, first=None, scale=None):
    """q [n, heads, 128] against k, v [m, kv heads, 128]; query i sees keys up to
    ``first + i`` (default: the last query sees the last key); a query that sees
    none returns 0. -> out [n, heads, 128] and sum_p p |v| of the same shape."""
    n, h, d = q.shape
    m, kv = k.shape[:2]
    first = m - n if first is None else first
    scale = d ** -0.5 if scale is None else scale
    out, size = np.zeros((n, h, d)), np.zeros((n, h, d))
    seen = np.arange(m)[None] <= np.arange(n)[:, None] + first
    for i in range(h):
        s = np.where(seen, q[:, i] @ k[:, i * kv // h].T * scale, -np.inf)
        top = s.max(-1, keepdims=True) if m else np.full((n, 1), -np.inf)
        p = np.where(seen, np.exp(s - np.where(np.isfinite(top), top, 0)), 0)
        p /= np.maximum(p.sum(-1, keepdims=True), 1e-300)
        out[:, i] = p @ v[:, i * kv // h]
        size[:, i] = p @ np.abs(v[:, i * kv // h])
    return out, size
