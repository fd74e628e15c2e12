"""Thin Python wrappers over the C ABI, one per kernel.

Each wrapper validates shapes / dtypes on the host (raising ``ValueError`` or
``TypeError`` the way the reference's asserts reject bad input,
kernel/src/routed_gemm.py:163-174), allocates outputs through the torch
caching allocator on the input's device, and launches on the current torch
stream with no host synchronisation, so every call is CUDA-graph capturable.
"""
from __future__ import annotations

import ctypes
import math
import struct

import torch

from . import _lib
from ._lib import check, lib, ptr


def _need_cuda(*ts: torch.Tensor) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("parallel-serve ops take CUDA tensors")


def _need_contig(*ts: torch.Tensor) -> None:
    for t in ts:
        if t is not None and not t.is_contiguous():
            raise ValueError("parallel-serve ops take contiguous tensors")


def _counts_arg(counts: torch.Tensor | None) -> int | None:
    if counts is None:
        return None
    if counts.dtype != torch.int32 or counts.numel() < 2 or not counts.is_cuda:
        raise TypeError("counts must be a CUDA int32 tensor of 2 elements")
    return counts.data_ptr()


def route_partition(model_id: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Stable partition of per-token model ids (0/1) -> (perm[M], counts[2]), int32 on device."""
    _need_cuda(model_id)
    if model_id.dtype != torch.int32 or model_id.dim() != 1:
        raise TypeError("model_id must be a 1-D int32 CUDA tensor")
    model_id = model_id.contiguous()
    M = model_id.numel()
    perm = torch.empty(M, dtype=torch.int32, device=model_id.device)
    counts = torch.empty(2, dtype=torch.int32, device=model_id.device)
    check(lib.ps_route_partition(ptr(model_id), M, ptr(perm), ptr(counts),
                                 ptr(_lib.status_tensor(model_id.device)),
                                 _lib.stream_handle(model_id.device)), "ps_route_partition")
    return perm, counts


def gather_rows(src: torch.Tensor, perm: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    _need_cuda(src, perm)
    _need_contig(src, perm)
    M = perm.numel()
    if src.shape[0] != M:
        raise ValueError("gather_rows: src must have one row per perm entry")
    out = torch.empty_like(src) if out is None else out
    row_bytes = src[0].numel() * src.element_size() if M else 16
    check(lib.ps_gather_rows(ptr(src), ptr(perm), ptr(out), M, row_bytes,
                             ptr(_lib.status_tensor(src.device)), _lib.stream_handle(src.device)),
          "ps_gather_rows")
    return out


def scatter_rows(src: torch.Tensor, perm: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    _need_cuda(src, perm)
    _need_contig(src, perm)
    M = perm.numel()
    out = torch.empty_like(src) if out is None else out
    row_bytes = src[0].numel() * src.element_size() if M else 16
    check(lib.ps_scatter_rows(ptr(src), ptr(perm), ptr(out), M, row_bytes,
                              ptr(_lib.status_tensor(src.device)), _lib.stream_handle(src.device)),
          "ps_scatter_rows")
    return out


def gemm_workspace(device: torch.device, M: int, N: int, epilogue: int) -> torch.Tensor:
    idx = torch.device(device).index or 0
    nbytes = lib.ps_routed_gemm_workspace_bytes(M, N, epilogue, idx)
    return _lib.workspace(device, nbytes, "gemm")


def routed_gemm_raw(x: torch.Tensor, W: torch.Tensor, out: torch.Tensor, *, split_point: int = 0,
                    counts: torch.Tensor | None = None, scatter: torch.Tensor | None = None,
                    residual: torch.Tensor | None = None, epilogue: int = _lib.PS_EPI_STORE,
                    workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Launch ps_routed_gemm with every option exposed (no allocation besides workspace)."""
    M, K = x.shape
    N = W.shape[-1]
    ws = workspace if workspace is not None else gemm_workspace(x.device, M, N, epilogue)
    check(lib.ps_routed_gemm(ptr(x), ptr(W), ptr(out), M, K, N, split_point, _counts_arg(counts),
                             ptr(scatter), ptr(residual), epilogue, _lib.dtype_code(x.dtype),
                             ptr(ws), ws.numel(), ptr(_lib.status_tensor(x.device)),
                             _lib.stream_handle(x.device)), "ps_routed_gemm")
    return out


def gemm_epilogue(mode: int = _lib.PS_EPI_STORE, *, scatter: torch.Tensor | None = None,
                  residual: torch.Tensor | None = None, in_sumsq: torch.Tensor | None = None,
                  norm_dim: int = 0, eps: float = 0.0, out_sumsq: torch.Tensor | None = None,
                  k_pools: tuple = (None, None),
                  v_pools: tuple = (None, None), pos: torch.Tensor | None = None,
                  rope_cos: torch.Tensor | None = None, rope_sin: torch.Tensor | None = None,
                  n_heads: int = 0, block_table: torch.Tensor | None = None,
                  kv_rows: torch.Tensor | None = None,
                  max_model_rows: int = 0, max_ctas: int = 0) -> _lib.GemmEpilogue:
    """Build a ps_gemm_epilogue_t. ``in_sumsq`` is [rows, parts] fp32 (partial sums
    of squares of x's rows). The descriptor holds references to every tensor
    it points to, so they live at least as long as the descriptor."""
    e = _lib.GemmEpilogue()
    e._keep = (scatter, residual, in_sumsq, out_sumsq, k_pools, v_pools, pos, rope_cos, rope_sin,
               block_table, kv_rows)
    e.mode = mode
    e.scatter_rows, e.residual = ptr(scatter), ptr(residual)
    e.in_sumsq, e.norm_dim, e.eps = ptr(in_sumsq), int(norm_dim), float(eps)
    e.in_parts = 0 if in_sumsq is None else (in_sumsq.shape[-1] if in_sumsq.dim() > 1 else 1)
    e.out_sumsq = ptr(out_sumsq)
    e.max_model_rows = int(max_model_rows)
    e.max_ctas = int(max_ctas)
    if mode == _lib.PS_EPI_QKV_ROPE:
        k0, k1, v0, v1, L_cap, s0, s1 = _pool_args(k_pools, v_pools, n_heads)
        e.k_pool0, e.v_pool0, e.k_pool1, e.v_pool1 = ptr(k0), ptr(v0), ptr(k1), ptr(v1)
        e.pos, e.rope_cos, e.rope_sin = ptr(pos), ptr(rope_cos), ptr(rope_sin)
        e.n_heads, e.L_cap, e.slots0, e.slots1 = n_heads, L_cap, s0, s1
        e.apply_rope = 1 if rope_cos is not None else 0
        if block_table is not None:     # page pools: [pages, n_heads, page_size, 128]
            if block_table.dtype != torch.int32 or block_table.dim() != 2:
                raise ValueError("block_table must be int32 [M, max_pages]")
            e.block_table, e.max_pages, e.page_size = ptr(block_table), block_table.shape[1], L_cap
            e.table_rows = block_table.shape[0]
        e.kv_rows = ptr(kv_rows)
    return e


def routed_gemm_ex(x: torch.Tensor, W: torch.Tensor, out: torch.Tensor,
                   epi: _lib.GemmEpilogue, *, split_point: int = 0,
                   counts: torch.Tensor | None = None,
                   workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Launch ps_routed_gemm_ex (routed GEMM + fused decode-layer epilogue)."""
    M, K = x.shape
    N = W.shape[-1]
    ws = workspace if workspace is not None else gemm_workspace(
        x.device, M, N, 1 if epi.mode == _lib.PS_EPI_SWIGLU else 0)
    check(lib.ps_routed_gemm_ex(ptr(x), ptr(W), ptr(out), M, K, N, split_point,
                                _counts_arg(counts), ctypes.byref(epi), _lib.dtype_code(x.dtype),
                                ptr(ws), ws.numel(), ptr(_lib.status_tensor(x.device)),
                                _lib.stream_handle(x.device)), "ps_routed_gemm_ex")
    return out


def rmsnorm_routed(x: torch.Tensor, w: torch.Tensor, *, split_point: int = 0,
                   counts: torch.Tensor | None = None, eps: float | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Per-model RMSNorm. ``w`` is [2, H] (or [1, H] when every row is model 0).

    ``eps=None`` follows F.rms_norm: the machine epsilon of x's dtype.
    """
    _need_cuda(x, w)
    _need_contig(x, w)
    M, H = x.shape
    if eps is None:
        eps = torch.finfo(x.dtype).eps
    out = torch.empty_like(x) if out is None else out
    check(lib.ps_rmsnorm_routed(ptr(x), ptr(w), ptr(out), M, H, split_point, _counts_arg(counts),
                                float(eps), _lib.dtype_code(x.dtype),
                                ptr(_lib.status_tensor(x.device)), _lib.stream_handle(x.device)),
          "ps_rmsnorm_routed")
    return out


def swiglu(gu: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    _need_cuda(gu)
    _need_contig(gu)
    M, N2 = gu.shape
    FF = N2 // 2
    out = torch.empty(M, FF, dtype=gu.dtype, device=gu.device) if out is None else out
    check(lib.ps_swiglu(ptr(gu), ptr(out), M, FF, _lib.dtype_code(gu.dtype),
                        _lib.stream_handle(gu.device)), "ps_swiglu")
    return out


def segment_attention(qkv: torch.Tensor, n_heads: int, *, split_point: int = 0,
                      counts: torch.Tensor | None = None, out: torch.Tensor | None = None,
                      scale: float | None = None) -> torch.Tensor:
    """Reference no-KV attention: each token attends to its own model's segment."""
    _need_cuda(qkv)
    _need_contig(qkv)
    M, H3 = qkv.shape
    H = H3 // 3
    if H != n_heads * 128:
        raise ValueError("segment_attention supports head_dim 128 only")
    scale = 1.0 / math.sqrt(128) if scale is None else scale
    out = torch.empty(M, H, dtype=qkv.dtype, device=qkv.device) if out is None else out
    check(lib.ps_segment_attention(ptr(qkv), ptr(out), M, n_heads, split_point, _counts_arg(counts),
                                   float(scale), _lib.dtype_code(qkv.dtype),
                                   ptr(_lib.status_tensor(qkv.device)),
                                   _lib.stream_handle(qkv.device)), "ps_segment_attention")
    return out


def _pool_args(k_pools, v_pools, n_heads: int):
    """Validate the two models' K / V pools [slots, n_heads, L_cap, 128] (same
    L_cap, dtype and device; a model without slots passes None)."""
    k0, k1 = k_pools
    v0, v1 = v_pools
    live = [t for t in (k0, k1, v0, v1) if t is not None]
    if not live:
        raise ValueError("at least one model needs a KV pool")
    L_cap = live[0].shape[2]
    for t in live:
        if t.dim() != 4 or t.shape[1] != n_heads or t.shape[2] != L_cap or t.shape[3] != 128:
            raise ValueError("KV pools must be [slots, n_heads, L_cap, 128] with one L_cap")
        if not (t.is_cuda and t.is_contiguous()):
            raise ValueError("KV pools must be contiguous CUDA tensors")
    if (k0 is None) != (v0 is None) or (k1 is None) != (v1 is None):
        raise ValueError("each model needs both a K and a V pool (or neither)")
    s0 = 0 if k0 is None else k0.shape[0]
    s1 = 0 if k1 is None else k1.shape[0]
    if k0 is not None and v0.shape != k0.shape or k1 is not None and v1.shape != k1.shape:
        raise ValueError("K and V pools of a model must have the same shape")
    return k0, k1, v0, v1, L_cap, s0, s1


def rope_tables(max_pos: int, head_dim: int = 128, theta: float = 10000.0,
                device: torch.device | str = "cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """cos / sin tables [max_pos, head_dim/2] (fp32), rotate-half convention.

    angle[p, i] = p * theta^(-2i/head_dim), evaluated in float64 then rounded.
    """
    i = torch.arange(head_dim // 2, dtype=torch.float64)
    inv = theta ** (-2.0 * i / head_dim)
    ang = torch.arange(max_pos, dtype=torch.float64)[:, None] * inv[None, :]
    return (ang.cos().to(torch.float32).to(device).contiguous(),
            ang.sin().to(torch.float32).to(device).contiguous())


def rope_kv_append(qkv: torch.Tensor, q_out: torch.Tensor, k_pools: tuple, v_pools: tuple,
                   rope_cos: torch.Tensor | None, rope_sin: torch.Tensor | None,
                   pos: torch.Tensor, *, n_heads: int, split_point: int = 0,
                   counts: torch.Tensor | None = None, slot: torch.Tensor | None = None) -> None:
    """RoPE q and the new k, append k / v to the token's model pool at pos[j].

    Pools are [slots, n_heads, L_cap, 128]; ``k_pools = (k_pool_model0, k_pool_model1)``,
    either may be None when that model has no slots.
    """
    M = qkv.shape[0]
    k0, k1, v0, v1, L_cap, s0, s1 = _pool_args(k_pools, v_pools, n_heads)
    apply = rope_cos is not None
    check(lib.ps_rope_kv_append(ptr(qkv), ptr(q_out), ptr(k0), ptr(v0), ptr(k1), ptr(v1),
                                ptr(rope_cos), ptr(rope_sin), ptr(pos), ptr(slot),
                                _counts_arg(counts), split_point, M, n_heads, L_cap, s0, s1,
                                1 if apply else 0, _lib.dtype_code(qkv.dtype),
                                ptr(_lib.status_tensor(qkv.device)),
                                _lib.stream_handle(qkv.device)), "ps_rope_kv_append")


def attention_workspace(device: torch.device, M: int, n_heads: int, max_len: int,
                        chunk: int = 0) -> torch.Tensor:
    with torch.cuda.device(device):
        nbytes = lib.ps_decode_attention_workspace_bytes(M, n_heads, max_len, chunk)
    return _lib.workspace(device, nbytes, "attn")


def decode_attention(q: torch.Tensor, k_pools: tuple, v_pools: tuple, pos: torch.Tensor, *,
                     n_heads: int, max_len: int, split_point: int = 0,
                     counts: torch.Tensor | None = None, slot: torch.Tensor | None = None,
                     out: torch.Tensor | None = None, chunk: int = 0,
                     scale: float | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Two-model decode attention over the models' KV pools (positions 0..pos[j])."""
    M = q.shape[0]
    k0, k1, v0, v1, L_cap, s0, s1 = _pool_args(k_pools, v_pools, n_heads)
    scale = 1.0 / math.sqrt(128) if scale is None else scale
    out = torch.empty(M, n_heads * 128, dtype=q.dtype, device=q.device) if out is None else out
    ws = workspace if workspace is not None else attention_workspace(q.device, M, n_heads, max_len, chunk)
    check(lib.ps_decode_attention(ptr(q), ptr(k0), ptr(v0), ptr(k1), ptr(v1), ptr(out), ptr(pos),
                                  ptr(slot), _counts_arg(counts), split_point, M, n_heads, L_cap,
                                  s0, s1, max_len, chunk, float(scale), _lib.dtype_code(q.dtype),
                                  ptr(ws), ws.numel(), ptr(_lib.status_tensor(q.device)),
                                  _lib.stream_handle(q.device)), "ps_decode_attention")
    return out


def paged_attention_workspace(device: torch.device, M: int, n_heads: int, max_len: int,
                              page_size: int, chunk: int = 0) -> torch.Tensor:
    with torch.cuda.device(device):
        nbytes = lib.ps_paged_decode_attention_workspace_bytes(M, n_heads, max_len, chunk,
                                                               page_size)
    return _lib.workspace(device, nbytes, "attn")


def paged_decode_attention(q: torch.Tensor, k_pages: tuple, v_pages: tuple, pos: torch.Tensor,
                           block_table: torch.Tensor, *, n_heads: int, max_len: int,
                           seq_rows: torch.Tensor | None = None,
                           split_point: int = 0, counts: torch.Tensor | None = None,
                           out: torch.Tensor | None = None, chunk: int = 0,
                           scale: float | None = None,
                           workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Decode attention over paged KV: pools ``[pages, n_heads, page_size, 128]`` per
    model, ``block_table`` int32 ``[M, max_pages]`` (routed rows) of page ids."""
    M = q.shape[0]
    k0, k1, v0, v1, page_size, p0, p1 = _pool_args(k_pages, v_pages, n_heads)
    if block_table.dtype != torch.int32 or block_table.dim() != 2:
        raise ValueError("block_table must be int32 [rows, max_pages]")
    if seq_rows is None and block_table.shape[0] < M:
        raise ValueError("block_table needs a row per token when seq_rows is not given")
    if not block_table.is_contiguous():
        raise ValueError("block_table must be contiguous")
    scale = 1.0 / math.sqrt(128) if scale is None else scale
    out = torch.empty(M, n_heads * 128, dtype=q.dtype, device=q.device) if out is None else out
    ws = workspace if workspace is not None else paged_attention_workspace(
        q.device, M, n_heads, max_len, page_size, chunk)
    check(lib.ps_paged_decode_attention(ptr(q), ptr(k0), ptr(v0), ptr(k1), ptr(v1), ptr(out),
                                        ptr(pos), ptr(block_table), block_table.shape[0],
                                        ptr(seq_rows), block_table.shape[1],
                                        page_size, _counts_arg(counts), split_point, M, n_heads,
                                        p0, p1, max_len, chunk, float(scale),
                                        _lib.dtype_code(q.dtype), ptr(ws), ws.numel(),
                                        ptr(_lib.status_tensor(q.device)),
                                        _lib.stream_handle(q.device)), "ps_paged_decode_attention")
    return out


def prefill_attention(q: torch.Tensor, k_pools: tuple, v_pools: tuple, blocks: torch.Tensor, *,
                      n_heads: int, out: torch.Tensor | None = None,
                      scale: float | None = None,
                      block_table: torch.Tensor | None = None) -> torch.Tensor:
    """Causal prefill attention on the tensor cores over the KV pools.
    ``blocks`` int32 [nblocks, 5] = (row0, nq <= 128, p0, model, slot): rows
    row0.. of q are prompt tokens at positions p0.. of that sequence. With
    ``block_table`` [rows, max_pages] the pools are page pools and `slot` is the
    sequence's block-table row."""
    T = q.shape[0]
    k0, k1, v0, v1, L_cap, s0, s1 = _pool_args(k_pools, v_pools, n_heads)
    bt_rows = max_pages = page_size = 0
    if block_table is not None:
        page_size, max_pages = L_cap, block_table.shape[1]
        bt_rows, L_cap = block_table.shape[0], max_pages * page_size
    if blocks.dtype != torch.int32 or blocks.dim() != 2 or blocks.shape[1] != 5:
        raise ValueError("blocks must be int32 [nblocks, 5]")
    scale = 1.0 / math.sqrt(128) if scale is None else scale
    out = torch.empty(T, n_heads * 128, dtype=q.dtype, device=q.device) if out is None else out
    check(lib.ps_prefill_attention(ptr(q), ptr(k0), ptr(v0), ptr(k1), ptr(v1), ptr(out),
                                   ptr(blocks.contiguous()), blocks.shape[0], T, n_heads, L_cap,
                                   s0, s1, ptr(block_table), bt_rows, max_pages, page_size,
                                   float(scale), _lib.dtype_code(q.dtype),
                                   ptr(_lib.status_tensor(q.device)),
                                   _lib.stream_handle(q.device)), "ps_prefill_attention")
    return out


def embed_routed(emb: torch.Tensor, tokens: torch.Tensor, perm: torch.Tensor | None,
                 counts: torch.Tensor | None, out: torch.Tensor, *,
                 out_sumsq: torch.Tensor | None = None) -> torch.Tensor:
    """out[j] = emb[m(j)][tokens[perm[j]]]; emb [2, vocab, H]. Optionally
    out_sumsq[j] = sum(out[j]^2) (fp32)."""
    M, H = out.shape
    vocab = emb.shape[1]
    check(lib.ps_embed_routed(ptr(emb), ptr(tokens), ptr(perm), _counts_arg(counts), ptr(out), M, H,
                              vocab, ptr(out_sumsq), _lib.dtype_code(emb.dtype),
                              ptr(_lib.status_tensor(emb.device)),
                              _lib.stream_handle(emb.device)), "ps_embed_routed")
    return out


def argmax_rows(logits: torch.Tensor, perm: torch.Tensor | None, next_tokens: torch.Tensor,
                seq_len: torch.Tensor | None = None) -> torch.Tensor:
    M, V = logits.shape
    check(lib.ps_argmax_rows(ptr(logits), ptr(perm), ptr(next_tokens), ptr(seq_len), M, V,
                             _lib.dtype_code(logits.dtype), _lib.stream_handle(logits.device)),
          "ps_argmax_rows")
    return next_tokens


def positions_routed(seq_len: torch.Tensor, perm: torch.Tensor | None, out: torch.Tensor) -> torch.Tensor:
    check(lib.ps_positions_routed(ptr(seq_len), ptr(perm), ptr(out), out.numel(),
                                  _lib.stream_handle(seq_len.device)), "ps_positions_routed")
    return out


# ---------------------------------------------------------------- 4-bit KV cache, head norms
#
# These calls follow one another every few microseconds in a decode step, so
# their host side is kept short: plain comparisons, no keyword dictionaries, and
# descriptors packed as bytes.

_HD = 128
_CACHE = struct.Struct("=4Qi4x4Qi4xQ5i4x")       # ps_kv4_cache_t
_POOL_SHAPE = ("a 4-bit pool is codes [rows, n_kv_heads, length, 64] and meta [rows, n_kv_heads, "
               "length, 4, 2], for K and for V")
_U8, _DENSE = torch.uint8, torch.contiguous_format
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _heads(t: torch.Tensor, name: str) -> tuple[int, int, int]:
    """(tokens, heads, token stride) of ``[tokens, heads, 128]`` or ``[tokens,
    heads * 128]`` whose heads lie one after another (views of a qkv row do)."""
    sh, st = t.shape, t.stride()
    if len(sh) == 3:
        n, h, d = sh
        ok = d == _HD and st[2] == 1 and (h == 1 or st[1] == _HD)
    elif len(sh) == 2:
        n, d = sh
        h = d // _HD
        ok = d % _HD == 0 and st[1] == 1
    else:
        ok = False
    if not ok or h == 0:
        raise ValueError(f"{name} must be [tokens, heads, 128] (or [tokens, heads * 128]) with "
                         "contiguous heads")
    stride = st[0] if n > 1 else h * _HD
    if stride < h * _HD or stride % 8:
        raise ValueError(f"{name}: token stride {stride} must be a multiple of 8 and hold every head")
    return n, h, stride


def _int32(t: torch.Tensor | None, name: str, n: int, idx: int) -> int | None:
    """Pointer of a contiguous int32 tensor of at least n entries (None stays None)."""
    if t is None:
        return None
    if t.dtype != torch.int32 or t.get_device() != idx or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor on cuda:{idx}")
    if t.numel() < n:
        raise ValueError(f"{name} needs {n} entries, has {t.numel()}")
    return t.data_ptr()


def _on(t: torch.Tensor, name: str, idx: int, dtype: torch.dtype) -> None:
    if t.get_device() != idx:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{idx}")
    if t.dtype != dtype:
        raise TypeError(f"{name} is {t.dtype}, expected {dtype}")


def _first(t: torch.Tensor) -> tuple[int, int]:
    """(device index, dtype code) that the other tensors of a call have to match."""
    idx = t.get_device()
    if idx < 0:
        raise ValueError("parallel-serve ops take CUDA tensors")
    return idx, _lib.dtype_code(t.dtype)


def _head_weight(w: torch.Tensor | None, name: str, idx: int, dtype: torch.dtype) -> int | None:
    if w is None:
        return None
    _on(w, name, idx, dtype)
    if w.shape != (2, _HD) or not w.is_contiguous():
        raise ValueError(f"{name} must be contiguous [2, 128] (one row per model)")
    return w.data_ptr()


def _rope_args(cos, sin, idx: int) -> tuple:
    """(cos, sin pointers, positions, rotary_dim) of the rotation tables."""
    if cos is None and sin is None:
        return None, None, 0, 0
    if cos is None or sin is None:
        raise ValueError("rope_cos and rope_sin come together")
    _on(cos, "rope_cos", idx, torch.float32)
    _on(sin, "rope_sin", idx, torch.float32)
    sh = cos.shape
    if len(sh) != 2 or sh != sin.shape or not (cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError("rope tables must be contiguous [positions, rotary_dim / 2]")
    n, rotary = sh[0], 2 * sh[1]
    if rotary % 16 or not 0 < rotary <= _HD or n == 0:
        raise ValueError("rotary_dim must be a multiple of 16 up to 128, with at least one position")
    return cos.data_ptr(), sin.data_ptr(), n, rotary


def _split_counts(split_point: int | None, counts: torch.Tensor | None, M: int,
                  idx: int) -> tuple[int, int | None]:
    """(split point, counts pointer); neither given: every token is model 0's."""
    if counts is not None:
        return 0, _int32(counts, "counts", 2, idx)
    if split_point is None:
        return M, None
    if not 0 <= split_point <= M:
        raise ValueError(f"split_point must be in [0, {M}]")
    return split_point, None


def _call(fn, what: str, idx: int, *args) -> None:
    """Launch on the tensors' device (made current for the call when it is not),
    on its current torch stream, with its status word."""
    if _current_device() == idx:
        rc = fn(*args, _lib.status_ptr(idx), _raw_stream(idx))
    else:
        with torch.cuda.device(idx):
            rc = fn(*args, _lib.status_ptr(idx), _raw_stream(idx))
    if rc:
        check(rc, what)


def _kv4_cache(pools, block_table: torch.Tensor | None, idx: int,
               dtype: torch.dtype) -> tuple[bytes, int, int]:
    """Both models' 4-bit pools (``KV4Pool`` or None) and the block table, checked:
    (ps_kv4_cache_t as bytes, KV heads, positions a sequence can have)."""
    if len(pools) != 2:
        raise ValueError("pools are (model 0's, model 1's), either may be None")
    n_kv = length = 0
    desc = []
    for p in pools:
        if p is None:
            desc += (0, 0, 0, 0, 0)
            continue
        kc, km, vc, vm = p
        sh = kc.shape
        if len(sh) != 4:
            raise ValueError(_POOL_SHAPE)
        rows, heads, n, code_bytes = sh
        if rows == 0:
            desc += (0, 0, 0, 0, 0)
            continue
        ms = (rows, heads, n, 4, 2)
        if code_bytes != 64 or vc.shape != sh or km.shape != ms or vm.shape != ms:
            raise ValueError(_POOL_SHAPE)
        if kc.dtype is not _U8 or vc.dtype is not _U8 or km.dtype is not dtype or \
                vm.dtype is not dtype:
            raise TypeError(f"a 4-bit pool holds uint8 codes and {dtype} meta here")
        if not (kc.get_device() == km.get_device() == vc.get_device() == vm.get_device() == idx
                and kc.is_contiguous() and km.is_contiguous() and vc.is_contiguous()
                and vm.is_contiguous()):
            raise ValueError(f"4-bit pools must be contiguous tensors on cuda:{idx}")
        if n_kv and (n_kv != heads or length != n):
            raise ValueError("both models' pools must have the same heads and length")
        n_kv, length = heads, n
        desc += (kc.data_ptr(), km.data_ptr(), vc.data_ptr(), vm.data_ptr(), rows)
    if not n_kv or not length:
        raise ValueError("at least one model needs a 4-bit pool")
    if block_table is None:
        return _CACHE.pack(*desc, 0, n_kv, length, 0, 0, 0), n_kv, length
    sh = block_table.shape
    if len(sh) != 2 or not sh[0] or not sh[1]:
        raise ValueError("block_table must be int32 [rows, max_pages]")
    if length < 8 or length > 4096 or length & (length - 1):
        raise ValueError("page_size must be a power of two in [8, 4096]")
    return (_CACHE.pack(*desc, _int32(block_table, "block_table", 1, idx), n_kv, 0, length, sh[1],
                        sh[0]), n_kv, sh[1] * length)


def _home_arg(rows, block_table, M: int, idx: int) -> int | None:
    """Pointer of the tokens' cache rows; without them a table needs a row per token."""
    if rows is None and block_table is not None and block_table.shape[0] < M:
        raise ValueError("block_table needs a row per token when rows is not given")
    return _int32(rows, "rows", M, idx)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, pos: torch.Tensor, *,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                 eps: float = 1e-6, rope_cos: torch.Tensor | None = None,
                 rope_sin: torch.Tensor | None = None, interleaved: bool = False,
                 split_point: int | None = None, counts: torch.Tensor | None = None,
                 q_out: torch.Tensor | None = None,
                 k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """RMSNorm of every q and k head and the position rotation, in one pass.

    ``q`` [tokens, n_heads, 128] and ``k`` [tokens, n_kv_heads, 128] may be views
    of one qkv row. ``q_weight`` / ``k_weight`` [2, 128] (one row per model;
    None: that norm is left out); ``rope_cos`` / ``rope_sin`` [positions,
    rotary_dim / 2] fp32 (``rope_tables``; None: no rotation) turn the first
    rotary_dim channels, as pairs (i, i + rotary_dim / 2), or (2i, 2i + 1) when
    ``interleaved``. Tokens are in routed order: the first ``split_point`` (or
    counts[0], read on the device; default: all) belong to model 0.
    ``q_out`` may be ``q`` itself and ``k_out`` ``k``; they overlap the inputs in no other
    way. A position outside the tables raises PS_ERR_BAD_INDEX in the status word and leaves its rows unwritten.
    """
    idx, code = _first(q)
    dt = q.dtype
    M, nh, qs = _heads(q, "q")
    Mk, nkv, ks = _heads(k, "k")
    _on(k, "k", idx, dt)
    if Mk != M:
        raise ValueError("q and k must have the same tokens")
    if q_out is None:
        q_out, qos = torch.empty_like(q, memory_format=_DENSE), nh * _HD
    else:
        _on(q_out, "q_out", idx, dt)
        n, h, qos = _heads(q_out, "q_out")
        if (n, h) != (M, nh):
            raise ValueError("q_out must have the shape of q")
    if k_out is None:
        k_out, kos = torch.empty_like(k, memory_format=_DENSE), nkv * _HD
    else:
        _on(k_out, "k_out", idx, dt)
        n, h, kos = _heads(k_out, "k_out")
        if (n, h) != (M, nkv):
            raise ValueError("k_out must have the shape of k")
    rc, rs, rope_len, rotary = _rope_args(rope_cos, rope_sin, idx)
    split, cnt = _split_counts(split_point, counts, M, idx)
    _call(lib.ps_qk_norm_rope, "ps_qk_norm_rope", idx, q.data_ptr(), qs, k.data_ptr(), ks,
          q_out.data_ptr(), qos, k_out.data_ptr(), kos, _head_weight(q_weight, "q_weight", idx, dt),
          _head_weight(k_weight, "k_weight", idx, dt), eps, rc, rs, rope_len, rotary,
          1 if interleaved else 0, _int32(pos, "pos", M, idx), cnt, split, M, nh, nkv, code)
    return q_out, k_out


def kv4_append(k: torch.Tensor, v: torch.Tensor, pools: tuple, pos: torch.Tensor, *,
               q: torch.Tensor | None = None, q_weight: torch.Tensor | None = None,
               k_weight: torch.Tensor | None = None, eps: float = 1e-6,
               rope_cos: torch.Tensor | None = None, rope_sin: torch.Tensor | None = None,
               interleaved: bool = False, rows: torch.Tensor | None = None,
               block_table: torch.Tensor | None = None, split_point: int | None = None,
               counts: torch.Tensor | None = None,
               q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Quantise the tokens' k and v into the 4-bit cache at positions ``pos``.

    ``pools`` = (model 0's ``KV4Pool``, model 1's), either None. Token j goes to
    its model's slot ``rows[j]`` (default: its rank within its model), or with
    ``block_table`` [rows, max_pages] to the pages of table row ``rows[j]``
    (default: j). Norms and rotation as in ``qk_norm_rope`` (all optional) happen
    in the same pass: k is quantised from their fp32 result, ``q`` (optional)
    returns in 16 bits (``q_out`` may be ``q`` itself). Two tokens of a call must not
    share a position of a sequence. Returns q_out, or None without ``q``.
    """
    idx, code = _first(k)
    dt = k.dtype
    M, nkv, ks = _heads(k, "k")
    Mv, nv, vs = _heads(v, "v")
    _on(v, "v", idx, dt)
    if (Mv, nv) != (M, nkv):
        raise ValueError("k and v must have the same shape")
    cache, n, _ = _kv4_cache(pools, block_table, idx, dt)
    if n != nkv:
        raise ValueError(f"k has {nkv} heads, the pools {n}")
    nh = qs = qos = 0
    qp = qop = None
    if q is not None:
        _on(q, "q", idx, dt)
        Mq, nh, qs = _heads(q, "q")
        if Mq != M:
            raise ValueError("q must have one row per token of k")
        if q_out is None:
            q_out, qos = torch.empty_like(q, memory_format=_DENSE), nh * _HD
        else:
            _on(q_out, "q_out", idx, dt)
            n, h, qos = _heads(q_out, "q_out")
            if (n, h) != (M, nh):
                raise ValueError("q_out must have the shape of q")
        qp, qop = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out needs q")
    rc, rs, rope_len, rotary = _rope_args(rope_cos, rope_sin, idx)
    split, cnt = _split_counts(split_point, counts, M, idx)
    _call(lib.ps_kv4_append, "ps_kv4_append", idx, qp, qs, k.data_ptr(), ks, v.data_ptr(), vs, qop,
          qos, cache, _head_weight(q_weight, "q_weight", idx, dt),
          _head_weight(k_weight, "k_weight", idx, dt), eps, rc, rs, rope_len, rotary,
          1 if interleaved else 0, _int32(pos, "pos", M, idx),
          _home_arg(rows, block_table, M, idx), cnt, split, M, nh, code)
    return q_out


def kv4_gather(pools: tuple, seqs: torch.Tensor, cu: torch.Tensor, total: int, *,
               block_table: torch.Tensor | None = None,
               out: tuple[torch.Tensor, torch.Tensor] | None = None
               ) -> tuple[torch.Tensor, torch.Tensor]:
    """Read cached rows back in 16 bits, packed: (k, v) [total, n_kv_heads, 128].

    Sequence i (``seqs`` int32 [n, 3]: model, slot or block-table row, first
    position) fills rows ``cu[i]`` to ``cu[i + 1]`` (``cu`` int32 [n + 1] on the
    device). Rows of no sequence are left as ``out`` had them; without ``out`` they hold
    whatever the memory did.
    """
    if len(pools) != 2:
        raise ValueError("pools are (model 0's, model 1's), either may be None")
    p = pools[0] if pools[0] is not None and pools[0][0].shape[0] else pools[1]
    if p is None:
        raise ValueError("at least one model needs a 4-bit pool")
    meta = p[1]
    idx, code = _first(meta)
    dt = meta.dtype
    cache, nkv, _ = _kv4_cache(pools, block_table, idx, dt)
    sh = seqs.shape
    if len(sh) != 2 or sh[1] != 3:
        raise ValueError("seqs must be int32 [n, 3] (model, slot or block-table row, first position)")
    n = sh[0]
    if total < 0:
        raise ValueError("total must be >= 0")
    if out is None:
        k, v = meta.new_empty((total, nkv, _HD)), meta.new_empty((total, nkv, _HD))
    else:
        k, v = out
        for t in out:
            _on(t, "out", idx, dt)
            if t.shape != (total, nkv, _HD) or not t.is_contiguous():
                raise ValueError("out must be two contiguous [total, n_kv_heads, 128] tensors")
    _call(lib.ps_kv4_gather, "ps_kv4_gather", idx, cache, _int32(seqs, "seqs", 3 * n, idx),
          _int32(cu, "cu", n + 1, idx), n, total, k.data_ptr(), v.data_ptr(), code)
    return k, v


def _counter_workspace(like: torch.Tensor, idx: int, nbytes: int, tag: str,
                       counter_bytes: int) -> torch.Tensor:
    """Workspace whose first ``counter_bytes`` are zero at rest. Under graph capture
    (of device idx's current stream, whichever device is current) a workspace of
    the graph's own (two captured graphs may run at the same time), else the stream's."""
    if _current_device() != idx:
        with torch.cuda.device(idx):
            return _counter_workspace(like, idx, nbytes, tag, counter_bytes)
    if torch.cuda.is_current_stream_capturing():
        ws = like.new_empty(nbytes, dtype=torch.uint8)
        ws[:counter_bytes].zero_()
        return ws
    return _lib.stream_workspace(idx, _raw_stream(idx), nbytes, tag)


def kv4_decode_attention(q: torch.Tensor, pools: tuple, pos: torch.Tensor, *, max_len: int,
                         rows: torch.Tensor | None = None,
                         block_table: torch.Tensor | None = None,
                         split_point: int | None = None, counts: torch.Tensor | None = None,
                         out: torch.Tensor | None = None, scale: float | None = None,
                         workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Decode attention over the 4-bit cache: token j sees positions 0..pos[j] of
    its sequence; query head h reads KV head h // (n_heads / n_kv_heads).

    ``q`` [M, n_heads, 128] (or [M, n_heads * 128]); ``rows``, ``block_table``,
    ``split_point`` and ``counts`` as in ``kv4_append``; ``max_len`` bounds
    pos[j] + 1. ``workspace`` (default: the stream's own) has
    ps_kv4_decode_attention_workspace_bytes bytes, the first 4096 zero before its
    first use; without one, a call that is captured into a graph zeroes its own (one
    launch more a replay). ``scale`` is any finite number below 2e38 in magnitude
    (default: 128^-1/2). Returns [M, n_heads * 128].
    """
    idx, code = _first(q)
    dt = q.dtype
    M, nh, qs = _heads(q, "q")
    cache, nkv, cap = _kv4_cache(pools, block_table, idx, dt)
    if nh % nkv:
        raise ValueError(f"{nh} query heads do not divide over {nkv} KV heads")
    if not 0 < max_len <= cap:
        raise ValueError(f"max_len must be in [1, {cap}]")
    if scale is None:
        scale = 0.08838834764831845
    elif not -2e38 < scale < 2e38:
        raise ValueError("scale must be finite, its magnitude below 2e38")
    if out is None:
        out = q.new_empty((M, nh * _HD))
    else:
        _on(out, "out", idx, dt)
        if out.shape != (M, nh * _HD) or not out.is_contiguous():
            raise ValueError("out must be contiguous [M, n_heads * 128]")
    split, cnt = _split_counts(split_point, counts, M, idx)
    pp, home = _int32(pos, "pos", M, idx), _home_arg(rows, block_table, M, idx)
    if workspace is None:
        if _current_device() == idx:
            nbytes = lib.ps_kv4_decode_attention_workspace_bytes(M, nh, nkv, max_len)
        else:
            with torch.cuda.device(idx):
                nbytes = lib.ps_kv4_decode_attention_workspace_bytes(M, nh, nkv, max_len)
        workspace = _counter_workspace(q, idx, nbytes, "kv4_attn", 4096)
    elif workspace.get_device() != idx or not workspace.is_contiguous():
        raise ValueError(f"workspace must be a contiguous tensor on cuda:{idx}")
    _call(lib.ps_kv4_decode_attention, "ps_kv4_decode_attention", idx, q.data_ptr(), qs, cache,
          out.data_ptr(), pp, home, cnt, split, M, nh, max_len,
          scale, code, workspace.data_ptr(), workspace.nbytes)
    return out


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor,
                     cu_k: torch.Tensor | None = None, *, scale: float | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention over packed prompts of different lengths, grouped heads.

    Sequence i's queries are rows ``cu_q[i]`` to ``cu_q[i + 1]`` of ``q`` [tokens,
    n_heads, 128], its keys and values rows ``cu_k[i]`` to ``cu_k[i + 1]`` (default:
    the same rows) of ``k``, ``v`` [keys, n_kv_heads, 128]; the last query sees every
    key, so keys that precede the queries are their history. A query that sees
    no key gets 0. q, k, v may be views of one qkv row. ``cu_q``, ``cu_k`` are int32
    on the device. Rows outside every sequence are left as ``out`` had them (without
    ``out`` they hold whatever the memory did); ``out`` overlaps no input. ``scale`` is
    positive and below 2e38 (default: 128^-1/2). Returns [tokens, n_heads * 128].
    """
    idx, code = _first(q)
    dt = q.dtype
    Tq, nh, qs = _heads(q, "q")
    Tk, nkv, ks = _heads(k, "k")
    Tv, nv, vs = _heads(v, "v")
    _on(k, "k", idx, dt)
    _on(v, "v", idx, dt)
    if (Tv, nv) != (Tk, nkv):
        raise ValueError("k and v must have the same shape")
    if nh % nkv:
        raise ValueError(f"{nh} query heads do not divide over {nkv} KV heads")
    n = cu_q.numel() - 1
    if n < 0:
        raise ValueError("cu_q needs at least one entry")
    if cu_k is None:
        if Tk != Tq:
            raise ValueError("without cu_k, k must have one row per query")
        cu_k = cu_q
    elif cu_k.numel() != n + 1:
        raise ValueError("cu_q and cu_k must have the same length")
    if scale is None:
        scale = 0.08838834764831845
    elif not 0.0 < scale < 2e38:
        raise ValueError("scale must be positive and below 2e38")
    if out is None:
        out, os_ = q.new_empty((Tq, nh * _HD)), nh * _HD
    else:
        _on(out, "out", idx, dt)
        To, no, os_ = _heads(out, "out")
        if (To, no) != (Tq, nh):
            raise ValueError("out must have a row of n_heads * 128 per query")
    _call(lib.ps_prompt_attention, "ps_prompt_attention", idx, q.data_ptr(), qs, k.data_ptr(), ks,
          v.data_ptr(), vs, out.data_ptr(), os_, _int32(cu_q, "cu_q", 1, idx),
          _int32(cu_k, "cu_k", 1, idx), n, Tq, Tk, nh, nkv, scale, code)
    return out
