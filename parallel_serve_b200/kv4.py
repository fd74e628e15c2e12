"""A KV cache held in 4 bits: pools, and what their bytes stand for.

The reference keeps no cache (its decode benchmarks size one per batch,
kernel/FRIDAY_REPORT.md:131); this one is an addition of this library. The 128
channels of one (position, KV head) are 4 groups of 32; a group stores a zero
``z = T(min)`` and a scale ``s = T((max - z) / 15)`` in the model's 16-bit type
and 32 codes ``c = clamp(rint((x - z) / s), 0, 15)``, and stands for ``s * c + z``:
160 bytes per position and head for K and V together, where 16 bits take 512.

``ops.kv4_append`` writes it, ``ops.kv4_gather`` reads it back and
``ops.kv4_decode_attention`` attends over it.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

CODE_BYTES = 64      # per (position, KV head), for K and for V
GROUPS = 4           # of 32 channels


class KV4Pool(NamedTuple):
    """One model's pools: codes uint8 ``[rows, n_kv_heads, length, 64]`` and meta
    ``[rows, n_kv_heads, length, 4, 2]`` = (scale, zero) of the 4 groups. Rows
    are sequence slots with ``length = L_cap``, or pages with ``length =
    page_size``."""
    k_codes: torch.Tensor
    k_meta: torch.Tensor
    v_codes: torch.Tensor
    v_meta: torch.Tensor

    @classmethod
    def zeros(cls, rows: int, n_kv_heads: int, length: int, dtype: torch.dtype = torch.float16,
              device: torch.device | str = "cuda") -> "KV4Pool":
        """Pools of ``rows`` slots (or pages) whose every value reads back as 0."""
        if dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"parallel-serve kernels take float16 or bfloat16, got {dtype}")

        def codes():
            return torch.zeros(rows, n_kv_heads, length, CODE_BYTES, dtype=torch.uint8, device=device)

        def meta():
            return torch.zeros(rows, n_kv_heads, length, GROUPS, 2, dtype=dtype, device=device)
        return cls(codes(), meta(), codes(), meta())

    @staticmethod
    def bytes_per_position(n_kv_heads: int) -> int:
        """Bytes that K and V of one position take."""
        return n_kv_heads * 2 * (CODE_BYTES + GROUPS * 4)
