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
