"""bi_paged_sdpa refuses calls whose work items cannot be counted on the device (in 32 bits that
stop at 2^30); without a GPU what is below that gets as far as the device."""

import pytest
import torch

from mlx_batch_invariant_b200 import _lib
from test_paged_cpu import c_attention

WS = 1 << 40  # made up, like the pointers


@pytest.mark.parametrize("kw", [
    dict(T=1 << 23, R=1 << 23, H=128, Hkv=128, D=32, dtype=1),          # 2^30 tiles of one token
    dict(T=(1 << 30) + 4096, R=1 << 30, H=1, Hkv=1, D=32),              # 2^30 requests
    dict(T=5, R=(1 << 31) - 2, H=4, Hkv=2),
    dict(T=1 << 30, R=1, H=256, Hkv=16, D=64, dtype=2, page=16),        # 2^27 tiles of 8 tokens, 16 heads
    dict(T=1 << 29, R=1 << 29, H=258, Hkv=2, D=32, dtype=2),            # 17 groups of a KV head
])
def test_too_many_items(kw):
    assert c_attention(ws_bytes=WS, **kw) == -2
    assert b"2^30" in _lib.lib().bi_last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are made up")
@pytest.mark.parametrize("kw", [
    dict(T=1 << 22, R=1 << 22, H=128, Hkv=128, D=32, dtype=1),
    dict(T=1 << 29, R=1, H=128, Hkv=1, D=64, dtype=2, page=16),  # 2^29 tiles of one token
])
def test_what_fits_gets_past_the_count(kw):
    assert c_attention(ws_bytes=WS, **kw) != 0
    assert b"2^30" not in _lib.lib().bi_last_error()
