"""paged_attention's results go to places of their own: an expanded `out`, whose rows or heads
share theirs, is refused."""

import pytest
import torch

import mlx_batch_invariant_b200 as bi
from mlx_batch_invariant_b200 import _lib
from test_paged_cpu import attention_args, c_attention


@pytest.mark.parametrize("shape", [(1, 4, 32), (5, 1, 32)])
def test_expanded_out_is_refused(shape):
    a = attention_args()
    with pytest.raises(ValueError, match="expanded"):
        bi.paged_attention(*list(a.values())[:6], out=torch.zeros(shape).expand(5, 4, 32))


@pytest.mark.parametrize("kw, status", [
    (dict(os=(0, 32)), -3), (dict(os=(128, 0)), -3), (dict(os=(-128, 32)), -3),
    (dict(os=(128, -32)), -3),
])
def test_c_out_strides(kw, status):
    assert c_attention(**kw) == status
    assert _lib.lib().bi_last_error()


@pytest.mark.gpu
def test_out_of_one_row_or_head_may_have_any_stride():
    """Dimensions of one, whose strides say nothing."""
    from test_paged_gpu import BF16, Batch, same_bits
    for q, H in (([1], 4), ([3], 1)):
        b = Batch(q, [40], H, 1, 64, 16, BF16)
        want = b.run()
        n, strides = want.numel(), list(want.stride())
        strides[0 if len(b.tokens) == 1 else 1] = 0
        out = torch.zeros(n, dtype=BF16, device="cuda").as_strided(want.shape, strides)
        assert same_bits(b.run(out=out), want)
    with pytest.raises(ValueError, match="expanded"):
        b.run(out=torch.zeros((1, 1, 64), dtype=BF16, device="cuda").expand(3, 1, 64))
