"""paged_attention where several special values meet: non-finite values of keys in a step whose
scores move the running maximum, and sink logits that are infinite.

Everything here is compared bit for bit with a call that lacks the special value, or element by
element within the bound that test_paged_gpu.py derives."""

import pytest
import torch

import mlx_batch_invariant_b200 as bi
from mlx_batch_invariant_b200 import _lib
from test_paged_gpu import BF16, FP16, FP32, Batch, ints, randn, same_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_device_error():
    _lib.device_error()
    yield
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


def rising(q, c, D, dtype, junk, H=8, Hkv=2, page=16):
    """Scores that rise by 0.15 a key on top of N(0, 1): 65 keys further the maximum is 2^14
    higher, so that every step of 128 keys moves it and rescales what came before."""
    b = Batch(q, c, H, Hkv, D, page, dtype, seed=D, junk=junk)
    b.tokens[..., 0] = D ** 0.5
    for k in b.keys:
        k[..., 0] = 0.15 * torch.arange(k.shape[0], device="cuda")[:, None]
    b.fill()
    return b


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("q, c", [
    ([64], [320]),               # two tiles over the same keys
    ([1, 1, 1], [379, 250, 130]),  # one token each, steps 2, 1 and 1 of a block of 512 keys
    ([20, 1, 90], [300, 700, 900]),
])
def test_masked_values_where_the_maximum_moves(q, c, D, dtype):
    """What lies behind a sequence in its last page, and later tokens' values, at a step that
    also rescales the result of the steps before it."""
    plain = rising(q, c, D, dtype, 1.0)
    want = plain.check()
    for junk in float("nan"), float("inf"):
        assert same_bits(rising(q, c, D, dtype, junk).check(), want)
    # the last tokens' own values: the rows before them see none of it
    at = 0
    for r, n in enumerate(q):
        for bad in float("nan"), -float("inf"):
            b = rising(q, c, D, dtype, 1.0)
            b.vals[r][c[r] + n - 1] = bad
            b.fill()
            got = b.run()
            last = at + n - 1
            assert same_bits(got[:last], want[:last]) and same_bits(got[last + 1:], want[last + 1:])
            assert not got[last].isfinite().any()
        at += n


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
def test_visible_values_where_the_maximum_moves(D, dtype):
    """One infinite element: its column in the rows that see it, and not a bit anywhere else."""
    for q, c, key in (([64], [320], 350), ([1, 1], [379, 250], 370), ([90], [900], 950)):
        want = rising(q, c, D, dtype, 1.0).run()
        b = rising(q, c, D, dtype, 1.0)
        b.vals[0][key, 1, 5] = float("inf")
        b.fill()
        got = b.run()
        first = max(0, key - c[0])
        assert (got[first:q[0], 4:, 5] == float("inf")).all()
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[first:q[0], 4:, 5] = True
        assert same_bits(got.masked_fill(hit, 0), want.masked_fill(hit, 0))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("sink", [-float("inf"), float("inf"), float("nan")])
def test_rows_that_see_nothing_whatever_the_sink(dtype, sink):
    """Zeros, as documented, where a row sees no key: whole and split over the grid."""
    b = Batch([5, 3, 2, 40], [0, 0, 0, 9000], 8, 2, 64, 16, dtype)
    b.lens = ints([2, 3, 0, 20])  # rows without a position: 3 of the first, 2, 20 of the last
    got = b.run(sinks=torch.full((8,), sink, device="cuda"))
    for lo, hi in ((0, 3), (8, 10), (10, 30)):
        assert not got[lo:hi].any() and not got[lo:hi].isnan().any()
    # a long request whose first tokens lie before its sequence, its keys split
    s = Batch([300], [9000], 32, 8, 128 if dtype != FP32 else 64, 64, dtype, seed=6)
    s.lens = ints([200])
    got = s.run(sinks=torch.full((32,), sink, device="cuda"))
    assert not got[:100].any() and not got[:100].isnan().any()
    if sink == -float("inf"):
        assert got[100:].isfinite().all() and got[100:].any(-1).all()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_a_sink_of_minus_infinity_is_none(dtype):
    """e^-inf = 0: the bits of a call without sinks, next to heads that have one."""
    b = Batch([1, 150, 9], [7000, 0, 800], 8, 2, 64, 32, dtype, seed=3)
    none, sinks = b.run(), randn((8,), dtype, 4)
    some = b.run(sinks=sinks)
    off = sinks.clone()
    off[::2] = -float("inf")
    got = b.run(sinks=off)
    assert same_bits(got[:, ::2], none[:, ::2]) and same_bits(got[:, 1::2], some[:, 1::2])
