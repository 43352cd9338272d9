"""paged_attention where a prompt's keys are split over several blocks of the grid: the first
piece of a tile of many rows joins its key blocks itself, the others leave theirs to the join.
Values against 64 bits, and the bits of calls that split nothing."""

import pytest
import torch

import mlx_batch_invariant_b200 as bi
from mlx_batch_invariant_b200 import _lib
from test_paged_gpu import BF16, FP16, FP32, Batch, ints, randn, same_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_device_error():
    yield
    assert _lib.device_error() == 0


def unsplit(b, window=0, first_tokens=0, sinks=None):
    """The same call with the least workspace, which holds no partial results."""
    lib, (T, H, D), (R, W) = _lib.lib(), b.tokens.shape, b.table.shape
    size = lib.bi_paged_sdpa_workspace(0, R, H, D, W, b.page)
    ws, out = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.zeros_like(b.tokens)
    _lib.check(lib.bi_paged_sdpa(
        b.tokens.data_ptr(), _lib.i64_2((H * D, D)), b.k.data_ptr(), _lib.i64_3(b.k.stride()[:3]),
        b.v.data_ptr(), _lib.i64_3(b.v.stride()[:3]), b.n_pages, b.page, b.table.data_ptr(), W, W,
        b.start.data_ptr(), b.lens.data_ptr(), None if sinks is None else sinks.data_ptr(),
        D ** -0.5, window, first_tokens, T, R, H, b.Hkv, D, _lib.dtype_code(b.dtype),
        out.data_ptr(), _lib.i64_2((H * D, D)), ws.data_ptr(), size,
        _lib.stream_handle(out.device)), "bi_paged_sdpa")
    return out


# new and cached tokens, H, Hkv, D: the pieces of a tile's key blocks that follow
SPLITS = [
    ([200], [7000], 8, 2, 128),              # one block a piece
    ([260], [9000], 32, 8, 128),             # two pieces of about ten
    ([100, 1, 64], [12000, 5000, 300], 16, 2, 64),
    ([37], [9100], 24, 1, 128),              # 5 tokens a tile
    ([90, 33], [4000, 16000], 6, 6, 64),     # 128 tokens a tile, one that is not full
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("q, c, H, Hkv, D", SPLITS)
def test_split_prompts(q, c, H, Hkv, D, dtype):
    b = Batch(q, c, H, Hkv, D, 64, dtype, seed=3)
    assert same_bits(b.check(), unsplit(b))


@pytest.mark.parametrize("window, first", [(5000, 0), (3000, 700), (9000, 4)])
def test_split_prompts_with_a_window(window, first):
    b = Batch([260, 1], [9000, 7000], 32, 8, 128, 32, BF16, seed=4)
    sinks = randn((32,), BF16, 5)
    kw = dict(window=window, first_tokens=first, sinks=sinks)
    assert same_bits(b.check(**kw), unsplit(b, **kw))


def test_split_rows_that_see_nothing():
    """Positions below zero in a request that is split: zeros."""
    b = Batch([300], [9000], 32, 8, 128, 64, BF16, seed=6)
    b.lens = ints([200])  # the first 100 tokens lie before the sequence
    b.tokens = b.tokens.contiguous()
    got = b.run()
    assert not got[:100].any() and got[100:].isfinite().all() and got[100:].any(-1).all()
    assert same_bits(got, unsplit(b))


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_split_non_finite_values_stay_in_their_rows(bad):
    b = Batch([260], [9000], 32, 8, 128, 64, BF16, seed=7)
    want = b.run()
    at = 9130  # seen by tokens 130 and behind
    b.v[b.table[0, at // 64], :, at % 64] = bad
    got = b.run()
    assert same_bits(got[:130], want[:130]) and not got[130:].isfinite().any()
    assert same_bits(got, unsplit(b))


@pytest.mark.parametrize("R", [31, 32, 33, 64, 65])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_request_counts(R, dtype):
    """Around the number of requests from which a kernel of its own looks for the items."""
    q = [1 + (5 * r) % 40 if r % 3 == 0 else 1 for r in range(R)]
    c = [(331 * r) % 2300 for r in range(R)]
    b = Batch(q, c, 8, 2, 64, 16, dtype, seed=8)
    got = b.check()
    at = sum(q[:R - 1])
    alone = bi.paged_attention(b.tokens[at:], b.k, b.v, b.table[R - 1:], ints([0, q[-1]]),
                               b.lens[R - 1:])
    assert same_bits(got[at:], alone)


def test_empty_requests_between():
    """Requests without tokens or without a sequence, first, last and in between."""
    b = Batch([0, 0, 150, 0, 1, 0], [0, 900, 6000, 0, 4000, 77], 32, 8, 128, 64, BF16, seed=9)
    assert same_bits(b.check(), unsplit(b))
