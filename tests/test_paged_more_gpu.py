"""The paged operators called in ways that the other tests do not: captured before their first
use, groups of more heads than a tile has rows, results over the queries, a step cut off by a
table that is a view of a wider one, the short way against the full one."""

import os
import subprocess
import sys

import pytest
import torch

import mlx_batch_invariant_b200 as bi
from mlx_batch_invariant_b200 import _lib, _paged
from test_paged_gpu import BF16, FP16, FP32, Batch, ints, randn, same_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_device_error():
    yield
    assert _lib.device_error() == 0


FIRST_USE = """
import torch, mlx_batch_invariant_b200 as bi
i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
q, c, table = i([3, 1]), i([0, 0]), torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
free, head = i([5, 2, 0, 1]), i([0])
qkv = torch.randn(4, 12 * 128, device="cuda").to({dtype})
cos = torch.ones(64, 64, device="cuda"); sin = torch.zeros_like(cos)
k = torch.zeros(6, 2, 16, 128, dtype=qkv.dtype, device="cuda"); v = torch.zeros_like(k)
def step():
    p = bi.paged_plan(q, c, table, 16, 4, free_pages=free, free_head=head)
    r = bi.rope_kv_paged(qkv, cos, sin, p.positions, p.slots, k, v)
    return bi.paged_attention(r, k, v, table, p.query_start, p.seq_lens)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = step()
g.replay()
got = out.clone()
assert torch.equal(got, step()) and got.isfinite().all() and got.any()
# the first token of a request sees itself only
assert torch.equal(got[3].view(2, 4, 128), qkv[3].view(12, 1, 128)[10:].expand(2, 4, 128))
assert bi._lib.device_error() == 0
"""


@pytest.mark.parametrize("dtype", ["torch.bfloat16", "torch.float32"])
def test_captured_before_their_first_use(dtype):
    env = dict(os.environ, PYTHONPATH=os.pathsep.join(p for p in sys.path if p))
    r = subprocess.run([sys.executable, "-c", FIRST_USE.replace("{dtype}", dtype)], env=env,
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("H, Hkv", [(129, 1), (256, 1), (128, 1), (260, 2)])
def test_large_groups(H, Hkv, dtype):
    """Around the 128 query heads of a KV head that the tensor cores take."""
    Batch([3, 1], [140, 700], H, Hkv, 64, 16, dtype, seed=11).check()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_results_over_the_queries(dtype):
    b = Batch([150, 1], [6000, 4000], 32, 8, 128, 64, dtype, seed=12)
    want = b.run()
    assert same_bits(b.run(out=b.tokens), want) and same_bits(b.tokens, want)


def test_more_requests_than_tokens_and_repeated_rows():
    """A table row that appears twice (two requests over one sequence), and many idle ones."""
    b = Batch([2], [900], 8, 2, 128, 16, BF16, seed=13)
    want = b.run()
    rows = [0] * 80
    start = [0] * 40 + [2] * 40 + [4]
    got = bi.paged_attention(torch.cat((b.tokens, b.tokens)), b.k, b.v, b.table[rows],
                             ints(start), b.lens[rows])
    assert same_bits(got[:2], want) and same_bits(got[2:], want)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_the_short_way_and_the_full_one(dtype):
    """What the module takes gives what the checks in Python give."""
    b = Batch([5, 1], [90, 300], 8, 2, 64, 16, dtype, seed=14)
    sinks = randn((8,), dtype, 3)
    short = b.run(window=64, first_tokens=2, sinks=sinks)
    full = _paged._attention_eager(b.tokens, b.k, b.v, b.table, b.start, b.lens, 64 ** -0.5, 64, 2,
                                   sinks, None, _lib.dtype_code(dtype), b.k.device)
    assert same_bits(short, full)
    q, c = ints([5, 1]), ints([90, 300])
    plan = bi.paged_plan(q, c, b.table, 16, 8)
    other = _paged._plan_eager(q, c, b.table, 16, 8, None, None, b.k.device)
    assert plan.next_head is None and other[4] is None
    for x, y in zip(plan[:4], other[:4]):
        assert x.dtype == y.dtype and torch.equal(x, y)
    qkv, tab = randn((8, 12 * 64), dtype, 4), torch.rand((400, 32), device="cuda")
    k, v = b.k.clone(), b.v.clone()
    r = bi.rope_kv_paged(qkv, tab, tab, plan.positions, plan.slots, b.k, b.v)
    s = _paged._rope_eager(qkv, tab, tab, plan.positions, plan.slots, k, v, None, b.k.device)
    assert same_bits(r[:6], s[:6]) and same_bits(k, b.k) and same_bits(v, b.v)
