"""The short way from Python to the paged operators takes plain tensors and nothing else: tensors
under functional transforms and nested ones go the full way and raise there; running out of memory
is torch's own exception."""

import os
import subprocess
import sys

import pytest
import torch

import mlx_batch_invariant_b200 as bi
from mlx_batch_invariant_b200 import _lib
from test_paged_gpu import BF16, Batch, ints, same_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_device_error():
    _lib.device_error()
    yield
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


def child(code):
    env = dict(os.environ, PYTHONPATH=os.pathsep.join(p for p in sys.path if p))
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, (r.returncode, r.stderr[-2000:])
    return r.stdout


TRANSFORMS = """
import torch, mlx_batch_invariant_b200 as bi
zeros = lambda shape, dtype=torch.bfloat16: torch.zeros(shape, dtype=dtype, device="cuda")
q, k, v = zeros((5, 4, 64)), zeros((3, 2, 16, 64)), zeros((3, 2, 16, 64))
table, start, lens = (zeros(s, torch.int32) for s in ((2, 2), 3, 2))
def fn(q=q, k=k, v=v):
    return bi.paged_attention(q, k, v, table, start, lens)
calls = dict(
    vmap_q=lambda: torch.vmap(fn)(q[None]),
    vmap_caches=lambda: torch.vmap(lambda a, b: fn(k=a, v=b))(k[None], v[None]),
    jvp=lambda: torch.func.jvp(fn, (q,), (q,)),
    grad=lambda: torch.func.grad(lambda a: fn(a).float().sum())(q),
    nested=lambda: fn(torch.nested.nested_tensor([q[:2], q[2:]])),
)
for name, call in calls.items():
    try:
        call()
        print(name, "returned")
    except Exception as e:
        print(name, "raised")
torch.cuda.synchronize()
"""


def test_transforms_and_nested_tensors_raise():
    lines = child(TRANSFORMS).split("\n")[:-1]
    assert len(lines) == 5 and all(x.endswith(" raised") for x in lines), lines


OUT_OF_MEMORY = """
import torch, mlx_batch_invariant_b200 as bi
i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
a = i(1), i(0), i(0).view(1, 1)
bi.paged_plan(*a, 4, 1)
torch.cuda.set_per_process_memory_fraction(0.01)
try:
    bi.paged_plan(*a, 4, 1 << 28)
except torch.OutOfMemoryError:
    print("out of memory")
"""


def test_out_of_memory_is_torch_s():
    assert child(OUT_OF_MEMORY) == "out of memory\n"


def test_the_short_way_takes_plain_tensors():
    """... with and without gradients asked for, under inference mode and autocast."""
    b = Batch([2, 1], [30, 5], 4, 2, 64, 16, BF16)
    short = _lib.short_way()
    args = lambda q: (q, b.k, b.v, b.table, b.start, b.lens, None, None, 0, None, None)
    want = b.run()
    assert same_bits(short.attention(*args(b.tokens)), want)
    assert same_bits(short.attention(*args(b.tokens.clone().requires_grad_())), want)
    with torch.autocast("cuda", dtype=BF16):
        assert same_bits(short.attention(*args(b.tokens)), want)
    with torch.inference_mode():
        assert same_bits(short.attention(*args(b.tokens.clone())), want)
    assert short.plan(ints([1]), ints([0]), ints([[3]]), 4, 1, None, None) is not None
    tab, at = torch.zeros((9, 32), device="cuda"), torch.tensor([3], device="cuda")
    qkv = torch.zeros((1, 8 * 64), dtype=BF16, device="cuda")
    assert short.rope(qkv, tab, tab, at, at, b.k.clone(), b.v.clone(), None) is not None
