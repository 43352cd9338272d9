"""The paged operators under functional transforms: arguments that are of the exact tensor type
and say they are CUDA tensors, but have no storage.  They end in a Python exception, not in the
end of the process (the calls have one of their own).  No GPU: the tensors inside are fake."""

import os
import subprocess
import sys

CALLS = """
import torch, mlx_batch_invariant_b200 as bi
from torch._subclasses.fake_tensor import FakeTensorMode
I32, I64 = torch.int32, torch.int64
zeros = lambda shape, dtype=torch.float32: torch.zeros(shape, dtype=dtype, device="cuda")
cache = lambda: zeros((3, 2, 4, 32))
with FakeTensorMode():
    calls = dict(
        plan=(lambda *a: bi.paged_plan(*a, 4, 5), (zeros(2, I32), zeros(2, I32), zeros((2, 4), I32))),
        rope=(bi.rope_kv_paged, (zeros((5, 8 * 32)), zeros((9, 16)), zeros((9, 16)),
                                 zeros(5, I64), zeros(5, I64), cache(), cache())),
        attention=(bi.paged_attention, (zeros((5, 4, 32)), cache(), cache(), zeros((2, 2), I32),
                                        zeros(3, I32), zeros(2, I32))))
    for name, (fn, args) in calls.items():
        def call(*a):
            assert all(type(t) is torch.Tensor and t.is_cuda for t in a)
            print(name, how, end=" ", flush=True)
            return fn(*a)
        for how in "vmap", "functional":
            try:
                if how == "vmap":
                    torch.vmap(call)(*[t[None] for t in args])
                else:
                    call(*[torch._to_functional_tensor(t) for t in args])
                print("returned")
            except Exception as e:
                print("raised", flush=True)
"""


def test_tensors_without_storage_raise():
    env = dict(os.environ, PYTHONPATH=os.pathsep.join(p for p in sys.path if p))
    r = subprocess.run([sys.executable, "-c", CALLS], env=env, capture_output=True, text=True,
                       timeout=600)
    assert r.stdout.split("\n")[:-1] == [
        "%s %s raised" % (op, how) for op in ("plan", "rope", "attention")
        for how in ("vmap", "functional")], r.stdout + r.stderr[-2000:]
    assert r.returncode == 0
