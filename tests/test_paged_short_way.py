"""The paged operators where the short way from Python (the _bind module) cannot be used: one
warning, then every call through the full checks and ctypes."""

import importlib.util
import os
import sys
import types
import warnings

import pytest
import torch

import mlx_batch_invariant_b200 as bi
from mlx_batch_invariant_b200 import _lib

PKG = "mlx_batch_invariant_b200"
NAME = PKG + "._bind"


@pytest.fixture(params=["missing", "for another torch", "of an earlier version"])
def unusable(request, monkeypatch):
    def init(*a):
        raise AssertionError("it must not be used")
    module = None  # an import of None raises ImportError
    if request.param != "missing":
        module = types.ModuleType(NAME)
        module.init = init
        if request.param == "for another torch":
            module.torch_version = "0.1"
    monkeypatch.setattr(_lib, "_short", None)
    monkeypatch.delattr(sys.modules[PKG], "_bind", raising=False)
    monkeypatch.setitem(sys.modules, NAME, module)
    if module is not None:
        monkeypatch.setattr(sys.modules[PKG], "_bind", module, raising=False)


def test_arguments_are_checked_all_the_same(unusable):
    vec, table = torch.zeros(2, dtype=torch.int32), torch.zeros((2, 3), dtype=torch.int32)
    with pytest.warns(RuntimeWarning, match="ctypes") as seen:
        with pytest.raises(ValueError, match="page_size"):
            bi.paged_plan(vec, vec, table, 0, 3)
        with pytest.raises(ValueError, match="CUDA tensors"):
            bi.paged_plan(vec, vec, table, 4, 3)
        with pytest.raises(ValueError, match="q must be"):
            bi.paged_attention(table, table, table, table, vec, vec)
        with pytest.raises(ValueError, match="qkv"):
            bi.rope_kv_paged(vec, vec, vec, vec, vec, table, table)
    assert len(seen) == 1


@pytest.mark.gpu
def test_the_results_are_the_same(unusable):
    from test_paged_gpu import BF16, I32, ints, randn, same_bits, step
    H, Hkv, D, page = 8, 2, 64, 16
    ang = torch.rand((300, D // 2), device="cuda")

    def run():
        k, v = randn((9, Hkv, page, D), BF16, 1), randn((9, Hkv, page, D), BF16, 2)
        table = torch.full((2, 4), -1, device="cuda", dtype=I32)
        out, plan = step(ints([40, 3]), ints([0, 0]), table, ints(list(range(9))), ints([0]),
                         randn((45, (H + 2 * Hkv) * D), BF16, 3), ang.cos(), ang.sin(), k, v, page)
        return out[:43], k, v, table, plan.slots, plan.next_head

    with pytest.warns(RuntimeWarning, match="ctypes"):
        got = run()
    assert _lib.short_way() is _lib.FullWay
    _lib._short = None  # and now the module that was built
    sys.modules.pop(NAME)
    if hasattr(sys.modules[PKG], "_bind"):
        del sys.modules[PKG]._bind
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        want = run()
    assert _lib.short_way() is not _lib.FullWay
    assert all(same_bits(a, b) for a, b in zip(got, want))
    assert _lib.device_error() == 0


def test_it_is_built_anew_for_another_torch(tmp_path, monkeypatch):
    root = os.path.dirname(os.path.dirname(os.path.abspath(bi.__file__)))
    spec = importlib.util.spec_from_file_location("_bi_build", os.path.join(root, "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    module, version = tmp_path / "_bind.so", tmp_path / "bind.torch"
    monkeypatch.setattr(build, "BIND", str(module))
    monkeypatch.setattr(build, "BIND_TORCH", str(version))
    assert build._bind_stale()  # not there
    module.write_text("")
    assert build._bind_stale()  # nobody knows which torch it is for
    version.write_text("0.1")
    assert build._bind_stale()
    version.write_text(build._torch_version())
    assert not build._bind_stale()
    os.utime(module, (0, 0))
    assert build._bind_stale()  # older than its source
