"""The paged-cache operators' refusals: arguments that the Python functions and the C ABI
turn down before anything is launched (no GPU needed)."""

import pytest
import torch

import mlx_batch_invariant_b200 as bi
from mlx_batch_invariant_b200 import _lib

I32, I64 = torch.int32, torch.int64


def ints(*v, dtype=I32):
    return torch.tensor(v, dtype=dtype)


def plan_args(**kw):
    a = dict(query_lens=ints(1, 2), context_lens=ints(3, 4),
             block_table=torch.zeros((2, 4), dtype=I32), page_size=4, num_tokens=3)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw, what", [
    (dict(page_size=0), "page_size"),
    (dict(num_tokens=-1), "num_tokens"),
    (dict(query_lens=ints(1, 2, dtype=I64)), "query_lens"),
    (dict(query_lens=ints(1, 2, 3, 4)[::2]), "query_lens"),
    (dict(context_lens=ints(1)), "context_lens"),
    (dict(block_table=torch.zeros((3, 4), dtype=I32)), "3 rows"),
    (dict(block_table=torch.zeros((2, 4), dtype=I64)), "block_table"),
    (dict(block_table=torch.zeros((4, 2), dtype=I32).t()), "block_table"),
    (dict(block_table=torch.zeros((1, 4), dtype=I32).expand(2, 4)), "block_table"),
    (dict(free_pages=ints(1, 2)), "go together"),
    (dict(free_head=ints(0)), "go together"),
    (dict(free_pages=ints(1, 2), free_head=ints(0, 1)), "free_head"),
    (dict(free_pages=ints(1, 2, dtype=I64), free_head=ints(0)), "free_pages"),
    (dict(), "CUDA tensors"),
])
def test_plan_refuses(kw, what):
    with pytest.raises(ValueError, match=what):
        a = plan_args(**kw)
        bi.paged_plan(a.pop("query_lens"), a.pop("context_lens"), a.pop("block_table"),
                      a.pop("page_size"), a.pop("num_tokens"), **a)


def rope_args(**kw):
    cache = torch.zeros((3, 2, 4, 8))
    a = dict(qkv=torch.zeros((5, 48)), cos=torch.zeros((9, 4)), sin=torch.zeros((9, 4)),
             positions=torch.zeros(5, dtype=I64), slots=torch.zeros(5, dtype=I64),
             k_cache=cache, v_cache=cache.clone(), out=None)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw, what", [
    (dict(qkv=torch.zeros((1, 5, 48))), "qkv"),
    (dict(qkv=torch.zeros((5, 48), dtype=torch.float64)), "unsupported dtype"),
    (dict(qkv=torch.zeros((5, 47))), "47 elements"),
    (dict(qkv=torch.zeros((5, 24))), "24 elements"),
    (dict(qkv=torch.zeros((5, 48), dtype=torch.bfloat16)), "dtype"),
    (dict(v_cache=torch.zeros((3, 2, 4, 16))), "one shape"),
    (dict(k_cache=torch.zeros((3, 2, 8)), v_cache=torch.zeros((3, 2, 8))), "cache is"),
    (dict(k_cache=torch.zeros((3, 2, 8, 4)).transpose(2, 3)), "last dimension"),
    (dict(k_cache=torch.zeros((1, 2, 4, 8)).expand(3, 2, 4, 8)), "expanded"),
    (dict(cos=torch.zeros((9, 4), dtype=torch.float64)), "cos and sin"),
    (dict(sin=torch.zeros((8, 4))), "cos and sin"),
    (dict(cos=torch.zeros((9, 5)), sin=torch.zeros((9, 5))), "rot = 10"),
    (dict(positions=torch.zeros(4, dtype=I64)), "positions"),
    (dict(slots=torch.zeros(5, dtype=I32)), "slots"),
    (dict(out=torch.zeros((5, 2, 8)).transpose(0, 1)), "out"),
    (dict(), "CUDA tensors"),
])
def test_rope_refuses(kw, what):
    a = rope_args(**kw)
    with pytest.raises(ValueError, match=what):
        bi.rope_kv_paged(a["qkv"], a["cos"], a["sin"], a["positions"], a["slots"], a["k_cache"],
                         a["v_cache"], out=a["out"])


def attention_args(**kw):
    cache = torch.zeros((3, 2, 4, 32))
    a = dict(q=torch.zeros((5, 4, 32)), k_cache=cache, v_cache=cache.clone(),
             block_table=torch.zeros((2, 2), dtype=I32), query_start=ints(0, 1, 5),
             seq_lens=ints(3, 4))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw, what", [
    (dict(q=torch.zeros((5, 128))), "q must be"),
    (dict(q=torch.zeros((5, 4, 32), dtype=torch.float64)), "unsupported dtype"),
    (dict(q=torch.zeros((5, 4, 64))), "head dim 64"),
    (dict(q=torch.zeros((5, 3, 32))), "multiple of kv head"),
    (dict(q=torch.zeros((5, 4, 32), dtype=torch.float16)), "dtype"),
    (dict(q=torch.zeros((5, 4, 48)), k_cache=torch.zeros((3, 2, 4, 48)),
          v_cache=torch.zeros((3, 2, 4, 48))), "multiple of 32"),
    (dict(scale=float("nan")), "scale"),
    (dict(scale=-1.0), "scale"),
    (dict(scale=float("inf")), "scale"),
    (dict(window=-1), "window"),
    (dict(first_tokens=-2), "window and first"),
    (dict(first_tokens=2), "needs a window"),
    (dict(seq_lens=ints(3, 4, dtype=I64)), "seq_lens"),
    (dict(query_start=ints(0, 5)), "query_start"),
    (dict(block_table=torch.zeros((3, 2), dtype=I32)), "3 rows"),
    (dict(block_table=torch.zeros((2, 0), dtype=I32)), "empty"),
    (dict(sinks=torch.zeros(2)), "sinks"),
    (dict(k_cache=torch.zeros(3 * 256 + 1)[1:].view(3, 2, 4, 32)), "16-byte"),
    (dict(out=torch.zeros((5, 32, 4)).transpose(1, 2)), "out must be"),
    (dict(), "CUDA tensors"),
])
def test_attention_refuses(kw, what):
    a = attention_args(**kw)
    with pytest.raises(ValueError, match=what):
        bi.paged_attention(a.pop("q"), a.pop("k_cache"), a.pop("v_cache"), a.pop("block_table"),
                           a.pop("query_start"), a.pop("seq_lens"), **a)


def test_attention_head_dim_not_built():
    c = torch.zeros((3, 2, 4, 288))
    a = attention_args(q=torch.zeros((5, 4, 288)), k_cache=c, v_cache=c)
    with pytest.raises(NotImplementedError, match="288"):
        bi.paged_attention(*a.values())


# --------------------------------------------------------------------------- the C ABI
def c_attention(**kw):
    """bi_paged_sdpa on made-up pointers; every case is refused before a launch."""
    a = dict(q=64, qs=(128, 32), k=64, ks=(256, 128, 32), v=64, vs=(256, 128, 32), n_pages=3,
             page=4, table=64, stride=2, width=2, start=64, seq=64, sinks=None, scale=1.0,
             window=0, first=0, T=5, R=2, H=4, Hkv=2, D=32, dtype=0, out=64, os=(128, 32),
             ws=64, ws_bytes=1 << 20)
    a.update(kw)
    return _lib.lib().bi_paged_sdpa(
        a["q"], _lib.i64_2(a["qs"]), a["k"], _lib.i64_3(a["ks"]), a["v"], _lib.i64_3(a["vs"]),
        a["n_pages"], a["page"], a["table"], a["stride"], a["width"], a["start"], a["seq"],
        a["sinks"], a["scale"], a["window"], a["first"], a["T"], a["R"], a["H"], a["Hkv"],
        a["D"], a["dtype"], a["out"], _lib.i64_2(a["os"]), a["ws"], a["ws_bytes"], None)


@pytest.mark.parametrize("kw, status", [
    (dict(dtype=7), -1), (dict(T=-1), -1), (dict(Hkv=3), -1), (dict(Hkv=0), -1), (dict(D=48), -1),
    (dict(D=288), -2), (dict(scale=-1.0), -1), (dict(scale=float("nan")), -1),
    (dict(first=3), -1), (dict(T=1 << 31), -2), (dict(q=None), -1), (dict(table=None), -1),
    (dict(width=0, stride=0), -1), (dict(n_pages=0), -1), (dict(stride=1), -1), (dict(q=72), -3),
    (dict(ks=(256, 130, 32)), -3), (dict(vs=(256, 0, 32)), -3), (dict(ws=None), -1),
    (dict(ws_bytes=16), -1), (dict(page=0), -1), (dict(window=-1), -1),
    (dict(T=0), 0), (dict(R=0), 0),
])
def test_c_attention_refuses(kw, status):
    assert c_attention(**kw) == status
    assert bool(_lib.lib().bi_last_error()) == (status != 0)


@pytest.mark.parametrize("kw, status", [
    (dict(R=-1), -1), (dict(T=-1), -1), (dict(page=0), -1), (dict(T=1 << 31), -2),
    (dict(ql=None), -1), (dict(table=None), -1), (dict(start=None), -1), (dict(slots=None), -1),
    (dict(free=64), -1), (dict(free=64, head=64), -1), (dict(stride=3), -1),
])
def test_c_plan_refuses(kw, status):
    a = dict(ql=64, cl=64, R=2, T=3, table=64, stride=4, width=4, page=4, free=None, n_free=2,
             head=None, start=64, seq=64, pos=64, slots=64, next=None)
    a.update(kw)
    assert _lib.lib().bi_paged_plan(
        a["ql"], a["cl"], a["R"], a["T"], a["table"], a["stride"], a["width"], a["page"],
        a["free"], a["n_free"], a["head"], a["start"], a["seq"], a["pos"], a["slots"], a["next"],
        None) == status


@pytest.mark.parametrize("kw, status", [
    (dict(dtype=3), -1), (dict(T=-1), -1), (dict(hd=7), -1), (dict(rot=3), -1),
    (dict(rot=10), -1), (dict(page=0), -1), (dict(T=1 << 31), -2), (dict(stride=40), -1),
    (dict(qkv=None), -1), (dict(cos=None), -1), (dict(slots=None), -1), (dict(k=None), -1),
    (dict(out=None), -1),
])
def test_c_rope_refuses(kw, status):
    a = dict(qkv=64, stride=48, T=5, hq=2, hk=2, hd=8, rot=8, cos=64, sin=64, n_pos=9, pos=64,
             slots=64, out=64, k=64, v=64, n_pages=3, page=4, dtype=0)
    a.update(kw)
    s = _lib.i64_3((64, 32, 8))
    assert _lib.lib().bi_rope_kv_paged(
        a["qkv"], a["stride"], a["T"], a["hq"], a["hk"], a["hd"], a["rot"], a["cos"], a["sin"],
        a["n_pos"], a["pos"], a["slots"], a["out"], a["k"], s, a["v"], s, a["n_pages"],
        a["page"], a["dtype"], None) == status


def test_workspace_size():
    size = _lib.lib().bi_paged_sdpa_workspace
    least = size(0, 64, 32, 128, 512, 16)
    assert 0 < least < 4096
    # one row of every key block, (m, l, o) in fp32
    assert size(64, 64, 32, 128, 512, 16) >= 64 * 32 * (512 * 16 // 512) * (128 + 2) * 4
    assert size(1 << 20, 64, 32, 128, 1 << 20, 16) <= (256 << 20) + 4096
    assert size(-1, 1, 1, 32, 1, 1) == 0
