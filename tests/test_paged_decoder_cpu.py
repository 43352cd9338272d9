"""What the paged decoder refuses before it needs a GPU, and its page counts."""

import types

import pytest
import torch

from mlx_batch_invariant_b200 import decoder as dec

TINY = dict(layers=1, hidden=32, heads=4, kv_heads=2, head_dim=8, inter=48, vocab=64)


def test_takes_a_model_on_a_gpu():
    m = dec.Decoder(dec.DecoderConfig(**TINY), max_batch=1, max_len=8, dtype=torch.float32,
                    device="cpu", single=True)
    with pytest.raises(ValueError, match="CUDA"):
        dec.PagedDecoder(m, 1, 4)


def test_sizes_are_checked():
    m = types.SimpleNamespace(device=torch.device("cuda"), _fused={}, max_batch=2, max_len=8)
    for sizes in ((0, 4, 16), (1, 0, 16), (1, 4, 0)):
        with pytest.raises(ValueError, match="positive"):
            dec.PagedDecoder(m, *sizes)
    m._fused = {"head": None}
    with pytest.raises(ValueError, match="exchange"):
        dec.PagedDecoder(m, 3, 4, 16)


def server(lens, pages, page=4, max_len=20, fused=False):
    s = dec.PagedDecoder.__new__(dec.PagedDecoder)
    s.model = types.SimpleNamespace(max_len=max_len, max_batch=1, _fused=fused)
    s.lens, s.pages, s.page_size, s.requests = lens, pages, page, len(lens)
    return s


def test_pages_are_counted():
    s = server([0, 1, 4, 5], 8)
    assert s.pages_used == 4
    assert s._lens_after([4, 3, 1, 0]) == [4, 4, 5, 5]  # 1 + 1 + 2 + 2 pages
    assert s.lens == [0, 1, 4, 5]
    with pytest.raises(ValueError, match="9 pages, the cache has 8"):
        s._lens_after([17, 0, 0, 0])
    with pytest.raises(ValueError, match="request 2 would have 21"):
        s._lens_after([0, 0, 17, 0])
    with pytest.raises(ValueError, match="exchange"):
        server([0, 0], 99, fused=True)._lens_after([11, 10])


def test_what_generate_paged_refuses():
    s = types.SimpleNamespace(requests=2)
    ids = torch.zeros((2, 5), dtype=torch.long)
    for args in ((torch.zeros((3, 5), dtype=torch.long), 1), (ids[:, :0], 1), (ids, 1, 0),
                 (ids, -1)):
        with pytest.raises(ValueError, match="prompts"):
            dec.generate_paged(s, *args)
