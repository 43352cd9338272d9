"""PagedDecodeGraph.start on the host: what it refuses, and that a refusal changes nothing."""

import types

import pytest
import torch

from mlx_batch_invariant_b200 import decoder as dec


def graph(requests=3, vocab=64):
    g = dec.PagedDecodeGraph.__new__(dec.PagedDecodeGraph)
    model = types.SimpleNamespace(cfg=types.SimpleNamespace(vocab=vocab))
    g.server = types.SimpleNamespace(requests=requests, model=model)
    g.tok = torch.zeros(requests, dtype=torch.long)
    g.running = torch.zeros(requests, dtype=torch.int32)
    g._active = [0] * requests
    return g


@pytest.mark.parametrize("bad", [64, -1, 1 << 40])
def test_tokens_outside_the_vocabulary(bad):
    """The embedding would read out of its table: a fault on the GPU."""
    g = graph()
    g.start([5, None, 63])
    with pytest.raises(ValueError, match=r"\[0, 64\)"):
        g.start([1, bad, None])
    assert g.tok.tolist() == [5, 0, 63] and g.running.tolist() == [1, 0, 1]
    assert g._active == [1, 0, 1]


def test_entries_are_counted():
    g = graph()
    with pytest.raises(ValueError, match="2 entries for 3"):
        g.start([1, 2])
    g.start([None, torch.tensor(7), 0])
    assert g.tok.tolist() == [0, 7, 0] and g.running.tolist() == [0, 1, 1]
