"""rope_kv_paged on caches whose heads have no elements: a ValueError like every other refusal."""

import pytest
import torch

import mlx_batch_invariant_b200 as bi
from test_paged_cpu import rope_args


def test_heads_without_elements():
    empty = torch.zeros((3, 2, 4, 0))
    a = rope_args(k_cache=empty, v_cache=empty.clone(), cos=torch.zeros((9, 0)),
                  sin=torch.zeros((9, 0)))
    with pytest.raises(ValueError, match="head_dim"):
        bi.rope_kv_paged(*list(a.values())[:7])
