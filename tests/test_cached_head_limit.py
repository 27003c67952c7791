"""More groups of query heads than a launch has room for are refused on every device, as an argument that does not fit."""

import pytest
import torch

from dual_mod_public_b200.ops import cached_attention

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("dev", DEVICES)
def test_groups_of_heads(dev):
    def call(hkv, group):
        q = torch.ones(1, hkv * group, 8, dtype=torch.bfloat16, device=dev)
        kv = torch.ones(1, 2, hkv, 8, dtype=torch.bfloat16, device=dev)
        return cached_attention(q, kv, kv, torch.ones(1, dtype=torch.int32, device=dev))
    with pytest.raises(ValueError):
        call(4095, 16 * 16 + 1)                                   # 17 groups of each: 69615
    for hkv, group in ((4095, 16 * 16), (1, 16 * 600 + 1)):       # 65520, and 601 of one
        assert (call(hkv, group) == 1).all()
