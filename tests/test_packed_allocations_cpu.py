"""Without a GPU the allocator that is not public does not answer, and the public one is chosen."""

import torch

from dual_mod_public_b200.ops import cuda_ops


def test_public_allocator_where_the_other_fails(monkeypatch):
    import torch._C._dynamo.guards as guards

    def fail(*args):
        raise TypeError("another signature")
    monkeypatch.setattr(guards, "_empty_strided_cuda", fail, raising=False)
    assert cuda_ops._choose_empty() is cuda_ops._public_empty
    monkeypatch.setattr(guards, "_empty_strided_cuda", lambda size, stride, dtype: torch.empty(2, 3, dtype=dtype))
    assert cuda_ops._choose_empty() is cuda_ops._public_empty            # not on a GPU
