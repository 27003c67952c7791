"""Outputs of the packed operators are allocations that dispatch modes see, and do not hang on an entry of torch that is not public."""

import sys
import types

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from dual_mod_public_b200.ops import cached_attention, cuda_ops, packed_attention, token_logprobs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Allocations(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.made = []

    def __torch_dispatch__(self, func, kinds, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if "empty" in str(func):
            self.made.append((tuple(out.shape), out.dtype))
        return out


def calls():
    q, k = torch.randn(40, 2, 64, device=DEV).bfloat16(), torch.randn(40, 1, 64, device=DEV).bfloat16()
    cu, n = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([0, 40], [7]))
    x, y = torch.randn(5, 100, device=DEV), torch.zeros(5, dtype=torch.int64, device=DEV)
    return [(lambda: (packed_attention(q, k, k, cu),), [((40, 2, 64), torch.bfloat16)]),
            (lambda: (cached_attention(q[:1], k[None], k[None], n),), [((1, 2, 64), torch.bfloat16)]),
            (lambda: tuple(token_logprobs(x, y, top=2)), [((5,), torch.float32)] * 2 + [((5, 2), torch.float32), ((5, 2), torch.int64)])]


def test_dispatch_modes_see_them():
    for call, want in calls():
        plain = call()
        with Allocations() as seen:
            out = call()
        assert sorted(seen.made, key=str) == sorted(want, key=str)
        assert all(torch.equal(a, b) for a, b in zip(out, plain))


@pytest.mark.parametrize("entry", [None, lambda size: None, lambda size, stride, dtype: torch.empty(1, device=DEV)])
def test_without_the_entry(monkeypatch, entry):
    want = [call() for call, _ in calls()]
    guards = types.ModuleType("guards")
    if entry is not None:
        guards._empty_strided_cuda = entry
    monkeypatch.setitem(sys.modules, "torch._C._dynamo.guards", guards)
    assert cuda_ops._choose_empty() is cuda_ops._public_empty
    monkeypatch.setattr(cuda_ops, "_empty", cuda_ops._choose_empty())
    torch.manual_seed(0)
    for (call, shapes), _ in zip(calls(), want):
        assert [tuple(t.shape) for t in call()] == [s for s, _ in shapes]
