"""Forward-mode derivatives are refused, on every device and with or without a reverse-mode gradient: the kernels see values
only, and a tangent that is dropped is a wrong derivative."""

import pytest
import torch
from torch.autograd import forward_ad

from dual_mod_public_b200.ops import cached_attention, packed_attention, token_logprobs

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


def calls(dev, dtype):
    """name -> (function, its differentiable arguments)"""
    rnd = lambda *s: torch.randn(s, generator=torch.Generator().manual_seed(len(s))).to(dev, dtype)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)
    y = torch.tensor([1, 2], device=dev)
    return {"packed": (lambda q, k, v: packed_attention(q, k, v, ints(0, 10)), [rnd(10, 2, 64), rnd(10, 1, 64), rnd(10, 1, 64)]),
            "cached": (lambda q, k, v: cached_attention(q, k, v, ints(4, 5)), [rnd(2, 2, 64), rnd(2, 6, 1, 64), rnd(2, 6, 1, 64)]),
            "scores": (lambda x: token_logprobs(x, y, top=1), [rnd(2, 50)])}


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("name", ["packed", "cached", "scores"])
def test_dual_inputs_are_refused(dev, dtype, name):
    fn, args = calls(dev, dtype)[name]
    for i in range(len(args)):
        for grad in (False, True):
            if grad and name == "cached":
                continue                                           # refused for its gradient already
            with forward_ad.dual_level():
                dual = list(args)
                dual[i] = forward_ad.make_dual(args[i].clone().requires_grad_(grad), torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError):
                    fn(*dual)
        with pytest.raises(NotImplementedError):
            torch.func.jvp(lambda t: fn(*args[:i], t, *args[i + 1:]), (args[i],), (torch.ones_like(args[i]),))
    with forward_ad.dual_level():
        fn(*args)                                                  # plain tensors inside a level are fine


@pytest.mark.parametrize("dev", DEVICES)
def test_a_tangent_that_another_level_closed_is_no_tangent(dev):
    fn, args = calls(dev, torch.bfloat16)["packed"]
    want = fn(*args)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(args[0], torch.ones_like(args[0]))
    assert torch.equal(fn(dual, *args[1:]), want)
