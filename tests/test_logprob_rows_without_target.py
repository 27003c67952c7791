"""Rows without a target: no gradient reaches them, whatever their logits hold; with a gradient of the entropy they have that alone."""

import math

import pytest
import torch

import packed_oracles as ref
from dual_mod_public_b200.ops import token_logprobs

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [1, 50, 3001])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_padding_rows(dev, dtype, V, bad):
    clean = torch.randn(6, V, generator=torch.Generator().manual_seed(V)).to(dev, dtype)
    y = torch.tensor([0, -1, V // 2, -7, V - 1, -1], device=dev)
    x = clean.clone()
    x[1] = bad
    x[3, V // 3] = bad
    x.requires_grad_()
    r = token_logprobs(x, y)
    assert torch.equal(r.logp[[1, 3, 5]], torch.zeros(3, device=dev))
    dx, = torch.autograd.grad(r.logp.sum(), x, retain_graph=True)
    assert not dx[[1, 3, 5]].any()
    want = ref.logprobs(clean, y, 0, torch.ones(6, device=dev))["dx"]
    bound = 2.0 ** -20 + (ref.u_of(dtype) + 2.0 ** -20) * want.abs()        # p <= 1 in fp32, one rounding
    ref.close(dx, (want, bound), "dx")
    # a weight of zero for the padding rows' entropy, as a masked mean gives it
    keep = (y >= 0).float()
    both, = torch.autograd.grad((r.logp, r.entropy), x, (keep, keep), retain_graph=True)
    assert not both[[1, 3, 5]].any() and both[[0, 2, 4]].isfinite().all()
    # the entropy's own gradient stays: NaN for a row that has none
    h, = torch.autograd.grad(r.entropy.sum(), x)
    assert h[1].isnan().all()
    alone = ref.logprobs(clean, y, 0, None, torch.ones(6, device=dev))["dx"]
    ref.close(h[5], (alone[5], 2.0 ** -17 + (ref.u_of(dtype) + 2.0 ** -20) * alone[5].abs()), "entropy")
