"""The scores' factor: what fp32 cannot hold is refused, its smallest normal value is taken."""

import math

import pytest
import torch

from dual_mod_public_b200.ops import cached_attention, packed_attention

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


def calls(dev, dim):
    q, k, v = (torch.randn(200, h, dim, generator=torch.Generator().manual_seed(h)).to(dev, torch.bfloat16) for h in (2, 1, 1))
    cu = torch.tensor([0, 90, 200], dtype=torch.int32, device=dev)
    n = torch.tensor([150], dtype=torch.int32, device=dev)
    return (lambda s: packed_attention(q, k, v, cu, scale=s)), (lambda s: cached_attention(q[:1], k[None], v[None], n, scale=s)), v


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("scale", [1e-50, 2.0 ** -127, 2.0 ** 128, 1e39, 1e300, math.inf, -1.0, 0.0, math.nan])
def test_refused(dev, scale):
    for call in calls(dev, 64)[:2]:
        with pytest.raises(ValueError):
            call(scale)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
def test_smallest_is_the_mean(dev, dim):
    """Scores of zero: a row is the mean of the values that it sees."""
    packed, cached, v = calls(dev, dim)
    mean = lambda x: x.double().cumsum(0) / torch.arange(1, len(x) + 1, device=dev)[:, None, None]
    alone = mean(v)[149]
    want = torch.cat((mean(v[:90]), mean(v[90:])))
    bound = lambda x: 2.0 ** -8 * x.abs() + 1e-5               # weights of one are exact in 16 bits; sums in fp32, one rounding
    assert ((packed(2.0 ** -126).double() - want).abs() <= bound(want)).all()
    assert ((cached(2.0 ** -126).double() - alone).abs() <= bound(alone)).all()
