"""Scores far from zero: finite ones of up to 2^120 give the softmax that they have.  They are exact here, so the bound is that of
the rounded weights and outputs alone.  Gradients are NaN where fp32 does not hold a row's log sum to within an octave."""

import math

import pytest
import torch

import packed_oracles as ref
from dual_mod_public_b200.ops import cached_attention, packed_attention

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]
T, BASE, STEP = 400, 2.0 ** 30, 2.0 ** 8


def inputs(dev, dtype, dim, signs):
    """q . k = sign 2^30 + 2^8 {0 .. 4}: whole numbers that fp32 holds.  `signs`: per stretch of 37 keys, taken in turn."""
    q, k = torch.zeros(T, 2, dim), torch.zeros(T, 1, dim)
    q[:, :, 0], q[:, :, 1] = 2.0 ** 15, 2.0 ** 4
    i = torch.arange(T)
    k[:, 0, 0] = torch.tensor(signs)[i // 37 % len(signs)] * 2.0 ** 15
    k[:, 0, 1] = 2.0 ** 4 * (i * 3 % 5)
    v = torch.randn(T, 1, dim, generator=torch.Generator().manual_seed(1))
    return (x.to(dev, dtype) for x in (q, k, v))


def oracle(q, k, v, scale):
    """(o, bound) of one sequence in 64 bits.  A weight is off by u where it is rounded, by 2^-24 of its exponent for the factor, and by a
    few ulp of the exponential and the sums."""
    s = q[:, 0].double() @ k[:, 0].double().T * scale
    s = torch.where(torch.ones(T, T, device=q.device).tril().bool(), s, -math.inf)
    p, V, u = torch.softmax(s, -1), v[:, 0].double(), ref.u_of(q.dtype)
    far = torch.where(p > 0, p * (s.amax(-1, keepdim=True) - s).clamp(max=200.0), 0.0) * 2.0 ** -23
    o = (p @ V)[:, None].expand(T, 2, -1)
    b = (((u + 2.0 ** -20) * p + far) @ V.abs())[:, None] * (1 + u) + u * o.abs() + 1e-30
    return o, b


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [40, 64, 128])
@pytest.mark.parametrize("signs", [(1,), (-1,), (0, 1, -1), (-1, 0), (1, -1, 0)], ids=str)
@pytest.mark.parametrize("log_size", [10, 20, 22, 24, 25, 27, 30, 33, 60, 120])
def test_forward(dev, dtype, dim, signs, log_size):
    q, k, v = inputs(dev, dtype, dim, signs)
    scale = 2.0 ** (log_size - 30)
    o, bound = oracle(q, k, v, scale)
    cu = torch.tensor([0, T], dtype=torch.int32, device=dev)
    got = packed_attention(q, k, v, cu, scale=scale)
    ref.close(got, (o, bound), "packed")
    for n in (1, 38, 150, 300, 400):
        one = cached_attention(q[n - 1:n], k[None], v[None], torch.tensor([n], dtype=torch.int32, device=dev), scale=scale)
        ref.close(one, (o[n - 1:n], bound[n - 1:n]), f"cached {n}")
    v[300, 0, 3] = math.inf                                  # rows before it share blocks with it and do not see it
    v[301, 0, 3] = math.nan
    wild = packed_attention(q, k, v, cu, scale=scale)
    assert not wild[300:, :, 3].isfinite().any()
    ref.close(wild[:300], (o[:300], bound[:300]), "behind a non-finite value")


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("log_size", [25, 40])
def test_gradients_beyond_fp32_are_nan(dev, dim, dtype, log_size):
    """Of the sequence with such scores; the other one, in the same blocks of rows, has its gradients."""
    q, k, v = inputs(dev, dtype, dim, (1,))
    n = 190
    g = torch.Generator().manual_seed(2)
    scale = 2.0 ** (log_size - 30)
    unit = 1 / math.sqrt(scale * math.sqrt(dim))
    if dtype is torch.float16 and log_size == 40:
        unit = 2.0 ** -8
    for x, h in ((q, 2), (k, 1)):
        x[:n] = (torch.randn(n, h, dim, generator=g) * unit).to(dev, dtype)
    do = torch.randn(T, 2, dim, generator=g).to(dev, dtype)
    cu = torch.tensor([0, n, T], dtype=torch.int32, device=dev)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(packed_attention(*leaves, cu, scale=scale), leaves, do)
    alone = ref.packed(q[:n], k[:n], v[:n], cu[:2], scale=scale, do=do[:n])
    for got, name in zip(grads, ("dq", "dk", "dv")):
        assert got[n:].isnan().all(), name
        assert got[:n].isfinite().all(), name
        ref.close(got[:n], alone[name], name)
