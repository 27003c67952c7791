"""Infinite scores inside a sequence: a score of +inf makes the row NaN, one of -inf has weight zero, and a row whose scores
all are -inf is zero like a row that sees no key.  The same on the torch statements and on the kernels."""

import math

import pytest
import torch

import packed_oracles as ref
from dual_mod_public_b200.ops import cached_attention, default_ops, packed_attention

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


def rnd(*shape, seed, dev, dtype):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dev, dtype)


def inputs(dev, dtype, dim, T=400):
    """q, k, v of one key head; the first dim of every query is a whole number of either sign, never zero."""
    q, k, v = (rnd(T, h, dim, seed=s, dev=dev, dtype=dtype) for h, s in ((2, 1), (1, 2), (1, 3)))
    q[:, :, 0] = torch.where(torch.arange(T) % 3 == 1, -1.0, 1.0).to(dev, dtype)[:, None]
    return q, k, v


def softmax_without(q, k, v, key):
    """64 bits, one sequence, causal, `key` hidden from all rows: o [T, Hq, D] and a bound on the kernels' roundings, the one
    of `packed_oracles.packed` (zero for a row that then sees nothing)."""
    T, Hq, D = q.shape
    scale, u = 1.0 / math.sqrt(D), ref.u_of(q.dtype)
    seen = torch.ones(T, T, device=q.device).tril().bool()
    seen[:, key] = False
    K, V = k[:, 0].double(), v[:, 0].double()
    K[key] = 0
    o, b = torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device), torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device)
    for h in range(Hq):
        Q = q[:, h].double()
        p = torch.softmax(torch.where(seen, Q @ K.T * scale, -math.inf), -1).nan_to_num(0.0)
        f32 = 4 * (D + 8) * 2.0 ** -24 * scale * (Q.abs() @ K.abs().T).max().item() + 2.0 ** -20
        o[:, h] = p @ V
        b[:, h] = ((u + f32) * (p @ V.abs()) + u * o[:, h].abs()) * (1 + u) + 1e-30
    return o, b


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [40, 64, 128])
@pytest.mark.parametrize("key", [0, 6, 7, 134, 255, 399])
def test_one_infinite_key(dev, dtype, dim, key):
    q, k, v = inputs(dev, dtype, dim)
    k[key, 0, 0] = math.inf
    cu = torch.tensor([0, 400], dtype=torch.int32, device=dev)
    want, bound = softmax_without(q, k, v, key)
    infinite = (q[:, :, 0] > 0) & (torch.arange(400, device=dev) >= key)[:, None]       # [T, Hq]
    o, lse = default_ops(q.device).packed_attn_fwd(q, k, v, cu, 0, 1.0 / math.sqrt(dim))
    assert torch.equal(o.isnan(), infinite[..., None].expand_as(o))
    assert torch.equal(lse.isnan(), infinite.T)
    ref.close(torch.where(infinite[..., None], want.to(dtype), o), (want, bound), "o")
    public = packed_attention(q, k, v, cu)
    assert torch.equal(public.nan_to_num(7.0), o.nan_to_num(7.0))
    # the last row as a single token over a cache
    one = cached_attention(q[-1:], k[None], v[None], torch.tensor([400], dtype=torch.int32, device=dev))
    assert torch.equal(one.isnan(), infinite[-1:, :, None].expand_as(one))
    ref.close(torch.where(infinite[-1:, :, None], want[-1:].to(dtype), one), (want[-1:], bound[-1:]), "one token")


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [40, 64, 128])
@pytest.mark.parametrize("residual", [False, True])
def test_rows_of_nothing_but_minus_infinity(dev, dtype, dim, residual):
    """The second of two sequences: every key is -inf in the dim where the queries are 1.  Then also with one finite key at its
    start, behind whole blocks of such keys."""
    q, k, v = inputs(dev, dtype, dim)
    q[:, :, 0] = 1.0
    cu = torch.tensor([0, 40, 400], dtype=torch.int32, device=dev)
    base = packed_attention(q, k, v, cu)
    k[40:, 0, 0] = -math.inf
    fwd = lambda: default_ops(q.device).packed_attn_fwd(q, k, v, cu, 0, 1.0 / math.sqrt(dim), residual=residual)
    got = fwd()
    assert torch.equal(got[0][:40], base[:40]) and not got[0][40:].any()
    assert got[1][:, :40].isfinite().all() and (got[1][:, 40:] == -math.inf).all()
    if residual:
        assert not got[2][40:].any()
    k[40, 0, 0] = 0.5
    o, lse, *_ = fwd()
    assert torch.equal(o[:40], base[:40]) and torch.equal(o[40:], v[40].expand_as(o[40:]))     # a single weight of one
    assert lse.isfinite().all()
    n = torch.tensor([0, 5, 360], dtype=torch.int32, device=dev)
    caches = [x[40:][None].expand(3, -1, -1, -1).clone() for x in (k, v)]
    caches[0][:2, :, :, 0] = -math.inf
    one = cached_attention(q[:3], *caches, n)
    assert not one[:2].any() and torch.equal(one[2], v[40].expand_as(one[2]))
