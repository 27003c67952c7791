"""The torch statements of the operators on packed sequences against 64-bit ones and against differences, the arguments
that are refused, and the plan of the single-token kernel."""

import pytest
import torch

import packed_oracles as ref
from dual_mod_public_b200.ops import cached_attention, packed_attention, token_logprobs

F64_NEAR = dict(rtol=2e-5, atol=2e-5)          # fp32 statements of values of order one, sums of at most some hundred terms


def rnd(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("edges", [(0, 50), (0, 1, 1, 20, 50), (3, 10, 40), (0,), (0, 0)])
@pytest.mark.parametrize("window", [0, 1, 7])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 2), (6, 1)])
def test_packed_statement(edges, window, hq, hkv):
    T, d = 50, 8
    q, k, v = rnd(T, hq, d, seed=1), rnd(T, hkv, d, seed=2), rnd(T, hkv, d, seed=3)
    g = rnd(T, hq, d, seed=4)
    cu = torch.tensor(edges, dtype=torch.int32)
    want = ref.packed(q, k, v, cu, window, do=g)
    for x in (q, k, v):
        x.requires_grad_()
    o = packed_attention(q, k, v, cu, window=window)
    grads = torch.autograd.grad(o, (q, k, v), g)
    for got, name in zip((o, *grads), ("o", "dq", "dk", "dv")):
        torch.testing.assert_close(got.double(), want[name][0], **F64_NEAR)


def test_packed_padding_is_not_read():
    q, k, v, g = (rnd(20, 2, 8, seed=s) for s in range(4))
    cu = torch.tensor([2, 15], dtype=torch.int32)
    want = ref.packed(q, k, v, cu, do=g)
    for x in (q, k, v, g):
        x[:2], x[15:] = float("nan"), float("inf")
    for x in (q, k, v):
        x.requires_grad_()
    o = packed_attention(q, k, v, cu)
    for got, name in zip((o, *torch.autograd.grad(o, (q, k, v), g)), ("o", "dq", "dk", "dv")):
        torch.testing.assert_close(got.double(), want[name][0], **F64_NEAR)


def test_packed_nonfinite_value_reaches_the_rows_that_see_it():
    q, k, v = (rnd(20, 2, 8, seed=s) for s in range(3))
    cu = torch.tensor([0, 8, 20], dtype=torch.int32)
    want = ref.packed(q, k, v, cu, window=4)["o"][0]
    v[5, 1, 3] = float("inf")
    o = packed_attention(q, k, v, cu, window=4)
    sees = torch.zeros(20, 2, 8, dtype=torch.bool)
    sees[5:8, 1, 3] = True
    assert not o[sees].isfinite().any()
    torch.testing.assert_close(o[~sees].double(), want[~sees], **F64_NEAR)


@pytest.mark.parametrize("window", [0, 1, 6])
def test_cached_statement(window):
    q, k, v = rnd(5, 4, 8, seed=1), rnd(5, 30, 2, 8, seed=2), rnd(5, 30, 2, 8, seed=3)
    n = torch.tensor([30, 0, 1, 17, 99], dtype=torch.int32)
    want = ref.cached(q, k, v, n, window)[0]
    k[3, 17:] = float("nan")
    v[3, 17:] = float("nan")
    torch.testing.assert_close(cached_attention(q, k, v, n, window=window).double(), want, **F64_NEAR)


def test_cached_empty():
    e = torch.empty(2, 0, 2, 8)
    assert not cached_attention(rnd(2, 4, 8), e, e, torch.zeros(2, dtype=torch.int32)).any()
    assert cached_attention(rnd(0, 4, 8), e[:0], e[:0], torch.zeros(0, dtype=torch.int32)).shape == (0, 4, 8)


@pytest.mark.parametrize("V", [1, 3, 50])
@pytest.mark.parametrize("lead", [(7,), (2, 3), ()])
def test_logprobs_statement(V, lead):
    x, n = rnd(*lead, V, seed=1) * 3, 1
    for s in lead:
        n *= s
    y = (torch.arange(n) % V).view(lead)
    if n > 1:
        y.view(-1)[1] = -1
    top = min(3, V)
    gl, gh = rnd(*lead, seed=2), rnd(*lead, seed=3)
    x.requires_grad_()
    r = token_logprobs(x, y, top=top)
    dx, = torch.autograd.grad((r.logp, r.entropy), x, (gl, gh))
    want = ref.logprobs(x.reshape(-1, V), y.reshape(-1), top, gl.reshape(-1), gh.reshape(-1))
    torch.testing.assert_close(r.logp.double().reshape(-1), want["logp"], **F64_NEAR)
    torch.testing.assert_close(r.entropy.double().reshape(-1), want["entropy"], **F64_NEAR)
    torch.testing.assert_close(dx.double().reshape(-1, V), want["dx"], **F64_NEAR)
    assert torch.equal(r.top_ids.reshape(-1, top), want["top_ids"]) and r.top_logp.shape == (*lead, top)
    only, = torch.autograd.grad(token_logprobs(x, y).entropy, x, gh)
    torch.testing.assert_close(only.double().reshape(-1, V),
                               ref.logprobs(x.reshape(-1, V), y.reshape(-1), 0, None, gh.reshape(-1))["dx"], **F64_NEAR)


def test_gradients_against_differences():
    """64-bit central differences of the oracle's loss against the oracle's own gradients (the formulas)."""
    T, d = 9, 4
    q, k, v, g = (rnd(T, h, d, seed=s).double() for h, s in ((2, 1), (1, 2), (1, 3), (2, 4)))
    cu = torch.tensor([0, 3, 9], dtype=torch.int32)
    want = ref.packed(q, k, v, cu, 2, do=g)
    loss = lambda: (ref.packed(q, k, v, cu, 2)["o"][0] * g).sum()
    for x, name in ((q, "dq"), (k, "dk"), (v, "dv")):
        flat = x.view(-1)
        for i in range(0, flat.numel(), 5):
            keep, eps = flat[i].item(), 1e-5
            flat[i] = keep + eps
            up = loss()
            flat[i] = keep - eps
            diff = (up - loss()) / (2 * eps)
            flat[i] = keep
            assert abs(diff - want[name][0].reshape(-1)[i]) < 1e-8
    x, y, gl, gh = rnd(3, 6, seed=1).double(), torch.tensor([2, -1, 5]), rnd(3, seed=2).double(), rnd(3, seed=3).double()
    dx = ref.logprobs(x, y, 0, gl, gh)["dx"]

    def score():
        r = ref.logprobs(x, y, 0)
        return (r["logp"] * gl + r["entropy"] * gh).sum()
    for i in range(18):
        flat = x.view(-1)
        keep, eps = flat[i].item(), 1e-5
        flat[i] = keep + eps
        up = score()
        flat[i] = keep - eps
        diff = (up - score()) / (2 * eps)
        flat[i] = keep
        assert abs(diff - dx.view(-1)[i]) < 1e-8


def test_attention_refusals():
    q, k, cu = rnd(10, 4, 8), rnd(10, 2, 8), torch.tensor([0, 10], dtype=torch.int32)
    bad = [
        (TypeError, (q.double(), k.double(), k.double(), cu), {}),
        (TypeError, (q, k.bfloat16(), k, cu), {}),
        (TypeError, (q, k, k, cu.long()), {}),
        (TypeError, (q, k, k, cu[None]), {}),
        (TypeError, (q, k, k, [0, 10]), {}),
        (ValueError, (q[0], k, k, cu), {}),
        (ValueError, (q, k, k[:, :1], cu), {}),
        (ValueError, (q, k[:9], k[:9], cu), {}),
        (ValueError, (q, k[..., :4], k[..., :4], cu), {}),
        (ValueError, (q[:, :3], k, k, cu), {}),
        (ValueError, (q, k[:, :0], k[:, :0], cu), {}),
        (ValueError, (q, k, k, cu[:0]), {}),
        (ValueError, (q, k, k, cu), {"window": -1}),
        (ValueError, (q, k, k, cu), {"window": 2.0}),
        (ValueError, (q, k, k, cu), {"scale": 0.0}),
        (ValueError, (q, k, k, cu), {"scale": float("nan")}),
        (ValueError, (q, k, k, cu.to("meta")), {}),
    ]
    for error, args, kw in bad:
        with pytest.raises(error):
            packed_attention(*args, **kw)
    kc, n = rnd(10, 6, 2, 8), torch.zeros(10, dtype=torch.int32)
    for error, args, kw in [
        (TypeError, (q, kc, kc, n.long()), {}),
        (ValueError, (q, kc, kc, n[:9]), {}),
        (ValueError, (q, k, k, n), {}),
        (ValueError, (q[:9], kc, kc, n[:9]), {}),
        (ValueError, (q, kc, kc[:, :5], n), {}),
        (ValueError, (q.clone().requires_grad_(), kc, kc, n), {}),
        (ValueError, (q, kc, kc, n), {"scale": -1.0}),
        (ValueError, (torch.zeros(65536, 1, 8), torch.zeros(65536, 0, 1, 8), torch.zeros(65536, 0, 1, 8),
                      torch.zeros(65536, dtype=torch.int32)), {}),
    ]:
        with pytest.raises(error):
            cached_attention(*args, **kw)


def test_logprobs_refusals():
    x, y = rnd(4, 10), torch.zeros(4, dtype=torch.int64)
    for error, args, kw in [
        (TypeError, (x.double(), y), {}),
        (TypeError, (x, y.int()), {}),
        (TypeError, (x.long(), y), {}),
        (TypeError, (x, 3), {}),
        (ValueError, (x, y[:3]), {}),
        (ValueError, (x[:, :0], y), {}),
        (ValueError, (x, y), {"top": -1}),
        (ValueError, (x, y), {"top": 11}),
        (ValueError, (rnd(4, 100), y), {"top": 33}),
        (ValueError, (x, y.to("meta")), {}),
    ]:
        with pytest.raises(error):
            token_logprobs(*args, **kw)


def test_cache_blocks():
    """A power of two that the kernel takes, more of them for longer caches, one where the streams fill the device."""
    from dual_mod_public_b200.ops.cuda_ops import CudaOps
    for streams in (1, 2, 16, 147, 148, 5000):
        got = [CudaOps.cache_blocks(streams, n) for n in (0, 1, 256, 257, 2048, 5000, 1 << 20)]
        assert got == sorted(got) and set(got) <= {1, 2, 4, 8, 16} and got[0] == 1 and got[-1] == 16
    assert CudaOps.cache_blocks(148, 2048) == 1 and CudaOps.cache_blocks(16, 2048) == 8
