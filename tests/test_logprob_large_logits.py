"""Token scores of rows with large finite logits: masks of -1e9, -1e10, -1e20 and the like, as part of a row, as all that some
of the threads of a row meet, as whole rows; and large positive entries."""

import pytest
import torch

import packed_oracles as ref
from dual_mod_public_b200.ops import token_logprobs

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]
MASKS = [-1e8, -9.9e8, -1e9, -1.01e9, -2e9, -1e10, -1e12, -1e20, -9e29, -1e31]


def rows_of(mask, n, V, dev, dtype):
    """Rows that differ in what is masked: the front, the back, all but a few entries, every second one, all but the last, all."""
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(n, V, generator=g) * 3).to(dev)
    i = torch.arange(V, device=dev)
    keep = [i >= V // 2, i < (V + 1) // 2, i % 97 == 5 % V, i % 2 == 0, i == V - 1, i < 0]
    for r in range(n):
        x[r] = torch.where(keep[r % len(keep)], x[r], mask)
    return x.to(dtype)


def bounds(x, V):
    """Per row: of a log probability and of the entropy.  2^-24 for every operation on a sum S of the row or its logarithm: at most
    V / 256 + 16 additions in a tree, the exponentials 2 ulp each, differences of values of at most the live entries' range R.  The entropy's sum is
    formed with exponents relative to a whole number next to the maximum in units of log 2, as near as fp32 values of that size lie: t of
    them, so its sum cancels down from t S."""
    xf = x.double()
    m = xf.amax(-1, keepdim=True)
    live = xf - m > -200
    r = (m - torch.where(live, xf, torch.inf).amin(-1, keepdim=True)).squeeze(-1) + 12
    b = (r * 8 + V / 256 + 20) * 2.0 ** -24
    t = (m.squeeze(-1).abs() * 1.4427 * 2.0 ** -24).clamp(max=64) + 1
    return b, 4 * b + t * (V / 256 + 40) * 2.0 ** -24


def check(x, y, top):
    V = x.shape[1]
    n = len(y)
    gl, gh = (torch.randn(n, generator=torch.Generator().manual_seed(s)).to(x.device) for s in (5, 6))
    x = x.clone().requires_grad_()
    r = token_logprobs(x, y, top=top)
    dx, = torch.autograd.grad((r.logp, r.entropy), x, (gl, gh))
    x = x.detach()
    want = ref.logprobs(x, y, top, gl, gh)
    b, bh = bounds(x, V)
    rel = lambda lp: 2.0 ** -22 * lp.abs()                       # two roundings of the value itself
    ref.close(r.logp, (want["logp"], b + rel(want["logp"])), "logp")
    ref.close(r.entropy, (want["entropy"], bh), "entropy")
    if top:
        assert torch.equal(r.top_ids, want["top_ids"])
        ref.close(r.top_logp, (want["top_logp"], b[:, None] + rel(want["top_logp"])), "top_logp")
    lp = torch.log_softmax(x.double(), -1)
    p, lp = lp.exp(), lp.clamp(min=-1000.0)
    far = (lp + want["entropy"][:, None]).abs()
    d = b[:, None] + rel(lp)                                     # of lp, so relative of p
    gl, gh = gl.abs().double()[:, None], gh.abs().double()[:, None]
    hot = torch.zeros_like(p).scatter_(-1, y.clamp_min(0)[:, None], 1.0)
    bound = (p * (gl * d + gh * (far * d + d + bh[:, None])) + 2.0 ** -22 * (gl * (p + hot) + gh * p * far)) * (1 + ref.u_of(x.dtype))
    ref.close(dx, (want["dx"], bound + ref.u_of(x.dtype) * want["dx"].abs() + 1e-30), "dx")


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("V, top", [(1, 0), (7, 1), (259, 8), (2047, 1), (2049, 0), (32001, 8)])
def test_masked_rows(dev, dtype, mask, V, top):
    x = rows_of(mask, 12, V, dev, dtype)
    y = torch.randint(0, V, (12,), generator=torch.Generator().manual_seed(1)).to(dev)
    y[4] = V - 1                                               # the only live entry; the others fall on live and masked ones
    y[7] = -1
    check(x, y, top)


@pytest.mark.gpu
@pytest.mark.parametrize("n, top", [(300, 0), (300, 8), (2400, 8), (4800, 1)])
def test_masked_rows_of_larger_batches(n, top):
    """Few and many threads per row."""
    x = rows_of(-1e10, n, 2053, "cuda:0", torch.float32)
    check(x, torch.arange(n, device="cuda:0") * 7 % 2053, top)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [5, 300, 5003])
def test_large_entries(dev, dtype, V):
    """Positive ones, alone and twice, and rows whose entries lie as near to one another as the type has them."""
    x = torch.randn(12, V, generator=torch.Generator().manual_seed(2)).to(dev)
    for r, big in enumerate((1e6, 1e8, 9e8, 1e9, 1.1e9, 2e9, 1e10, 1e20, 1e35)):
        x[r, r % V] = big
        x[r, V - 1] = big
    x = x.to(dtype)
    step = 2.0 ** 6 if dtype is torch.float32 else 2.0 ** 22
    x[9] = (1e9 - step * (torch.arange(V, device=dev) % 5)).to(dtype)
    x[10] = (-1e9 - step * (torch.arange(V, device=dev) % 3)).to(dtype)
    x[11] = (1e8 - 8 * (torch.arange(V, device=dev) % 7)).to(dtype)
    y = torch.arange(12, device=dev) % V
    check(x, y, min(5, V))
