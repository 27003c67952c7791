"""Token scores of rows with one entry far above the others: a log probability is never above zero, an entropy never below,
and both are right to a few fp32 roundings of one, as the sum of the row is little more than one."""

import pytest
import torch

import packed_oracles as ref
from dual_mod_public_b200.ops import token_logprobs

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


def peaked(n, V, margin, dev, dtype):
    """n rows around different offsets, the largest entry at a place of its own."""
    g = torch.Generator().manual_seed(V + margin)
    x = torch.randn(n, V, generator=g).clamp(-1.5, 1.5)
    at = torch.arange(n) * 5 % V
    x[torch.arange(n), at] = margin + 1.5
    return (x + torch.linspace(-30, 30, n)[:, None]).to(dtype).to(dev), at.to(dev)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("margin", [8, 12, 16, 24, 40])
@pytest.mark.parametrize("V, top", [(1, 0), (1, 1), (2, 1), (259, 2), (2049, 1), (32000, 2)])
def test_peaked_rows(dev, dtype, margin, V, top):
    x, y = peaked(64, V, margin, dev, dtype)
    r = token_logprobs(x, y, top=top)
    assert (r.logp <= 0).all() and (r.entropy >= 0).all() and (top == 0 or (r.top_logp <= 0).all())
    want = ref.logprobs(x, y, top)
    # Additions onto a partial sum that holds the largest entry, each off by at most 2^-24 of it: 16 of a set of vectors, one per set that
    # follows (of the at least 32 x 16 entries that a row's threads take at a time), the row's edges, the joins of a tree of 10.
    n = 32 + V / 512
    b = n * 2.0 ** -24 + 2.0 ** -22 * want["logp"].abs()
    ref.close(r.logp, (want["logp"], b), "logp")
    # its sum cancels down from t S with |t| <= 1, in units of log 2; then the difference of two values below 2^-10 x 12
    ref.close(r.entropy, (want["entropy"], 3 * n * 2.0 ** -24 + 2.0 ** -22 * want["entropy"]), "entropy")
    if top:
        ref.close(r.top_logp[:, 0], (want["top_logp"][:, 0], b), "top_logp")


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_signs_over_ordinary_rows(dev, dtype):
    g = torch.Generator().manual_seed(3)
    for V in (1, 2, 3, 100, 3001):
        for std in (0.01, 1.0, 10.0, 100.0):
            x = (torch.randn(200, V, generator=g) * std).to(dtype).to(dev)
            r = token_logprobs(x, torch.arange(200, device=dev) % V, top=1)
            assert (r.logp <= 0).all() and (r.entropy >= 0).all() and (r.top_logp <= 0).all()
            assert r.top_logp.isfinite().all()
