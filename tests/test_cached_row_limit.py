"""A cache may have as many rows as the kernel can share out with 32-bit row numbers: its arithmetic, restated, at the limit; more are
refused.  No cache of that size is read here."""

import pytest
import torch

from dual_mod_public_b200.ops import cached_attention
from dual_mod_public_b200.ops.packed import MAX_CACHE

TOP = (1 << 31) - 1


def shares(length, window, blocks, keys):
    """(first, last) row of every block's share as the kernel forms them; every intermediate value has to be a 32-bit number."""
    def fits(v):
        assert -TOP - 1 <= v <= TOP, v
        return v
    first = max(0, length - window) if window else 0
    share = fits(fits(fits(length - first + blocks - 1) // blocks + keys - 1) // keys * keys)
    out = []
    for part in range(blocks):
        a = min(length, fits(first + fits(part * share)))
        b = min(length, fits(a + share))
        tiles = fits(b - a + keys - 1) // keys
        fits(a + (tiles + 2 * 4) * keys)                             # the loads run up to two rounds of four warps ahead
        out.append((a, b))
    return out


@pytest.mark.parametrize("blocks", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("keys", [16, 32])
@pytest.mark.parametrize("short", [0, 1, 15, 33, 4097])
@pytest.mark.parametrize("window", [0, 1, 1000, TOP])
def test_rows_are_shared_out_at_the_limit(blocks, keys, short, window):
    length = MAX_CACHE - short
    got = shares(length, window, blocks, keys)
    assert got[0][0] == (max(0, length - window) if window else 0) and got[-1][1] == length
    assert all(a[1] == b[0] for a, b in zip(got, got[1:]))


def test_the_old_limit_did_not_fit():
    with pytest.raises(AssertionError):
        shares(TOP, 0, 16, 32)


def test_larger_caches_are_refused():
    q, n = torch.zeros(1, 1, 8, dtype=torch.bfloat16), torch.ones(1, dtype=torch.int32)
    for rows in (MAX_CACHE + 1, TOP):
        cache = torch.zeros(1, dtype=torch.bfloat16).expand(1, rows, 1, 8)     # no memory behind it
        with pytest.raises(ValueError):
            cached_attention(q, cache, cache, n)
