"""A row of logits may have as many columns as the kernel can number in 32 bits, with the threads that reach past its end; more are refused.
No row of that size is read here."""

import pytest
import torch

from dual_mod_public_b200.ops import token_logprobs
from dual_mod_public_b200.ops.packed import MAX_VOCAB

TOP = (1 << 31) - 1


def last_column(V, head, width, threads):
    """The largest column number that the kernels form for a row: that of the last thread behind the vectors."""
    return head + (V - head) // width * width + threads - 1


@pytest.mark.parametrize("threads", [32, 64, 128, 256, 1024])
@pytest.mark.parametrize("width", [4, 8])
def test_numbers_fit_at_the_limit(threads, width):
    for head in range(width):
        assert last_column(MAX_VOCAB, head, width, threads) <= TOP
    ahead = MAX_VOCAB // width + 1 + 4 * 4 * threads                       # vectors: two sets of four requested ahead
    assert ahead <= TOP
    assert last_column(TOP, 0, width, 32) > TOP                            # the limit that was: 2^31 - 1


def test_wider_rows_are_refused():
    for V in (MAX_VOCAB + 1, TOP, TOP + 1):
        with pytest.raises(ValueError):
            token_logprobs(torch.zeros(1, 1).expand(1, V), torch.zeros(1, dtype=torch.int64))
