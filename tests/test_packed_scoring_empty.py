"""Packed scoring of requests without tokens or without a continuation, alone and beside others."""

import pytest
import torch

from dual_mod_public_b200 import DualModConfig
from dual_mod_public_b200.eval.lm_eval_adapter import ByteTokenizer, DualModEval
from dual_mod_public_b200.models import DualModLM

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("dev", DEVICES)
def test_requests_without_tokens(dev):
    torch.manual_seed(0)
    m = DualModLM(DualModConfig(d_model=32, n_layers=1, n_heads=4, mlp_hidden_override=64, vocab_size=50, max_seq_len=16,
                                attn_mode="vanilla", dtype="fp32"))
    lm = DualModEval(packed=True, ckpt=None, tokenizer=ByteTokenizer(), model=m, device=dev, max_length=16)
    nothing = (0.0, True)
    assert lm._score_rows([]) == []
    for rows in ([([], 0)], [([], 0), ([], 0)], [([5], 0)], [([5], 0), ([], 0)]):
        got = lm._score_rows(rows)
        assert got == [nothing] * len(rows) and all(type(lp) is float for lp, _ in got)
    alone = lm._score_rows([([5, 6, 7], 2)])[0]
    assert lm._score_rows([([], 0), ([5, 6, 7], 2), ([], 0)]) == [nothing, alone, nothing] and alone[0] < 0
