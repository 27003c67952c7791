"""Packed generation answers with the model's weights of the moment, also where it decodes from a copy of them."""

import pytest
import torch

from dual_mod_public_b200 import DualModConfig
from dual_mod_public_b200.eval.lm_eval_adapter import ByteTokenizer, DualModEval
from dual_mod_public_b200.models import DualModLM

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("dev", DEVICES)
def test_weights_changed_between_calls(dev):
    torch.manual_seed(0)
    m = DualModLM(DualModConfig(d_model=64, n_layers=1, n_heads=2, mlp_hidden_override=64, vocab_size=259, max_seq_len=64,
                                attn_mode="vanilla", dtype="fp32"))
    m = m if dev != "cpu" else m.bfloat16()                        # a type that the decoder does not compute in on this device
    adapter = lambda: DualModEval(packed=True, ckpt=None, tokenizer=ByteTokenizer(), model=m, device=dev, max_length=64, gen_rows=2)
    reqs = [("abc", {"until": [], "max_gen_toks": 8}), ("hello", {"until": [], "max_gen_toks": 8})]
    lm = adapter()
    first = lm._greedy_batch([[5, 6, 7], [9]], 8, [])
    assert next(lm._engines["packed"][0].m.parameters()).data_ptr() != next(m.parameters()).data_ptr()
    with torch.no_grad():
        for p in m.parameters():
            p.add_(torch.randn_like(p) * 0.3)
    second = lm._greedy_batch([[5, 6, 7], [9]], 8, [])
    assert second == adapter()._greedy_batch([[5, 6, 7], [9]], 8, []) and second != first
    assert len(lm.generate_until(reqs)) == 2


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("copied", [True, False])
def test_configuration_changed_between_calls(dev, copied):
    """A longer position table, then a window: the decoder follows, whether it computes from a copy of the model or from the model."""
    torch.manual_seed(0)
    m = DualModLM(DualModConfig(d_model=64, n_layers=1, n_heads=2, mlp_hidden_override=64, vocab_size=259, max_seq_len=64,
                                attn_mode="vanilla", dtype="fp32"))
    m = m.bfloat16() if copied == (dev == "cpu") else m
    adapter = lambda: DualModEval(packed=True, ckpt=None, tokenizer=ByteTokenizer(), model=m, device=dev, max_length=64, gen_rows=2)
    lm, short, long = adapter(), [[5, 6, 7], [9]], [list(range(3, 203)), [9]]
    lm._greedy_batch(short, 8, [])
    m.set_rope_len(1024)
    assert lm._greedy_batch(long, 300, []) == adapter()._greedy_batch(long, 300, [])
    assert lm._greedy_batch(short, 8, []) == adapter()._greedy_batch(short, 8, [])
    m.cfg.local_window = 3
    assert lm._greedy_batch(long, 8, []) == adapter()._greedy_batch(long, 8, [])
