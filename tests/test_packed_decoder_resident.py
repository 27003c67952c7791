"""Packed generation over prompts of very different lengths holds one decoder, and one copy of the weights, at a time."""

import gc
import weakref

import pytest
import torch

from dual_mod_public_b200 import DualModConfig
from dual_mod_public_b200.eval import packed_decode
from dual_mod_public_b200.eval.lm_eval_adapter import ByteTokenizer, DualModEval
from dual_mod_public_b200.models import DualModLM

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("dev", DEVICES)
def test_one_decoder_at_a_time(dev, monkeypatch):
    torch.manual_seed(0)
    m = DualModLM(DualModConfig(d_model=64, n_layers=1, n_heads=2, mlp_hidden_override=64, vocab_size=259, max_seq_len=1024,
                                attn_mode="vanilla", dtype="fp32"))
    made, weights, most = [], set(), [0]
    inner = packed_decode.PackedDecoder.__init__

    def init(self, *a, **k):
        gc.collect()
        most[0] = max(most[0], 1 + sum(r() is not None for r in made))
        made.append(weakref.ref(self))
        inner(self, *a, **k)
        weights.add(next(self.m.parameters()).data_ptr())
    monkeypatch.setattr(packed_decode.PackedDecoder, "__init__", init)
    lm = DualModEval(packed=True, ckpt=None, tokenizer=ByteTokenizer(), model=m, device=dev, max_length=1024, gen_rows=2)
    kw = {"until": [], "max_gen_toks": 4}
    reqs = [("a" * n, kw) for n in (600, 3, 300, 900, 5, 301, 620, 901)]
    texts = lm.generate_until(reqs)
    assert len(made) == 4 and most[0] == 1 and len(weights) == 1            # caches of 256, 512, 768 and 1024 entries
    if dev == "cpu":                                                         # fp32: no other rounding in another batch
        lm._gcache.clear()
        assert [lm.generate_until([r])[0] for r in reqs] == texts
        assert most[0] == 1 and len(weights) == 1
