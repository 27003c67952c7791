"""A kernel that gave up on a pipeline wait leaves wrong outputs and a flag: generation, packed scoring and packed training read
the flag and raise before anything is answered or learned.  The flag is set on the host here; no kernel waits for it."""

import pytest
import torch

from dual_mod_public_b200 import DualModConfig
from dual_mod_public_b200.eval.lm_eval_adapter import ByteTokenizer, DualModEval
from dual_mod_public_b200.eval.packed_decode import PackedDecoder
from dual_mod_public_b200.models import DualModLM
from dual_mod_public_b200.ops import default_ops
from dual_mod_public_b200.train import train_baseline as TB

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


@pytest.fixture(params=DEVICES)
def dev(request):
    return request.param


@pytest.fixture
def flag(dev, monkeypatch):
    """flag(value) sets what `tc_check` of the device's table finds."""
    table = default_ops(torch.device(dev))
    if dev == "cpu":
        state = {"set": 0}

        def check():
            if state["set"]:
                raise RuntimeError("a pipeline wait ran out")
        monkeypatch.setattr(table, "tc_check", check)
        yield lambda value: state.update(set=value)
    else:
        yield lambda value: table._tc_err.fill_(value)
        table._tc_err.zero_()


def model(dev):
    torch.manual_seed(0)
    return DualModLM(DualModConfig(d_model=64, n_layers=1, n_heads=2, mlp_hidden_override=64, vocab_size=300, max_seq_len=64,
                                   attn_mode="vanilla", dtype="fp32")).to(dev)


def test_generation(dev, flag):
    dec = PackedDecoder(model(dev), rows=2, capacity=32)
    want = dec.generate([[1, 2, 3], [4]], 4)
    flag(1)
    with pytest.raises(RuntimeError):
        dec.generate([[1, 2, 3], [4]], 4)
    flag(0)
    assert dec.generate([[1, 2, 3], [4]], 4) == want


def test_scoring(dev, flag):
    lm = DualModEval(packed=True, ckpt=None, tokenizer=ByteTokenizer(), model=model(dev), device=dev, max_length=64)
    lm.loglikelihood([("a", "bc")])
    flag(1)
    with pytest.raises(RuntimeError):
        lm.loglikelihood([("a", "bc")])


def test_training(dev, flag, tmp_path, monkeypatch):
    """The step that finds the flag set does not change the weights."""
    seen = []
    step = torch.optim.AdamW.step
    monkeypatch.setattr(torch.optim.AdamW, "step", lambda self, *a, **k: (seen.append(1), step(self, *a, **k))[1])
    args = ["--arch", "vanilla", "--shape", "64,1,2,64", "--vocab", "50", "--seq_len", "16", "--global_batch", "4", "--micro_batch", "2",
            "--total_steps", "1", "--synthetic", "--device", "cpu" if dev == "cpu" else "", "--out_dir", str(tmp_path)]
    TB.main(args + ["--packed_docs", "--eos_id", "3"])
    assert len(seen) == 1
    flag(1)
    with pytest.raises(RuntimeError):
        TB.main(args + ["--packed_docs", "--eos_id", "3"])
    assert len(seen) == 1
    TB.main(args)                                                   # rows that are not packed use none of these kernels
    assert len(seen) == 2
