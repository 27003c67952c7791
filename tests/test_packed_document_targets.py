"""Packed training: no document is asked for a token of the next one, and a batch without targets trains nothing."""

import torch

from dual_mod_public_b200 import DualModConfig
from dual_mod_public_b200.models import DualModLM
from dual_mod_public_b200.train import train_baseline as TB

EOS = 3


def tiny():
    torch.manual_seed(0)
    return DualModLM(DualModConfig(d_model=32, n_layers=1, n_heads=4, mlp_hidden_override=64, vocab_size=50, max_seq_len=16,
                                   attn_mode="vanilla", dtype="fp32"))


def loss_of(m, rows):
    """As the trainer forms it, of rows [B, T + 1]."""
    x, y = rows[:, :-1], rows[:, 1:]
    return m(x.reshape(-1), targets=TB.document_targets(x, y, EOS).reshape(-1), cu_seqlens=TB.document_edges(x, EOS))[1]


def test_targets_end_with_their_document():
    x = torch.tensor([[5, EOS, 7, 8], [9, EOS, EOS, 4]])
    y = torch.tensor([[EOS, 7, 8, EOS], [EOS, EOS, 4, 6]])
    assert TB.document_targets(x, y, EOS).tolist() == [[EOS, -1, 8, EOS], [EOS, -1, -1, 6]]
    assert torch.equal(TB.document_targets(x, y, 40), y)


def test_packed_loss_is_that_of_the_documents_alone():
    m = tiny()
    a, b = torch.tensor([4, 9, 11, 8, EOS]), torch.tensor([21, 30, 5, 7, 41, 6])
    rows = torch.cat((a, b))[None]
    alone = lambda d: torch.nn.functional.cross_entropy(m(d[None, :-1])[0][0], d[1:], reduction="sum")
    torch.testing.assert_close(loss_of(m, rows), (alone(a) + alone(b)) / 9, rtol=1e-5, atol=1e-6)
    other = rows.clone()
    other[0, 5:] = torch.tensor([7, 7, 2, 1, 0, 9])                  # the document behind the first one
    torch.testing.assert_close(loss_of(m, other), (alone(a) + alone(other[0, 5:])) / 9, rtol=1e-5, atol=1e-6)


def test_a_batch_of_nothing_but_ends_trains_nothing():
    m = tiny()
    loss = loss_of(m, torch.full((2, 9), EOS))
    loss.backward()
    assert loss.item() == 0.0 and all(p.grad is None or not p.grad.any() for p in m.parameters())


def test_the_trainer_uses_them(tmp_path, monkeypatch):
    seen, inner = [], DualModLM.forward

    def forward(self, idx, targets=None, **kw):
        seen.append((idx, targets))
        return inner(self, idx, targets=targets, **kw)
    monkeypatch.setattr(DualModLM, "forward", forward)
    TB.main(["--arch", "vanilla", "--shape", "32,1,4,64", "--vocab", "8", "--seq_len", "16", "--global_batch", "4", "--micro_batch", "2",
             "--total_steps", "2", "--synthetic", "--device", "cpu", "--out_dir", str(tmp_path), "--packed_docs", "--eos_id", str(EOS)])
    assert len(seen) == 4 and sum(int((x == EOS).sum()) for x, _ in seen) > 0
    for x, y in seen:
        assert torch.equal(y < 0, x == EOS)
