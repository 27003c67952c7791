"""The paths that use the operators on packed sequences: the model's packed forward pass and its gradients against the
sequences one by one, generation for prompts of different lengths, the evaluation adapter and the baseline trainer."""

import json

import pytest
import torch

from dual_mod_public_b200 import DualModConfig
from dual_mod_public_b200.eval.lm_eval_adapter import ByteTokenizer, DualModEval
from dual_mod_public_b200.eval.packed_decode import PackedDecoder
from dual_mod_public_b200.models import DualModLM
from dual_mod_public_b200.train import train_baseline as TB

LENS = (1, 7, 20, 3)


def tiny(**kw):
    torch.manual_seed(0)
    base = dict(d_model=32, n_layers=2, n_heads=4, mlp_hidden_override=64, vocab_size=300, max_seq_len=64,
                attn_mode="vanilla", dtype="fp32")
    return DualModLM(DualModConfig(**{**base, **kw}))


def prompts(lens=LENS, vocab=300):
    g = torch.Generator().manual_seed(1)
    return [torch.randint(3, vocab, (n,), generator=g).tolist() for n in lens]


def edges(lens=LENS):
    return [0] + torch.tensor(lens).cumsum(0).tolist()


# fp32 on both sides, the same products in another order: single roundings of values of order one, some hundred of them
NEAR = dict(rtol=1e-4, atol=1e-5)

VARIANTS = [dict(), dict(n_kv_heads=2), dict(n_kv_heads=1, local_window=5), dict(attn_logn_ref=16), dict(v_norm="rms"),
            dict(use_rope=False)]


@pytest.mark.parametrize("kw", VARIANTS, ids=lambda k: ",".join(k) or "plain")
def test_packed_forward_equals_one_by_one(kw):
    m, seqs = tiny(**kw), prompts()
    flat = torch.tensor(sum(seqs, []))
    logits = m(flat, cu_seqlens=edges())[0]
    want = torch.cat([m(torch.tensor([s]))[0][0] for s in seqs])
    torch.testing.assert_close(logits, want, **NEAR)
    rows = torch.tensor([0, 7, 30])
    torch.testing.assert_close(m(flat[None], cu_seqlens=torch.tensor(edges(), dtype=torch.int32), logit_rows=rows)[0], want[rows], **NEAR)


@pytest.mark.parametrize("kw", VARIANTS[:4], ids=lambda k: ",".join(k) or "plain")
def test_packed_loss_and_gradients_equal_one_by_one(kw):
    m, seqs = tiny(**kw), prompts()
    flat = torch.tensor(sum(seqs, []))
    y = torch.roll(flat, -1)
    y[torch.tensor(edges()[1:]) - 1] = -1
    loss = m(flat, targets=y, cu_seqlens=edges())[1]
    got = torch.autograd.grad(loss, list(m.parameters()), allow_unused=True)
    total, n = 0.0, int((y >= 0).sum())
    for a, b in zip(edges(), edges()[1:]):
        if b - a > 1:
            lg = m(flat[None, a:b])[0][0]
            total = total + torch.nn.functional.cross_entropy(lg, y[a:b], ignore_index=-1, reduction="sum")
    want = torch.autograd.grad(total / n, list(m.parameters()), allow_unused=True)
    torch.testing.assert_close(loss, total / n, **NEAR)
    for a, b in zip(got, want):
        assert (a is None) == (b is None)
        if a is not None:
            torch.testing.assert_close(a, b, rtol=1e-3, atol=1e-6)


def test_packed_forward_refusals():
    m = tiny()
    flat = torch.zeros(10, dtype=torch.long)
    for bad in ([0, 5, 4], [0, 11], [-1, 5], [3]):
        with pytest.raises(ValueError):
            m(flat, cu_seqlens=bad)
    with pytest.raises(ValueError):
        m(torch.zeros(70, dtype=torch.long), cu_seqlens=[0, 65])          # longer than the RoPE table
    m(torch.zeros(130, dtype=torch.long), cu_seqlens=[0, 64, 128])        # many short ones may be
    dual = DualModLM(DualModConfig(d_model=32, n_layers=1, n_heads=4, mlp_hidden_override=64, vocab_size=50, max_seq_len=16))
    with pytest.raises(ValueError):
        dual(flat, cu_seqlens=[0, 10])
    with pytest.raises(ValueError):
        PackedDecoder(dual, 2, 8)


@pytest.mark.parametrize("kw", VARIANTS, ids=lambda k: ",".join(k) or "plain")
def test_packed_generation_is_greedy_decoding(kw):
    m, seqs = tiny(**kw), prompts()
    ids, logp = PackedDecoder(m, rows=6, capacity=40).generate(seqs, max_new=6)
    for s, got, lp in zip(seqs, ids, logp):
        want = list(s)
        for t, score in zip(got, lp):
            dist = torch.log_softmax(m(torch.tensor([want]))[0][0, -1], -1)
            assert t == int(dist.argmax()) and abs(score - float(dist.max())) < 1e-3
            want.append(t)
        assert len(got) == 6


def test_packed_generation_ends_rows():
    m, seqs = tiny(), prompts((5, 9))
    dec = PackedDecoder(m, rows=2, capacity=12)
    free = dec.generate(seqs, max_new=20)[0]
    assert [len(f) for f in free] == [8, 4]                               # a row ends with its cache: 12 - length + 1
    eos = free[0][2]
    cut = dec.generate(seqs, max_new=20, eos_id=eos)[0]
    assert cut[0] == free[0][:free[0].index(eos)]
    assert dec.generate(seqs, max_new=3, stop_fn=lambda ids: len(ids) == 2)[0] == [f[:2] for f in free]
    for bad in ([], [[]], [[1] * 13], [[1]] * 3):
        with pytest.raises(ValueError):
            dec.generate(bad, max_new=1)


def test_adapter_packed_equals_padded():
    m = tiny(vocab_size=300, max_seq_len=64)
    kw = dict(ckpt=None, tokenizer=ByteTokenizer(), model=m, device="cpu", max_length=64)
    plain, packed = DualModEval(**kw), DualModEval(packed=True, packed_tokens=40, **kw)
    reqs = [("The capital", " of"), ("", "abc"), ("x" * 80, "yz"), ("a", "b" * 30), ("q", "")]
    for (a, ga), (b, gb) in zip(plain.loglikelihood(reqs), packed.loglikelihood(reqs)):
        assert abs(a - b) < 1e-3 and ga == gb
    assert abs(plain.loglikelihood_rolling([("w" * 200,)])[0] - packed.loglikelihood_rolling([("w" * 200,)])[0]) < 1e-2
    gen = [("hello", {"until": ["\n"], "max_gen_toks": 5}), ("a longer prompt", {"until": ["\n"], "max_gen_toks": 5}),
           ("hello", {"until": [], "max_gen_toks": 3})]
    assert plain.generate_until(gen) == packed.generate_until(gen)
    dual = DualModLM(DualModConfig(d_model=32, n_layers=1, n_heads=4, mlp_hidden_override=64, vocab_size=300, max_seq_len=16))
    with pytest.raises(ValueError):
        DualModEval(packed=True, ckpt=None, tokenizer=ByteTokenizer(), model=dual, device="cpu")


def test_document_edges():
    x = torch.tensor([[5, 2, 7, 2], [9, 9, 9, 9]])
    assert TB.document_edges(x, 2).tolist() == [0, 2, 4, 8]
    assert TB.document_edges(x, 77).tolist() == [0, 4, 8]


def test_baseline_trainer_with_packed_documents(tmp_path):
    args = ["--arch", "vanilla", "--shape", "32,1,4,64", "--vocab", "50", "--seq_len", "16", "--global_batch", "4",
            "--micro_batch", "2", "--total_steps", "2", "--synthetic", "--device", "cpu", "--out_dir", str(tmp_path)]
    r = TB.main(args + ["--packed_docs", "--eos_id", "3"])
    assert r["loss"] == r["loss"]
    lines = [json.loads(x) for x in open(next(tmp_path.glob("*.jsonl")))]
    assert len(lines) >= 2
    for bad in (["--packed_docs"], ["--packed_docs", "--eos_id", "3", "--arch", "lstm"]):
        with pytest.raises(SystemExit):
            TB.main(args + bad)
