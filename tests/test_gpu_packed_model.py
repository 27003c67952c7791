"""The packed paths of the model on the kernels: forward and gradients under autocast against fp32, generation with and
without a recorded graph, the adapter."""

import pytest
import torch

from dual_mod_public_b200 import DualModConfig
from dual_mod_public_b200.models import DualModLM

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LENS = (1, 300, 129, 64, 17)
EDGES = [0] + torch.tensor(LENS).cumsum(0).tolist()


def model(**kw):
    torch.manual_seed(0)
    base = dict(d_model=256, n_layers=2, n_heads=4, n_kv_heads=2, mlp_hidden_override=512, vocab_size=515, max_seq_len=512,
                attn_mode="vanilla")
    return DualModLM(DualModConfig(**{**base, **kw})).to(DEV)


def tokens():
    return torch.randint(0, 515, (EDGES[-1],), generator=torch.Generator().manual_seed(1)).to(DEV)


def table():
    from dual_mod_public_b200.ops import default_ops
    return default_ops(torch.device(DEV))


@pytest.mark.parametrize("kw", [dict(), dict(local_window=40), dict(head_dim_override=128, n_kv_heads=1)])
def test_packed_forward_and_gradients_within_bf16_noise(kw):
    """Against the same model in fp32: no further off than the unpacked path is, which rounds at the same places (its
    attention is another kernel), with half as much again for that."""
    m, x = model(**kw), tokens()
    y = torch.roll(x, -1)
    y[torch.tensor(EDGES[1:], device=DEV) - 1] = -1
    n = (y >= 0).sum()

    def one_by_one():
        total = 0.0
        for a, b in zip(EDGES, EDGES[1:]):
            if b - a > 1:
                total = total + torch.nn.functional.cross_entropy(m(x[None, a:b])[0][0].float(), y[a:b], ignore_index=-1, reduction="sum")
        return total / n
    grads = lambda loss: [g.float() for g in torch.autograd.grad(loss, list(m.parameters()))]
    exact_loss = one_by_one()
    exact = grads(exact_loss)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        plain = grads(one_by_one())
    before, count = dict(table().fallbacks), table().launches
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = m(x, targets=y, cu_seqlens=EDGES)[1]
    got = grads(loss)
    assert table().fallbacks == before and table().launches - count == 2 * 2 + 2       # per layer two, two of the scores
    table().tc_check()
    assert abs(loss.item() - exact_loss.item()) < 2e-2
    off = lambda g: torch.cat([(a - b).reshape(-1) for a, b in zip(g, exact)]).norm()
    assert off(got) <= 1.5 * off(plain)


def test_generation_with_a_graph_equals_without():
    from dual_mod_public_b200.eval.packed_decode import PackedDecoder
    m = model().bfloat16()
    m.rope_cos, m.rope_sin = (t.float() for t in (m.rope_cos, m.rope_sin))
    prompts = [tokens()[a:b].tolist() for a, b in zip(EDGES, EDGES[1:])]
    eager, graph = PackedDecoder(m, 6, 512), PackedDecoder(m, 6, 512)
    graph.prefill(prompts[:2])
    graph.capture()                                       # in the middle of a generation: caches and lengths are kept
    a, b = eager.generate(prompts, 12), graph.generate(prompts, 12)
    assert a == b
    # At another place in the pack a sequence's keys fall into other blocks of 128 rows, so its fp32 sums associate otherwise
    # and bf16 values next to a rounding border fall to the other side: not the same bits, but the same first score within
    # the rounding of its bf16 logit (order 2: 2^-7) and of the hidden state that made it, once in each run.
    first = [s[0] for s in a[1]]
    turned = [s[0] for s in graph.generate(prompts[::-1], 12)[1]][::-1]
    assert all(abs(x - y) < 4 * 2.0 ** -7 for x, y in zip(first, turned))


def test_adapter_packed_scores():
    """Padded and packed scoring of the same requests: two bf16 paths, each within its noise of the other."""
    from dual_mod_public_b200.eval.lm_eval_adapter import ByteTokenizer, DualModEval
    kw = dict(ckpt=None, tokenizer=ByteTokenizer(), model=model(), device=DEV, max_length=512)
    plain, packed = DualModEval(**kw), DualModEval(packed=True, packed_tokens=600, **kw)
    reqs = [("The capital of France", " is Paris"), ("", "abc"), ("x" * 400, "y" * 40), ("a", "b" * 100)]
    for (a, _), (b, _), (_, cont) in zip(plain.loglikelihood(reqs), packed.loglikelihood(reqs), reqs):
        # logits of order 1 rounded to bf16 (2^-8 relative each, two paths): below 2^-6 per scored token
        assert abs(a - b) < len(cont) * 2.0 ** -6
    gen = [("hello", {"until": ["\n"], "max_gen_toks": 5}), ("a longer prompt", {"until": ["\n"], "max_gen_toks": 5})]
    assert all(isinstance(t, str) for t in packed.generate_until(gen))


def test_packed_training_step_updates():
    """Two optimizer steps on packed documents: finite, and the second loss on the same documents is another one."""
    m, x = model(), tokens()
    opt = torch.optim.AdamW(m.parameters(), lr=1e-3)
    y = torch.roll(x, -1)
    y[torch.tensor(EDGES[1:], device=DEV) - 1] = -1
    cu = torch.tensor(EDGES, dtype=torch.int32, device=DEV)
    losses = []
    for _ in range(2):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = m(x, targets=y, cu_seqlens=cu)[1]
        opt.zero_grad()
        loss.backward()
        assert all(p.grad.isfinite().all() for p in m.parameters())
        opt.step()
        losses.append(loss.item())
    assert all(v == v for v in losses) and losses[0] != losses[1]
