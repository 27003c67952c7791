"""Attention over packed prompts, attention of single tokens over a cache, and log probabilities of given tokens.

What a language model needs to score, train on and answer sequences of different lengths without padding them:

  prompt   causal attention with grouped heads over sequences packed one behind the other (forward)
  train    the same with its gradients
  decode   one new token per sequence against a cache [batch, capacity, kv heads, head dim] with a length per sequence
  logp     log probability of a given token per row of logits, entropy of the row, its `top` largest entries
  logp_train   the same with the gradient of the logits

A case is a dict of plain sizes.  `prepare` makes its inputs, `run` is one pass (the plain form, or with `own` the
framework's kernels), `exact` the same from the definition in 64 bits, `work` what a pass has to read, write and compute.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- cases ----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # scoring a handful of short multiple-choice requests with the 340M shape: latency of a small call
        {"name": "prompt_short_requests", "op": "prompt", "dtype": "bf16", "tokens": 731, "seqs": 19, "hq": 16, "hkv": 16,
         "dim": 64, "window": 0, "cut": 1},
        # prompts of mixed lengths in one batch, grouped heads of 128: the ordinary prefill
        {"name": "prompt_mixed_grouped", "op": "prompt", "dtype": "bf16", "tokens": 8192, "seqs": 7, "hq": 16, "hkv": 4,
         "dim": 128, "window": 0, "cut": 2},
        # a long document behind a shorter one, 36 heads of 64, half precision
        {"name": "prompt_long_document", "op": "prompt", "dtype": "fp16", "tokens": 12289, "seqs": 2, "hq": 36, "hkv": 36,
         "dim": 64, "window": 0, "cut": 3},
        # a training step of the 340M baseline arm on documents packed to four rows of 2048
        {"name": "train_packed_340m", "op": "train", "dtype": "bf16", "tokens": 8192, "seqs": 11, "hq": 16, "hkv": 16,
         "dim": 64, "window": 0, "cut": 4},
        # a training step of the 1.3B baseline arm, grouped heads of 128, two long documents
        {"name": "train_long_grouped", "op": "train", "dtype": "bf16", "tokens": 8192, "seqs": 2, "hq": 16, "hkv": 4,
         "dim": 128, "window": 0, "cut": 5},
        # one token of one conversation: nothing but latency
        {"name": "decode_one_sequence", "op": "decode", "dtype": "bf16", "batch": 1, "capacity": 2048, "hq": 16, "hkv": 16,
         "dim": 64, "window": 0, "cut": 6},
        # a serving batch of the 1.3B shape with grouped heads and sequences of very different lengths
        {"name": "decode_serving_batch", "op": "decode", "dtype": "bf16", "batch": 64, "capacity": 8192, "hq": 16, "hkv": 4,
         "dim": 128, "window": 0, "cut": 7},
        # the sampler's report for a decode step of eight rows: chosen token, entropy, eight alternatives
        {"name": "logp_decode_step", "op": "logp", "dtype": "bf16", "rows": 8, "vocab": 32000, "top": 8},
        # scoring a batch of requests: log probability and whether the token is the greedy one
        {"name": "logp_score_batch", "op": "logp", "dtype": "bf16", "rows": 8191, "vocab": 32000, "top": 1},
        # a vocabulary of odd size in 32 bits, with alternatives
        {"name": "logp_odd_vocabulary", "op": "logp", "dtype": "fp32", "rows": 1021, "vocab": 50257, "top": 5},
        # the loss of a small fine-tuning micro-batch with an entropy term
        {"name": "logp_train_small", "op": "logp_train", "dtype": "fp32", "rows": 509, "vocab": 50257, "top": 0},
        # the loss of a full micro-batch of 4 x 2048 tokens
        {"name": "logp_train_batch", "op": "logp_train", "dtype": "bf16", "rows": 8192, "vocab": 32000, "top": 0},
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prompt", "train", "decode", "logp", "logp_train"])
    if op in ("prompt", "train"):
        hkv = rng.choice([1, 2, 3, 4, 8, 15, 16])
        group = rng.choice([g for g in (1, 2, 3, 4, 5, 8) if g * hkv <= 36])
        tokens = _log_uniform(rng, 64, 8192)
        return {"op": op, "dtype": "bf16" if op == "train" else rng.choice(["bf16", "bf16", "fp16"]), "tokens": tokens,
                "seqs": _log_uniform(rng, 1, max(1, min(64, tokens // 8))), "hq": min(16, hkv * group) // hkv * hkv,
                "hkv": hkv, "dim": rng.choice([64, 128]), "window": rng.choice([0, 0, 0, _log_uniform(rng, 16, 1024)]),
                "cut": rng.randrange(1 << 20)}
    if op == "decode":
        hkv = rng.choice([1, 2, 4, 8, 15, 16])
        group = rng.choice([g for g in (1, 2, 3, 4, 8) if g * hkv <= 36])
        capacity = _log_uniform(rng, 64, 8192)
        batch = _log_uniform(rng, 1, max(1, min(96, (64 * 8192 * 4 * 128) // (capacity * hkv * 128))))
        return {"op": op, "dtype": rng.choice(["bf16", "bf16", "fp16"]), "batch": batch, "capacity": capacity,
                "hq": hkv * group, "hkv": hkv, "dim": rng.choice([64, 128]),
                "window": rng.choice([0, 0, 0, _log_uniform(rng, 16, 1024)]), "cut": rng.randrange(1 << 20)}
    vocab = rng.choice([128, 259, 32000, 50257, _log_uniform(rng, 100, 65536)])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    rows = _log_uniform(rng, 1, max(1, min(16384, 8192 * 32000 // (vocab * (2 if dtype == "fp32" else 1)))))
    return {"op": op, "dtype": dtype, "rows": rows, "vocab": vocab,
            "top": 0 if op == "logp_train" else rng.choice([0, 1, 2, 5, 8, 20])}


def _sequence_lengths(case):
    """`seqs` lengths that sum to `tokens`, drawn from the case's own number (a sequence may have one token, or none)."""
    rng = random.Random(case["cut"])
    cuts = sorted(rng.randrange(case["tokens"] + 1) for _ in range(case["seqs"] - 1))
    edges = [0] + cuts + [case["tokens"]]
    return [b - a for a, b in zip(edges, edges[1:])]


def _cache_lengths(case):
    """A live length per sequence: from one row to the whole capacity."""
    rng = random.Random(case["cut"])
    if case["batch"] == 1:
        return [rng.randrange(case["capacity"] // 2, case["capacity"] + 1)]
    return [rng.randrange(1, case["capacity"] + 1) for _ in range(case["batch"])]


# ---- inputs -----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(std).to(dtype)

    op = case["op"]
    if op in ("prompt", "train"):
        t, d = case["tokens"], case["dim"]
        lengths = torch.tensor([0] + _sequence_lengths(case), dtype=torch.int64)
        state = {"case": case, "q": normal(t, case["hq"], d, std=1.5), "k": normal(t, case["hkv"], d, std=1.5),
                 "v": normal(t, case["hkv"], d), "cu": lengths.cumsum(0).to(torch.int32).cuda()}
        if op == "train":
            state["grad"] = normal(t, case["hq"], d)
            for name in ("q", "k", "v"):
                state[name].requires_grad_()
        return state
    if op == "decode":
        b, p, d = case["batch"], case["capacity"], case["dim"]
        return {"case": case, "q": normal(b, case["hq"], d, std=1.5), "k": normal(b, p, case["hkv"], d, std=1.5),
                "v": normal(b, p, case["hkv"], d),
                "lengths": torch.tensor(_cache_lengths(case), dtype=torch.int32, device="cuda")}
    n, vocab = case["rows"], case["vocab"]
    logits = normal(n, vocab, std=2.5)
    # tokens as a model meets them: the ones of a text, likely under the model, here drawn from the softmax itself
    noise = torch.empty(n, vocab, device="cuda").exponential_(generator=gen).log_().neg_()
    tokens = noise.add_(logits).argmax(-1)
    state = {"case": case, "logits": logits, "tokens": tokens}
    if op == "logp_train":
        state["tokens"] = torch.where(torch.rand(n, generator=gen, device="cuda") < 0.05, -1, tokens)  # -1: no target
        state["logits"].requires_grad_()
        state["grad_logp"] = torch.randn(n, generator=gen, device="cuda").mul_(0.2).sub_(1.0)
        state["grad_entropy"] = torch.randn(n, generator=gen, device="cuda").mul_(0.1)
    return state


# ---- one pass -----------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _own(case, state)
    with torch.no_grad():
        return _plain(case, state)


def _own(case, s):
    from dual_mod_public_b200 import ops
    op = case["op"]
    if op == "prompt":
        return ops.packed_attention(s["q"], s["k"], s["v"], s["cu"], window=case["window"])
    if op == "train":
        o = ops.packed_attention(s["q"], s["k"], s["v"], s["cu"], window=case["window"])
        dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["grad"])
        return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}
    if op == "decode":
        return ops.cached_attention(s["q"], s["k"], s["v"], s["lengths"], window=case["window"])
    r = ops.token_logprobs(s["logits"], s["tokens"], top=case["top"])
    out = {"logp": r.logp.detach(), "entropy": r.entropy.detach()}
    if case["top"]:
        out |= {"top_logp": r.top_logp, "top_ids": r.top_ids}
    if op == "logp_train":
        out["dlogits"], = torch.autograd.grad((r.logp, r.entropy), s["logits"], (s["grad_logp"], s["grad_entropy"]))
    return out


def _packed_mask(cu, tokens, window):
    """[tokens, tokens]: the key is of the query's own sequence, not behind it and inside the window."""
    pos = torch.arange(tokens, device=cu.device)
    seq = torch.searchsorted(cu, pos, right=True)
    gap = pos[:, None] - pos[None, :]
    mask = (seq[:, None] == seq[None, :]) & (gap >= 0)
    return mask & (gap < window) if window else mask


def _plain(case, s):
    op = case["op"]
    if op in ("prompt", "train"):
        t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["dim"]
        dtype, g, scale = s["q"].dtype, hq // hkv, 1.0 / math.sqrt(d)
        mask = _packed_mask(s["cu"], t, case["window"])
        q = s["q"].float().view(t, hkv, g, d).permute(1, 2, 0, 3).reshape(hkv, g * t, d)     # [kv head, (group, row), dim]
        k, v = s["k"].float().transpose(0, 1), s["v"].float().transpose(0, 1)
        p = (q @ k.transpose(1, 2)).view(hkv, g, t, t).mul_(scale).masked_fill_(~mask, float("-inf"))
        p = p.sub_(p.amax(-1, keepdim=True)).exp_()
        p = p.div_(p.sum(-1, keepdim=True)).view(hkv, g * t, t)
        rows = lambda x: x.view(hkv, g, t, d).permute(2, 0, 1, 3).reshape(t, hq, d)
        o = p @ v
        if op == "prompt":
            return rows(o).to(dtype)
        do = s["grad"].float().view(t, hkv, g, d).permute(1, 2, 0, 3).reshape(hkv, g * t, d)
        dv = p.transpose(1, 2) @ do
        ds = (do @ v.transpose(1, 2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        dq, dk = ds @ k, ds.transpose(1, 2) @ q
        return {"o": rows(o).to(dtype), "dq": rows(dq).to(dtype), "dk": dk.transpose(0, 1).to(dtype),
                "dv": dv.transpose(0, 1).to(dtype)}
    if op == "decode":
        b, cap, hq, hkv, d = case["batch"], case["capacity"], case["hq"], case["hkv"], case["dim"]
        dtype, g = s["q"].dtype, hq // hkv
        pos, n = torch.arange(cap, device="cuda"), s["lengths"][:, None]
        mask = pos < n
        if case["window"]:
            mask = mask & (pos >= n - case["window"])
        q = s["q"].float().view(b, hkv, g, d)
        p = (q @ s["k"].float().permute(0, 2, 3, 1)).mul_(1.0 / math.sqrt(d)).masked_fill_(~mask[:, None, None], float("-inf"))
        p = p.sub_(p.amax(-1, keepdim=True)).exp_()
        p = p.div_(p.sum(-1, keepdim=True))
        return (p @ s["v"].float().transpose(1, 2)).reshape(b, hq, d).to(dtype)
    x = s["logits"].float()
    z = x - x.amax(-1, keepdim=True)
    e = z.exp()
    total = e.sum(-1, keepdim=True, dtype=torch.float64)
    log_total = total.log()
    lp = (z - log_total).float()
    p = (e / total).float()
    entropy = log_total.squeeze(-1) - (p * z).sum(-1, dtype=torch.float64)
    ok = s["tokens"] >= 0
    target = s["tokens"].clamp_min(0)[:, None]
    out = {"logp": torch.where(ok, lp.gather(-1, target).squeeze(-1), 0.0), "entropy": entropy.float()}
    if case["top"]:
        ids = x.sort(dim=-1, descending=True, stable=True).indices[:, :case["top"]]          # ties: the lowest index first
        out |= {"top_logp": lp.gather(-1, ids), "top_ids": ids}
    if op == "logp_train":
        g_lp = torch.where(ok, s["grad_logp"], 0.0)[:, None]
        grad = -p * (g_lp + s["grad_entropy"][:, None] * (lp + entropy.float()[:, None]))
        out["dlogits"] = grad.scatter_add_(-1, target, g_lp).to(s["logits"].dtype)
    return out


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] in ("prompt", "train"):
            return _exact_packed(case, s)
        if case["op"] == "decode":
            return _exact_decode(case, s)
        return _exact_logp(case, s)


def _exact_packed(case, s):
    """Sequence by sequence and head by head."""
    group, scale = case["hq"] // case["hkv"], case["dim"] ** -0.5
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    o = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    start = 0
    for n in _sequence_lengths(case):
        rows = slice(start, start + n)
        start += n
        if n == 0:
            continue
        i = torch.arange(n, device="cuda")
        seen = i[None, :] <= i[:, None]
        if case["window"]:
            seen &= i[None, :] > i[:, None] - case["window"]
        for h in range(case["hq"]):
            kh = h // group
            w = torch.softmax(torch.where(seen, q[rows, h] @ k[rows, kh].T * scale, -math.inf), dim=-1)
            o[rows, h] = w @ v[rows, kh]
            if case["op"] == "train":
                go = s["grad"][rows, h].double()
                dv[rows, kh] += w.T @ go
                gw = go @ v[rows, kh].T
                gs = w * (gw - (gw * w).sum(-1, keepdim=True)) * scale
                dq[rows, h] = gs @ k[rows, kh]
                dk[rows, kh] += gs.T @ q[rows, h]
    return {"o": o, "dq": dq, "dk": dk, "dv": dv} if case["op"] == "train" else o


def _exact_decode(case, s):
    group = case["hq"] // case["hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_cache_lengths(case)):
        first = max(0, n - case["window"]) if case["window"] else 0
        k, v = (s[c][b, first:n].double().repeat_interleave(group, dim=1) for c in ("k", "v"))
        w = torch.softmax(torch.einsum("hd,phd->hp", s["q"][b].double(), k) * case["dim"] ** -0.5, dim=-1)
        out[b] = torch.einsum("hp,phd->hd", w, v)
    return out


def _exact_logp(case, s):
    """In slabs of rows: 64 bits of a whole batch of logits would not be small."""
    parts = []
    slab = max(1, (1 << 27) // case["vocab"])
    for a in range(0, case["rows"], slab):
        x, y = s["logits"][a:a + slab].detach().double(), s["tokens"][a:a + slab]
        lp = torch.log_softmax(x, dim=-1)
        p = lp.exp()
        entropy = -(p * lp).sum(-1)
        has = (y >= 0).double()
        part = {"logp": lp[torch.arange(len(y), device="cuda"), y.clamp_min(0)] * has, "entropy": entropy}
        if case["top"]:
            part |= {"top_logp": lp.sort(dim=-1, descending=True).values[:, :case["top"]].clone(), "top_ids": None}
        if case["op"] == "logp_train":
            g = (s["grad_logp"][a:a + slab].double() * has)[:, None]
            hot = torch.zeros_like(p).scatter_(-1, y.clamp_min(0)[:, None], 1.0)
            part["dlogits"] = g * (hot - p) - s["grad_entropy"][a:a + slab].double()[:, None] * p * (lp + entropy[:, None])
        parts.append(part)
    return {n: None if parts[0][n] is None else torch.cat([part[n] for part in parts]) for n in parts[0]}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------
def _seen_pairs(n, window):
    """Query-key pairs of a causal sequence of n tokens."""
    w = min(window or n, n)
    return w * (w + 1) // 2 + (n - w) * w


def work(case):
    op = case["op"]
    if op in ("prompt", "train"):
        t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["dim"]
        pairs = hq * sum(_seen_pairs(n, case["window"]) for n in _sequence_lengths(case))
        rows_q, rows_kv = t * hq * d * 2, t * hkv * d * 2
        if op == "prompt":           # read q, k, v, write o; q k^T and p v
            return {"bytes": 2 * rows_q + 2 * rows_kv, "flops": 4 * pairs * d}
        # read q, k, v and the output's gradient, write o and three gradients; two products forward, four backward
        return {"bytes": 4 * rows_q + 4 * rows_kv, "flops": 12 * pairs * d}
    if op == "decode":
        rows = sum(min(n, case["window"] or n) for n in _cache_lengths(case))
        return {"bytes": 2 * rows * case["hkv"] * case["dim"] * 2 + 2 * case["batch"] * case["hq"] * case["dim"] * 2,
                "flops": 4 * rows * case["hq"] * case["dim"]}
    n, vocab, size = case["rows"], case["vocab"], 4 if case["dtype"] == "fp32" else 2
    small = n * (8 + 4 + 4 + 12 * case["top"])
    if op == "logp":                 # read the logits; maximum, exponential, two sums
        return {"bytes": n * vocab * size + small, "flops": 6 * n * vocab}
    return {"bytes": 2 * n * vocab * size + small + 8 * n, "flops": 12 * n * vocab}
