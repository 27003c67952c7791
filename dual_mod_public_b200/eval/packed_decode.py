"""Greedy generation for prompts of different lengths in one batch (plain KV cache, `attn_mode="vanilla"`).

  dec = PackedDecoder(model, rows=16, capacity=2048)
  ids, logp = dec.generate([[1, 17, 4], [1, 99]], max_new=64, eos_id=2)      # one list of new ids per prompt

The prompts are packed one behind the other and run through the layers in ONE pass (`ops.packed_attention`), their keys and
values are written to the rows' caches, and every further token is a step over the whole batch in which each row has a
position and a live length of its own (`ops.cached_attention`); the next token and its log probability come from
`ops.token_logprobs`.  Grouped KV heads, sliding windows and the log-n scale work as in training.  `capture()` records the
step as one CUDA graph.  Weights of another type than `dtype` are copied once; `refresh(model)` copies them again.
Where they are not copied, the model's tensors have to stay where they are, and its configuration as it is, while the decoder
lives.  (`eval.graph_decode.GraphDecoder` is the decoder for batches that share one position, and for the Dual-Mod write law.)"""

from __future__ import annotations

import copy

import torch

from ..ops import cached_attention, default_ops, packed_attention, token_logprobs


class PackedDecoder:
    def __init__(self, model, rows, capacity, dtype=None):
        cfg = model.cfg
        if cfg.attn_mode != "vanilla":
            raise ValueError("PackedDecoder is for attn_mode 'vanilla'")
        if not 0 < capacity <= cfg.max_seq_len:
            raise ValueError(f"capacity: 1 to {cfg.max_seq_len} is wanted, got {capacity}")
        self.rows, self.P = rows, capacity
        self.dev = next(model.parameters()).device
        self.dtype = dtype or (torch.bfloat16 if self.dev.type == "cuda" else torch.float32)
        if next(model.parameters()).dtype != self.dtype:
            # decode from a copy of the weights in the compute type; tables (RoPE) stay in their own precision
            src, model = model, copy.deepcopy(model).to(self.dtype)
            for name, buf in src.named_buffers():
                mod, _, leaf = name.rpartition(".")
                setattr(model.get_submodule(mod) if mod else model, leaf, buf.clone())
        self.m = model.eval()
        a = model.blocks[0].attn
        zeros = lambda: torch.zeros(rows, capacity, a.n_kv_heads, a.head_dim, device=self.dev, dtype=self.dtype)
        self.K, self.V = [zeros() for _ in model.blocks], [zeros() for _ in model.blocks]
        self.lengths = torch.zeros(rows, dtype=torch.int32, device=self.dev)
        self.tok = torch.zeros(rows, dtype=torch.long, device=self.dev)
        self.no_target = torch.full((rows,), -1, dtype=torch.long, device=self.dev)
        self.graph = None

    @torch.no_grad()
    def refresh(self, model):
        """Takes over the weights of `model`, which this decoder was made from, where it decodes from a copy of them (in place: a
        recorded step sees them)."""
        if model is not self.m:
            for mine, theirs in ((self.m.parameters(), model.parameters()), (self.m.buffers(), model.buffers())):
                for a, b in zip(mine, theirs):
                    a.copy_(b)

    def _pick(self, logits):
        r = token_logprobs(logits, self.no_target[:logits.shape[0]], top=1)
        return r.top_ids[:, 0], r.top_logp[:, 0]

    @torch.no_grad()
    def prefill(self, prompts):
        """Fills the caches with `prompts` (at most `rows` lists of ids, none empty) -> (next ids, their log probabilities)."""
        lens = [len(p) for p in prompts]
        if not 0 < len(lens) <= self.rows or min(lens) < 1 or max(lens) > self.P:
            raise ValueError(f"1 to {self.rows} prompts of 1 to {self.P} tokens are wanted, got lengths {lens}")
        n = torch.tensor(lens)
        edges = torch.cat((torch.zeros(1, dtype=torch.long), n.cumsum(0)))
        idx = torch.tensor([t for p in prompts for t in p], device=self.dev)
        row = torch.arange(len(lens)).repeat_interleave(n).to(self.dev)
        x = self.m.tok_emb(idx)
        cu, pos, cos, sin = self.m.packed_rows(edges, len(idx), self.dev)
        for li, blk in enumerate(self.m.blocks):
            a = blk.attn
            q, k, v = a._packed_qkv(blk.attn_norm(x), cos, sin)
            self.K[li][row, pos] = k
            self.V[li][row, pos] = v
            o = packed_attention(a._logn_queries(q, pos), k, v, cu, window=a.cfg.local_window or 0, scale=a.scale)
            x = x + a.wo(o.reshape(len(idx), a.d_attn))
            x = x + blk.mlp(blk.mlp_norm(x))
        logits = self.m.lm_head(self.m.norm_f(x[(edges[1:] - 1).to(self.dev)]))
        self.lengths.zero_()
        self.lengths[:len(lens)] = n.to(self.dev, torch.int32)
        return self._pick(logits)

    @torch.no_grad()
    def _step(self):
        """One token per row (`self.tok`) at the row's own position: extends the caches, returns (next ids, log probs).
        A row whose cache is full overwrites its last entry (`generate` has ended such a row)."""
        m, pos = self.m, self.lengths.clamp_max(self.P - 1).long()
        row = torch.arange(self.rows, device=self.dev)
        self.lengths.add_(1).clamp_max_(self.P)
        x = m.tok_emb(self.tok)
        cos, sin = m.rope_cos[pos], m.rope_sin[pos]
        for li, blk in enumerate(m.blocks):
            a = blk.attn
            q, k, v = a._packed_qkv(blk.attn_norm(x), cos, sin)
            self.K[li][row, pos] = k
            self.V[li][row, pos] = v
            o = cached_attention(a._logn_queries(q, pos), self.K[li], self.V[li], self.lengths,
                                 window=a.cfg.local_window or 0, scale=a.scale)
            x = x + a.wo(o.reshape(self.rows, a.d_attn))
            x = x + blk.mlp(blk.mlp_norm(x))
        logits = m.lm_head(m.norm_f(x))
        return self._pick(logits)

    def capture(self):
        """Records the step as a CUDA graph, on this decoder's device whichever is current (caches and lengths keep their
        contents); returns self."""
        with torch.cuda.device(self.dev):
            keep = self.lengths.clone()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                held = [(K[:, -1].clone(), V[:, -1].clone()) for K, V in zip(self.K, self.V)]
                self.lengths.fill_(self.P - 1)           # the warm-up writes the caches' last rows only
                self._step()
                for (k, v), K, V in zip(held, self.K, self.V):
                    K[:, -1], V[:, -1] = k, v
                self.lengths.copy_(keep)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):   # the stream that torch records on by default is of one device for good
                self.out = self._step()
        self.graph = graph
        return self

    def step(self, tokens):
        """tokens int64 [rows] -> (next ids, log probabilities) [rows].  Captured, every step returns the same two tensors."""
        self.tok.copy_(tokens)
        if self.graph is None:
            return self._step()
        self.graph.replay()
        return self.out

    def generate(self, prompts, max_new, eos_id=None, stop_fn=None):
        """Greedy continuations of up to `rows` prompts -> (list of id lists, list of their log probabilities).  A row ends at
        `eos_id` (not included), when `stop_fn(its ids)` says so, after max_new tokens or when its cache is full.
        RuntimeError where a kernel gave up on the way."""
        ids, logp = self.prefill(prompts)
        n = len(prompts)
        out, scores, alive = [[] for _ in prompts], [[] for _ in prompts], [True] * n
        for j in range(max_new):
            for r, (t, s) in enumerate(zip(ids[:n].tolist(), logp[:n].tolist())):
                if not alive[r]:
                    continue
                if t == eos_id or len(prompts[r]) + len(out[r]) > self.P:
                    alive[r] = False
                    continue
                out[r].append(t)
                scores[r].append(s)
                if stop_fn is not None and stop_fn(out[r]):
                    alive[r] = False
            if j + 1 == max_new or not any(alive):
                break
            nxt = torch.zeros_like(self.tok)
            nxt[:n] = ids[:n]
            ids, logp = self.step(nxt)
        default_ops(self.dev).tc_check()
        return out, scores
