"""Decoder-only LM around `DualModAttention`: RMSNorm pre-norm, RoPE, SwiGLU,
tied embedding / unembedding, no biases except the gate biases.

Parity with the reference `DualModLM` (models/dualmod/model.py:115-334): same
module tree and state-dict keys (`tok_emb`, `blocks.N.{attn_norm,attn,mlp_norm,mlp}`,
`norm_f`, `lm_head`; RoPE tables are non-persistent buffers), `forward` ->
(logits, loss) with fp32 cross-entropy and ignore_index=-1, and incremental
decode through the same per-position step as the training scan.
"""

from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..config import DualModConfig
from ..ops.packed import token_logprobs
from .attention import DualModAttention
from .init import init_dualmod_lm
from .layers import RMSNorm, SwiGLU
from .rope import build_rope_cache

_DUAL_PARAM_TAGS = ("w_kctx", "w_vctx", "w_gk", "w_gv", "norm_ctx")


class Block(nn.Module):
    def __init__(self, cfg: DualModConfig):
        super().__init__()
        self.attn_norm = RMSNorm(cfg.d_model)
        self.attn = DualModAttention(cfg)
        self.mlp_norm = RMSNorm(cfg.d_model)
        self.mlp = SwiGLU(cfg.d_model, cfg.mlp_hidden)

    def forward(self, x, cos, sin, collect=None, cu_seqlens=None):
        x = x + self.attn(self.attn_norm(x), cos, sin, collect=collect, cu_seqlens=cu_seqlens)
        return x + self.mlp(self.mlp_norm(x))

    def decode_step(self, x_j, pos, cache, cos, sin):
        x_j = x_j + self.attn.decode_step(self.attn_norm(x_j), pos, cache, cos, sin)
        return x_j + self.mlp(self.mlp_norm(x_j))


class DualModLM(nn.Module):
    def __init__(self, cfg: DualModConfig):
        super().__init__()
        self.cfg = cfg
        self.tok_emb = nn.Embedding(cfg.vocab_size, cfg.d_model)
        self.blocks = nn.ModuleList(Block(cfg) for _ in range(cfg.n_layers))
        self.norm_f = RMSNorm(cfg.d_model)
        self.lm_head = nn.Linear(cfg.d_model, cfg.vocab_size, bias=False)
        if cfg.tie_embeddings:
            self.lm_head.weight = self.tok_emb.weight
        cos, sin = build_rope_cache(cfg.max_seq_len, cfg.head_dim, cfg.rope_theta)
        if not cfg.use_rope:
            cos, sin = torch.ones_like(cos), torch.zeros_like(sin)
        self.register_buffer("rope_cos", cos, persistent=False)
        self.register_buffer("rope_sin", sin, persistent=False)
        init_dualmod_lm(self)

    # kept as a method so callers that re-initialise a model in place can do so
    def _init_weights(self):
        init_dualmod_lm(self)

    def set_rope_len(self, max_seq_len: int):
        """Rebuild the RoPE tables for a longer evaluation context."""
        dev = self.rope_cos.device
        cos, sin = build_rope_cache(max_seq_len, self.cfg.head_dim, self.cfg.rope_theta, device=dev)
        if not self.cfg.use_rope:
            cos, sin = torch.ones_like(cos), torch.zeros_like(sin)
        self.rope_cos, self.rope_sin = cos, sin
        self.cfg.max_seq_len = max_seq_len

    def forward(self, idx=None, targets=None, inputs_embeds=None, collect=None, cu_seqlens=None, logit_rows=None):
        """(logits [B,T,V], loss or None).  `collect`: optional list of per-layer
        dicts that receive telemetry tensors.

        `cu_seqlens` (attn_mode "vanilla"): idx / targets are [T] (or [1,T]), sequences of any lengths packed one behind
        the other, sequence s being the rows [cu_seqlens[s], cu_seqlens[s+1]); no row sees another sequence and positions
        restart with each.  Returns logits [T,V] (of the rows `logit_rows` only, where given: int64 [n], targets [n]).
        The loss is the mean over targets >= 0; zero, with zero gradients, where there is none."""
        if cu_seqlens is not None:
            return self._forward_packed(idx, targets, inputs_embeds, cu_seqlens, logit_rows)
        x = self.tok_emb(idx) if inputs_embeds is None else inputs_embeds
        T = x.shape[1]
        assert T <= self.cfg.max_seq_len, "sequence longer than the RoPE table"
        cos, sin = self.rope_cos[:T], self.rope_sin[:T]
        for i, blk in enumerate(self.blocks):
            x = blk(x, cos, sin, collect=None if collect is None else collect[i])
        logits = self.lm_head(self.norm_f(x))
        loss = None
        if targets is not None:
            loss = F.cross_entropy(logits.float().view(-1, logits.shape[-1]),
                                   targets.reshape(-1), ignore_index=-1)
        return logits, loss

    def packed_rows(self, cu_seqlens, T, device):
        """(table, position of every row, cos, sin) of T packed rows.  A table that the host holds (a list, a tensor on CPU)
        is checked; one on the device is taken as it is, and positions beyond the RoPE table keep its last angle."""
        longest = None
        if not (isinstance(cu_seqlens, torch.Tensor) and cu_seqlens.is_cuda):
            cu_seqlens = torch.as_tensor(cu_seqlens, dtype=torch.int32)
            gaps = cu_seqlens.diff()
            if cu_seqlens.dim() != 1 or len(gaps) == 0 or cu_seqlens[0] < 0 or gaps.min() < 0 or cu_seqlens[-1] > T:
                raise ValueError(f"cu_seqlens have to ascend within [0, {T}]")
            longest = int(gaps.max())
        if longest is not None and longest > self.cfg.max_seq_len:
            raise ValueError(f"a sequence of {longest} tokens is longer than the RoPE table ({self.cfg.max_seq_len})")
        cu = cu_seqlens.to(device=device, dtype=torch.int32)
        row = torch.arange(T, device=device, dtype=torch.int32)
        start = cu[(torch.searchsorted(cu, row, right=True) - 1).clamp_min(0)]
        pos = (row - start).clamp(0, self.cfg.max_seq_len - 1).long()
        return cu, pos, self.rope_cos[pos], self.rope_sin[pos]

    def _forward_packed(self, idx, targets, inputs_embeds, cu_seqlens, logit_rows):
        if self.cfg.attn_mode != "vanilla":
            raise ValueError("packed sequences are for attn_mode 'vanilla'")
        x = self.tok_emb(idx.reshape(-1)) if inputs_embeds is None else inputs_embeds.reshape(-1, self.cfg.d_model)
        cu, pos, cos, sin = self.packed_rows(cu_seqlens, x.shape[0], x.device)
        for blk in self.blocks:
            x = blk(x, cos, sin, cu_seqlens=(cu, pos))
        if logit_rows is not None:
            x = x[logit_rows]
        logits = self.lm_head(self.norm_f(x))
        loss = None
        if targets is not None:
            targets = targets.reshape(-1)
            loss = -token_logprobs(logits, targets).logp.sum() / (targets >= 0).sum().clamp_min(1)
        return logits, loss

    # ---- incremental decode ----------------------------------------------------------
    def decode_init(self):
        return [{"K": None, "V": None} for _ in self.blocks]

    @torch.no_grad()
    def decode_step(self, idx_j, pos, caches):
        """idx_j [B,1] at absolute position `pos` -> logits [B,1,V]; extends caches."""
        x = self.tok_emb(idx_j)
        for blk, cache in zip(self.blocks, caches):
            x = blk.decode_step(x, pos, cache, self.rope_cos, self.rope_sin)
        return self.lm_head(self.norm_f(x))

    @torch.no_grad()
    def generate(self, idx, max_new_tokens, temperature=1.0, top_k=None):
        """Token-by-token prefill then sampling (temperature, optional top-k)."""
        caches = self.decode_init()
        logits = None
        for t in range(idx.shape[1]):
            logits = self.decode_step(idx[:, t:t + 1], t, caches)
        out = idx
        for _ in range(max_new_tokens):
            pos = out.shape[1]
            if pos >= self.cfg.max_seq_len:
                break
            lg = logits[:, -1, :] / max(temperature, 1e-6)
            if top_k is not None:
                kth = torch.topk(lg, top_k, dim=-1).values[:, -1:]
                lg = lg.masked_fill(lg < kth, float("-inf"))
            nxt = torch.multinomial(torch.softmax(lg.float(), dim=-1), 1)
            out = torch.cat((out, nxt), dim=1)
            logits = self.decode_step(nxt, pos, caches)
        return out

    # ---- accounting ---------------------------------------------------------------------
    def num_params(self, non_embedding=True):
        n = sum(p.numel() for p in self.parameters())
        if non_embedding:
            n -= self.tok_emb.weight.numel()
            if not self.cfg.tie_embeddings:
                n -= self.lm_head.weight.numel()
        return n

    def param_breakdown(self):
        dual = sum(p.numel() for name, p in self.named_parameters()
                   if any(f".{tag}." in name for tag in _DUAL_PARAM_TAGS))
        total = sum(p.numel() for p in self.parameters())
        return {"base": total - dual, "dualmod_extra": dual, "total": total}
