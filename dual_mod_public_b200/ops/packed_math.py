"""Plain-torch statements of the operators on packed sequences (`ops/packed.py`): what the torch op table runs, and what
the kernel table runs for element types and layouts its kernels do not take.  Math in fp32, one rounding at the end; no
value is read back to the host, so the statements can be captured like the kernels."""

from __future__ import annotations

import math

import torch

ROWS = 1024                       # query rows per slab: bounds the scores held at a time
FAR = 2.0 ** 24 * math.log(2.0)   # fp32 holds a log sum to within an octave up to here; beyond it gives no weights back


def _bounds(cu, T, window):
    """First visible key of every row [T] (row + 1: none)."""
    row = torch.arange(T, device=cu.device)
    n = cu.numel() - 1
    u = torch.searchsorted(cu.long(), row, right=True)
    lo = cu.long()[(u - 1).clamp_min(0)]
    if window:
        lo = torch.maximum(lo, row - window + 1)
    return torch.where((u == 0) | (u == n + 1), row + 1, lo)


def _slabs(q, k, cu, window, scale):
    """(rows, scores [Hkv, g, rows, keys] with -inf at hidden keys, hidden [rows, keys]) slab by slab."""
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    lo = _bounds(cu, T, window)
    key = torch.arange(T, device=q.device)
    kf = k.float().permute(1, 2, 0)                                        # [Hkv, D, T]
    for a in range(0, T, ROWS):
        b = min(T, a + ROWS)
        qf = q[a:b].float().view(b - a, Hkv, Hq // Hkv, D).permute(1, 2, 0, 3)
        s = (qf @ kf[:, None, :, :b]) * scale
        hidden = (key[None, :b] < lo[a:b, None]) | (key[None, :b] > key[a:b, None])
        yield slice(a, b), s.masked_fill(hidden, float("-inf")), hidden


def _heads_last(x):
    """[Hkv, g, rows, D] -> [rows, Hq, D]"""
    h, g, n, d = x.shape
    return x.permute(2, 0, 1, 3).reshape(n, h * g, d)


def _inside(x, cu):
    """x with the rows of no sequence zeroed: their contents are the caller's padding."""
    row = torch.arange(x.shape[0], device=x.device)
    keep = (row >= cu[0]) & (row < cu[-1])
    return torch.where(keep.view(-1, *([1] * (x.dim() - 1))), x, torch.zeros((), dtype=x.dtype, device=x.device))


def packed_attn_fwd(q, k, v, cu, window, scale):
    """(o [T, Hq, D], lse [Hq, T] fp32, what the rounding of o left)"""
    T, Hq, _ = q.shape
    q, k, v = (_inside(x, cu) for x in (q, k, v))
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    o_lo = torch.empty_like(o)
    lse = torch.empty(Hq, T, dtype=torch.float32, device=q.device)
    for rows, s, hidden in _slabs(q, k, cu, window, scale):
        top = s.amax(-1, keepdim=True)
        top = top.masked_fill(top == float("-inf"), 0.0)
        p = (s - top).exp().masked_fill(hidden, 0.0)
        total = p.sum(-1, keepdim=True)
        vf = v[:rows.stop].float().transpose(0, 1)[:, None]
        some = total != 0
        wild = ~vf.isfinite()                              # a hidden one would reach the row as 0 x NaN, so: who sees one
        pv = (p @ vf.masked_fill(wild, 0.0)).masked_fill((~hidden).float() @ wild.float() > 0, float("nan"))
        full = _heads_last(torch.where(some, pv / total, 0.0))
        o[rows] = full.to(q.dtype)
        o_lo[rows] = (full - o[rows].float()).to(q.dtype)
        lse[:, rows] = torch.where(some, top + total.log(), float("-inf")).reshape(Hq, -1)
    return o, lse, o_lo


def packed_attn_bwd(do, q, k, v, o, lse, cu, window, scale, o_lo=None):
    """(dq, dk, dv) in the inputs' type"""
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    do, q, k, v, o = (_inside(x, cu) for x in (do, q, k, v, o.float() if o_lo is None else o.float() + o_lo.float()))
    dq = torch.empty_like(q, memory_format=torch.contiguous_format)
    dk = torch.zeros(Hkv, T, D, dtype=torch.float32, device=q.device)
    dv = torch.zeros_like(dk)
    split = lambda x: x.float().view(x.shape[0], Hkv, Hq // Hkv, D).permute(1, 2, 0, 3)
    for rows, s, hidden in _slabs(q, k, cu, window, scale):
        n, keys = rows.stop - rows.start, rows.stop
        L = lse[:, rows].view(Hkv, Hq // Hkv, n, 1)
        L = torch.where((L.abs() <= FAR) | (L == float("-inf")), L, float("nan"))
        p = (s - L.masked_fill(L == float("-inf"), 0.0)).exp().masked_fill(hidden, 0.0)
        dof, of, qf = split(do[rows]), split(o[rows]), split(q[rows])
        dp = dof @ v[:keys].float().permute(1, 2, 0)[:, None]
        ds = (p * (dp - (dof * of).sum(-1, keepdim=True)) * scale).masked_fill(hidden, 0.0)
        dq[rows] = _heads_last(ds @ k[:keys].float().transpose(0, 1)[:, None]).to(q.dtype)
        dk[:, :keys] += (ds.transpose(-1, -2) @ qf).sum(1)
        dv[:, :keys] += (p.transpose(-1, -2) @ dof).sum(1)
    return dq, dk.transpose(0, 1).to(k.dtype).contiguous(), dv.transpose(0, 1).to(v.dtype).contiguous()


def cached_attn(q, k, v, lengths, window, scale):
    """o [B, Hq, D]"""
    B, Hq, D = q.shape
    P, Hkv = k.shape[1], k.shape[2]
    n = lengths.long().clamp(0, P)[:, None]
    row = torch.arange(P, device=q.device)
    live = row < n
    if window:
        live = live & (row >= n - window)
    vf = torch.where(live[:, :, None, None], v.float(), 0.0).transpose(1, 2)                   # [B, Hkv, P, D]
    s = (q.float().view(B, Hkv, Hq // Hkv, D) @ k.float().permute(0, 2, 3, 1)) * scale
    s = s.masked_fill(~live[:, None, None], float("-inf"))
    if P == 0:
        return torch.zeros(B, Hq, D, dtype=q.dtype, device=q.device)
    top = s.amax(-1, keepdim=True)
    p = (s - top.masked_fill(top == float("-inf"), 0.0)).exp().masked_fill(~live[:, None, None], 0.0)
    total = p.sum(-1, keepdim=True)
    return torch.where(total != 0, (p @ vf) / total, 0.0).reshape(B, Hq, D).to(q.dtype)


def token_logprobs_fwd(x, tokens, top):
    """x [N, V], tokens [N] -> (logp, entropy, stats [N, 2] = (maximum, log of the sum), top_logp, top_ids)"""
    V = x.shape[1]
    x = x.float()
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = d.exp()
    total = e.sum(-1, keepdim=True)
    ls = total.log()
    entropy = (ls - torch.where(e > 0, e * d, e).sum(-1, keepdim=True) / total).squeeze(-1)
    y = tokens.clamp(0, V - 1)[:, None]
    logp = (d.gather(-1, y) - ls).squeeze(-1)
    logp = torch.where(tokens < 0, 0.0, torch.where(tokens >= V, float("nan"), logp))
    order = torch.where(x != x, float("-inf"), x).sort(dim=-1, descending=True, stable=True).indices[:, :top]
    return logp, entropy, torch.cat((m, ls), dim=-1), d.gather(-1, order) - ls, order


def token_logprobs_bwd(x, tokens, stats, entropy, g_logp, g_entropy):
    V = x.shape[1]
    lp = (x.float() - stats[:, :1]) - stats[:, 1:]
    p = lp.exp()
    zero = torch.zeros(x.shape[0], dtype=torch.float32, device=x.device)
    gl = zero if g_logp is None else torch.where(tokens < 0, zero, torch.where(tokens >= V, float("nan"), g_logp))
    gh = zero if g_entropy is None else g_entropy
    d = -p * (gh[:, None] * lp.clamp_min(-200.0) + (gl + gh * entropy)[:, None])
    d = d.masked_fill(((tokens < 0) & (gh == 0))[:, None], 0.0)          # no gradient reaches the row: also where its p is NaN
    has = (tokens >= 0) & (tokens < V)
    d.scatter_add_(-1, tokens.clamp(0, V - 1)[:, None], torch.where(has, gl, 0.0)[:, None])
    return d.to(x.dtype)
