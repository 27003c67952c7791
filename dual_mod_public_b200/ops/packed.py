"""Attention and token scores for sequences of different lengths, without padding.

    from dual_mod_public_b200.ops import packed_attention, cached_attention, token_logprobs

    o = packed_attention(q, k, v, cu_seqlens)             # q [T, Hq, D], k / v [T, Hkv, D]; differentiable
    o = cached_attention(q, k_cache, v_cache, lengths)    # q [B, Hq, D], caches [B, P, Hkv, D]; one token per sequence
    r = token_logprobs(logits, tokens, top=5)             # logits [..., V] -> r.logp, r.entropy, r.top_logp, r.top_ids

On a B200 these run the kernels of csrc/packed_attn_fwd.cu, packed_attn_bwd.cu, cached_attn.cu and logprob.cu, on the
tensors' own device and its current stream; on CPU the torch statements of `packed_math.py`.  No call reads a value back to
the host, so each can be captured into a CUDA graph, and none keeps state between calls.  (A captured backward pass wants what torch
asks of any: a first run on a side stream, and no eager graph of the same leaves alive.)  Results are bitwise repeatable.

Kernel arguments: bf16 or fp16 (attention; gradients: bf16), bf16, fp16 or fp32 (scores); head dims that are multiples of 8
up to 128.  Attention of other types or head dims runs the torch statement and is counted in `default_ops(device).fallbacks`
(`DMB_STRICT_OPS=1` raises instead).  Views whose strides a tensor map cannot describe (rows not on 16-byte boundaries,
expanded dims) are copied first.

Arguments that the host can see are checked and refused with TypeError or ValueError.  Device values are not: `cu_seqlens`
that do not ascend or lengths outside the cache give wrong outputs but never an access out of range (`lengths` are clamped
to [0, P]).  An attention kernel whose pipeline stands still for two seconds ends with wrong outputs and sets a flag instead of
holding the device: `default_ops(device).tc_check()` reads it (one value to the host) and raises RuntimeError.  Call it
before results are used outside of the device; what the framework itself answers or trains with is checked (`PackedDecoder.generate`,
packed scoring in the evaluation adapter, `train_baseline --packed_docs`).  Gradients are those of reverse mode, once: an input with a forward-mode tangent is refused with
NotImplementedError on every device.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import default_ops

MAX_TOP = 32
MAX_CACHE = (1 << 31) - 4096          # rows: the kernel shares them out in whole tiles, whose ends have to be 32-bit numbers too
MAX_VOCAB = (1 << 31) - 4096          # columns: a row's last vector and the 1024 threads behind it are 32-bit numbers too
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_T = torch.Tensor
_SCALES = 2.0 ** -126, 2.0 ** 127     # the kernels hold scale log2(e) in fp32: as zero it would turn a hidden key's -inf into NaN


def _check_attention(q, k, v, index, name, kv_dims, scale, window):
    """The scale; raises for arguments that do not fit.  One pass over the conditions that hold for a call that fits."""
    if not isinstance(q, _T) or not isinstance(k, _T) or not isinstance(v, _T) or not isinstance(index, _T):
        raise TypeError(f"q, k, v and {name}: tensors are wanted")
    dtype, device, qs, ks = q.dtype, q.device, q.shape, k.shape
    if dtype not in _FLOATS or k.dtype is not dtype or v.dtype is not dtype:
        raise TypeError(f"q, k and v of one type (bf16, fp16 or fp32) are wanted, got {q.dtype}, {k.dtype}, {v.dtype}")
    if index.dtype is not torch.int32 or index.dim() != 1:
        raise TypeError(f"{name}: a 1-d int32 tensor is wanted")
    if k.device != device or v.device != device or index.device != device:
        raise ValueError(f"q, k, v and {name} have to be on one device")
    if len(qs) != 3 or len(ks) != kv_dims or v.shape != ks:
        raise ValueError(f"q of 3 dims and k, v of {kv_dims} dims and equal shape are wanted, got {tuple(qs)}, {tuple(ks)}, "
                         f"{tuple(v.shape)}")
    Hq, D, Hkv = qs[1], qs[2], ks[-2]
    if qs[0] != ks[0] or ks[-1] != D or D == 0:
        raise ValueError(f"q and k, v differ in rows or head dim: {tuple(qs)}, {tuple(ks)}")
    if Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise ValueError(f"{Hq} query heads are not a multiple of {Hkv} key heads")
    if not isinstance(window, int) or not 0 <= window < 1 << 31:
        raise ValueError(f"window: a number of tokens (0: all) is wanted, got {window!r}")
    if scale is None:
        return 1.0 / math.sqrt(D)
    scale = float(scale)
    if not _SCALES[0] <= scale <= _SCALES[1]:
        raise ValueError(f"scale has to be positive and a normal fp32 number, 2^-126 to 2^127, got {scale}")
    return scale


def _check_tangents(name, *tensors):
    """Refuses dual tensors: the kernels read values only, so a tangent would be lost without a word.  Callers look for an open
    dual level first, which is all that a call outside of one pays for."""
    for t in tensors:
        if forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name} has no forward-mode derivative")


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu, window, scale):
        ops = default_ops(q.device)
        o, lse, o_lo = ops.packed_attn_fwd(q, k, v, cu, window, scale, residual=True)
        ctx.save_for_backward(q, k, v, o, lse, cu, o_lo)
        ctx.window, ctx.scale = window, scale
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse, cu, o_lo = ctx.saved_tensors
        dq, dk, dv = default_ops(q.device).packed_attn_bwd(do, q, k, v, o, lse, cu, ctx.window, ctx.scale, o_lo)
        return dq, dk, dv, None, None, None


def packed_attention(q, k, v, cu_seqlens, *, window=0, scale=None):
    """Causal attention over sequences packed on the row axis.

    q [T, Hq, D], k / v [T, Hkv, D] with Hq a multiple of Hkv (query head h reads key head h // (Hq // Hkv));
    cu_seqlens int32 [N + 1], ascending: sequence s is the rows [cu_seqlens[s], cu_seqlens[s + 1]) and may be empty.  A row
    sees the rows of its own sequence up to itself, the last `window` of them when window > 0.  Rows outside
    [cu_seqlens[0], cu_seqlens[N]) are padding: their output and gradients are zero and what they hold is not read into
    any other row.  `scale` defaults to 1 / sqrt(D); 2^-126 to 2^127 are taken.  Returns o [T, Hq, D] in q's type;
    differentiable in q, k and v.

    An output row depends on the rows that it sees and on no other, whatever those hold: an infinite or NaN entry of v makes
    the rows that see it infinite or NaN, and so does a NaN score or one of +inf.  A score of -inf has weight zero; a row whose
    scores all are -inf is zero, like a row without keys.  Finite scores may have any size; rows whose
    largest is beyond 1.2e7, and rows that share a block with a non-finite v that they do not see, are computed one by one, slowly.
    The gradients want finite inputs: their products run over blocks of 128 rows, and a weight of zero times an infinite or NaN
    entry is NaN, so such a row reaches the gradients of others in its block.  They form the weights from the logarithm of the
    row's sum in fp32: beyond 2^24 log 2 = 1.2e7 the gradients of the row and of the keys that it sees are NaN."""
    scale = _check_attention(q, k, v, cu_seqlens, "cu_seqlens", 3, scale, window)
    if cu_seqlens.shape[0] < 1:
        raise ValueError("cu_seqlens: at least one entry is wanted")
    if q.shape[0] >= (1 << 31) - 256:
        raise ValueError("too many rows")
    if getattr(forward_ad, "_current_level", 0) >= 0:
        _check_tangents("packed_attention", q, k, v)
    cu_seqlens = cu_seqlens.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _PackedAttention.apply(q, k, v, cu_seqlens, window, scale)
    return default_ops(q.device).packed_attn_fwd(q, k, v, cu_seqlens, window, scale, need_lse=False)[0]


def cached_attention(q, k_cache, v_cache, lengths, *, window=0, scale=None):
    """Attention of one new token per sequence over a cache with a live length per sequence.

    q [B, Hq, D]; k_cache / v_cache [B, P, Hkv, D]; lengths int32 [B]: sequence b reads the rows [0, lengths[b]) of its
    cache, which include the new token's own (the last `window` of them when window > 0).  Rows behind the live length are
    never read, whatever they hold.  A length of zero gives zeros.  Returns o [B, Hq, D].  Not differentiable: a tensor
    that requires a gradient is refused while gradients are enabled."""
    scale = _check_attention(q, k_cache, v_cache, lengths, "lengths", 4, scale, window)
    (B, Hq, _), (_, P, Hkv, _) = q.shape, k_cache.shape
    if lengths.shape[0] != B:
        raise ValueError("lengths: one entry per sequence is wanted")
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        raise ValueError("cached_attention has no gradient: call it under torch.no_grad()")
    if getattr(forward_ad, "_current_level", 0) >= 0:
        _check_tangents("cached_attention", q, k_cache, v_cache)
    if P > MAX_CACHE or B > 65535 or Hkv > 4095 or (Hq > 65535 and Hkv * -(-Hq // (16 * Hkv)) > 65535):
        raise ValueError("at most 65535 sequences, 4095 key heads, 65535 groups of up to 16 query heads of one key head and "
                         f"{MAX_CACHE} cache rows are wanted, got {B}, {Hkv}, {Hq} query heads and {P}")
    return default_ops(q.device).cached_attn(q, k_cache, v_cache, lengths.contiguous(), window, scale)


class TokenLogprobs(NamedTuple):
    logp: torch.Tensor                   # [...] fp32, differentiable
    entropy: torch.Tensor                # [...] fp32, differentiable
    top_logp: torch.Tensor | None        # [..., top] fp32, largest first
    top_ids: torch.Tensor | None         # [..., top] int64


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, tokens, top):
        logp, entropy, stats, top_logp, top_ids = default_ops(x.device).token_logprobs_fwd(x, tokens, top)
        ctx.save_for_backward(x, tokens, stats, entropy)
        if top:
            ctx.mark_non_differentiable(top_logp, top_ids)
        ctx.set_materialize_grads(False)
        return logp, entropy, top_logp, top_ids

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logp, g_entropy, *_):
        if g_logp is None and g_entropy is None:
            return None, None, None
        x, tokens, stats, entropy = ctx.saved_tensors
        return default_ops(x.device).token_logprobs_bwd(x, tokens, stats, entropy, g_logp, g_entropy), None, None


def token_logprobs(logits, tokens, *, top=0):
    """Scores of given tokens under rows of logits.

    logits [..., V] (bf16, fp16 or fp32), tokens int64 [...].  Returns `TokenLogprobs`: logp = log softmax(logits)[token],
    entropy of the row, and with top > 0 (at most 32) the `top` largest log probabilities with their ids, largest first,
    equal ones by ascending id.  All sums in fp32; outputs fp32.  A negative token means the row has no target: logp 0 and no
    gradient through it, whatever the row holds; a token >= V gives NaN.  logp and entropy are differentiable in the logits, the alternatives
    are not.  -inf logits (masked entries) are fine; a row of nothing else gives NaN."""
    if not isinstance(logits, _T) or not isinstance(tokens, _T):
        raise TypeError("logits and tokens: tensors are wanted")
    if logits.dtype not in _FLOATS:
        raise TypeError(f"logits of bf16, fp16 or fp32 are wanted, got {logits.dtype}")
    if tokens.dtype is not torch.int64:
        raise TypeError(f"tokens of int64 are wanted, got {tokens.dtype}")
    if logits.device != tokens.device:
        raise ValueError("logits and tokens have to be on one device")
    shape, lead = logits.shape, tokens.shape
    if len(shape) == 0 or shape[:-1] != lead or shape[-1] == 0:
        raise ValueError(f"tokens of the logits' leading shape are wanted, got {tuple(shape)} and {tuple(lead)}")
    V = shape[-1]
    if V > MAX_VOCAB or tokens.numel() >= 1 << 31:
        raise ValueError(f"at most {MAX_VOCAB} columns and 2^31 - 1 rows are wanted, got {V} and {tokens.numel()}")
    if not isinstance(top, int) or not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"top: 0 to {min(MAX_TOP, V)} is wanted, got {top!r}")
    if getattr(forward_ad, "_current_level", 0) >= 0:
        _check_tangents("token_logprobs", logits)
    flat = len(lead) == 1
    x, y = (logits, tokens.contiguous()) if flat else (logits.reshape(-1, V), tokens.reshape(-1).contiguous())
    if logits.requires_grad and torch.is_grad_enabled():
        logp, entropy, top_logp, top_ids = _TokenLogprobs.apply(x, y, top)
    else:
        logp, entropy, _, top_logp, top_ids = default_ops(x.device).token_logprobs_fwd(x, y, top, need_stats=False)
    if not flat:
        logp, entropy = logp.view(lead), entropy.view(lead)
        if top:
            top_logp, top_ids = top_logp.view(*lead, top), top_ids.view(*lead, top)
    return TokenLogprobs(logp, entropy, top_logp if top else None, top_ids if top else None)
