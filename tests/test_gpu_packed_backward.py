"""Gradients of the packed attention and of the token log probabilities: the kernels against 64-bit statements, element by
element within the bounds that their roundings allow."""

import pytest
import torch

import packed_oracles as ref
from test_gpu_packed_forward import DEV, PACKS, cu_of, logp_bound, ops, rnd, table  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu


def grads(ops, q, k, v, cu, g, window=0, scale=None):
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    before = dict(table(ops).fallbacks)
    o = ops.packed_attention(*leaves, cu, window=window, scale=scale)
    out = torch.autograd.grad(o, leaves, g)
    table(ops).tc_check()
    assert table(ops).fallbacks == before                          # the kernels ran
    return (o, *out)


def check(got, want):
    for x, name in zip(got, ("o", "dq", "dk", "dv")):
        ref.close(x, want[name], name)


@pytest.mark.parametrize("rows,edges", PACKS)
@pytest.mark.parametrize("hq,hkv,dim", [(2, 2, 64), (4, 1, 128), (6, 2, 72), (3, 1, 8)])
def test_packed_backward(ops, rows, edges, hq, hkv, dim):  # noqa: F811
    q, k, v, g = (rnd(rows, h, dim, seed=s, std=w) for h, s, w in ((hq, 1, 1.5), (hkv, 2, 1.5), (hkv, 3, 1.0), (hq, 4, 1.0)))
    check(grads(ops, q, k, v, cu_of(*edges), g), ref.packed(q, k, v, cu_of(*edges), do=g))


@pytest.mark.parametrize("window", [1, 2, 63, 128, 129, 500, 100000])
@pytest.mark.parametrize("dim", [64, 128])
def test_packed_backward_window(ops, window, dim):  # noqa: F811
    q, k, v, g = (rnd(900, 2, dim, seed=s) for s in (1, 2, 3, 4))
    cu = cu_of(0, 10, 500, 890)
    check(grads(ops, q, k, v, cu, g, window), ref.packed(q, k, v, cu, window, do=g))


@pytest.mark.parametrize("scale", [0.02, 1.0])
def test_packed_backward_large_scores(ops, scale):  # noqa: F811
    q, k, v, g = (rnd(1100, 2, 64, seed=s, std=w) for s, w in ((1, 2.0), (2, 2.0), (3, 1.0), (4, 1.0)))
    k[600:] *= 3.0
    cu = cu_of(0, 1100)
    check(grads(ops, q, k, v, cu, g, scale=scale), ref.packed(q, k, v, cu, scale=scale, do=g))


def test_packed_backward_views(ops):  # noqa: F811
    """One projection for q, k, v; a gradient that is expanded, one with a stride."""
    T, h, d = 333, 4, 64
    qkv = rnd(T, 3, h, d, seed=5)
    cu = cu_of(0, 100, 333)
    g = rnd(T, 2, h, d, seed=6)[:, 1]
    check(grads(ops, qkv[:, 0], qkv[:, 1], qkv[:, 2], cu, g), ref.packed(qkv[:, 0], qkv[:, 1], qkv[:, 2], cu, do=g))
    one = rnd(1, 1, d, seed=7).expand(T, h, d)
    check(grads(ops, qkv[:, 0], qkv[:, 1], qkv[:, 2], cu, one), ref.packed(qkv[:, 0], qkv[:, 1], qkv[:, 2], cu, do=one))


def test_packed_backward_of_rows_that_see_themselves_alone(ops):  # noqa: F811
    """Sequences of one token: o = v, ds = do . v - do . o = 0, so dq and dk are zero up to what delta is off.  delta comes
    from o and its residual (2^-16 of every product) and fp32 sums of D products (2^-23 each, twice)."""
    T, h, d = 300, 2, 64
    q, k, v, g = (rnd(T, h, d, seed=s) for s in (1, 2, 3, 4))
    o, dq, dk, dv = grads(ops, q, k, v, cu_of(*range(T + 1)), g)
    assert torch.equal(o, v) and torch.equal(dv, g)
    off = (g.double().abs() * v.double().abs()).sum(-1, keepdim=True) * (2.0 ** -16 + 2 * d * 2.0 ** -23) * d ** -0.5 * (1 + 2.0 ** -7)
    ref.close(dq, (torch.zeros_like(dq, dtype=torch.float64), off * k.double().abs() + 1e-30), "dq")
    ref.close(dk, (torch.zeros_like(dk, dtype=torch.float64), off * q.double().abs() + 1e-30), "dk")


def test_packed_backward_padding_is_not_read(ops):  # noqa: F811
    q, k, v, g = (rnd(500, 2, 64, seed=s) for s in (1, 2, 3, 4))
    cu = cu_of(2, 200, 450)
    want = ref.packed(q, k, v, cu, do=g)
    for x, bad in ((q, float("nan")), (k, float("inf")), (v, float("nan")), (g, float("inf"))):
        x[:2] = bad
        x[450:] = bad
    got = grads(ops, q, k, v, cu, g)
    for x in got:
        assert not x[:2].any() and not x[450:].any()
    check(got, want)


def test_packed_backward_leaf_twice(ops):  # noqa: F811
    """One tensor as key and value, broadcast to the heads by an expand: its gradient is the sum."""
    T, d = 260, 64
    q, x, g = rnd(T, 4, d, seed=1), rnd(T, 1, d, seed=2), rnd(T, 4, d, seed=3)
    cu = cu_of(0, 260)
    leaf = x.detach().requires_grad_()
    kv = leaf.expand(T, 4, d)
    dx, = torch.autograd.grad(ops.packed_attention(q, kv, kv, cu), leaf, g)
    want = ref.packed(q, x.expand(T, 4, d), x.expand(T, 4, d), cu, do=g)
    value = (want["dk"][0] + want["dv"][0]).sum(1, keepdim=True)
    u = ref.u_of(torch.bfloat16)
    # the two bf16 gradients are added (one rounding) and then summed over the heads (one rounding of the result)
    bound = ((want["dk"][1] + want["dv"][1]) * (1 + u) + u * (want["dk"][0] + want["dv"][0]).abs()).sum(1, keepdim=True) * (1 + u) + u * value.abs()
    ref.close(dx, (value, bound), "dx")


def test_packed_fp16_gradient_runs_the_statement(ops):  # noqa: F811
    q, k, v, g = (rnd(200, 2, 64, seed=s, dtype=torch.float16) for s in (1, 2, 3, 4))
    g *= 2.0 ** -10                                                # small gradients do not vanish
    cu = cu_of(0, 200)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    n = table(ops).fallbacks.get("packed_attn_bwd", 0)
    out = torch.autograd.grad(ops.packed_attention(*leaves, cu), leaves, g)
    assert table(ops).fallbacks["packed_attn_bwd"] == n + 1
    want = ref.packed(q, k, v, cu, do=g)
    for x, name in zip(out, ("dq", "dk", "dv")):
        value, bound = want[name]
        ref.close(x, (value, bound + 2.0 ** -25), name)            # half a step of the smallest fp16 numbers


def test_packed_bitwise_repeatable_and_captured(ops):  # noqa: F811
    """The same bits on another stream, on a second call and from a replayed graph; new inputs in the same buffers."""
    q, k, v, g = (rnd(700, h, 64, seed=s) for h, s in ((4, 1), (2, 2), (2, 3), (4, 4)))
    cu = cu_of(0, 100, 650)
    t = table(ops)

    def step():
        o, lse = t.packed_attn_fwd(q, k, v, cu, 0, 0.125)
        return (o, *t.packed_attn_bwd(g, q, k, v, o, lse, cu, 0, 0.125))
    first = [x.clone() for x in step()]
    for a, b in zip(first, step()):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, other):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    graph.replay()
    for a, b in zip(first, held):
        assert torch.equal(a, b)
    q.copy_(rnd(700, 4, 64, seed=9))
    cu.copy_(cu_of(0, 333, 700))                                   # the table is read on the device at every replay
    graph.replay()
    check(held, ref.packed(q, k, v, cu, scale=0.125, do=g))


# ---- scores -------------------------------------------------------------------------------------------------------------
def dx_bound(x, y, g_lp, g_h, want):
    """p carries the relative error of exp at its logp's absolute error; the result is rounded once."""
    lp = torch.log_softmax(x.detach().double(), -1)
    p = lp.exp()
    e = 4 * logp_bound(x, x.shape[1])[:, None]
    gl, gh = (0.0 if g is None else g.double().abs()[:, None] for g in (g_lp, g_h))
    terms = p * (gl + gh * (torch.where(p > 0, lp.abs(), 0.0) + want["entropy"].abs()[:, None] + 1))
    hot = torch.zeros_like(p).scatter_(-1, y.clamp_min(0)[:, None], 1.0) * gl
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 1e-37        # half a step of fp16's smallest; fp32 results below 2^-126
    return e * terms + (hot * 2.0 ** -23) + ref.u_of(x.dtype) * want["dx"].abs() * (1 + 1e-6) + tiny


@pytest.mark.parametrize("V", [1, 2, 7, 8, 259, 2049, 32000, 50257])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("which", ["both", "logp", "entropy"])
def test_logprobs_backward(ops, V, dtype, which):  # noqa: F811
    N = 11
    x = rnd(N, V, seed=V, dtype=dtype, std=3.0).requires_grad_()
    y = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(1)).to(DEV)
    y[3] = -1
    gl, gh = rnd(N, seed=1, dtype=torch.float32), rnd(N, seed=2, dtype=torch.float32)
    r = ops.token_logprobs(x, y, top=min(3, V))
    outs, gs = {"both": ((r.logp, r.entropy), (gl, gh)), "logp": ((r.logp,), (gl,)), "entropy": ((r.entropy,), (gh,))}[which]
    dx, = torch.autograd.grad(outs, x, gs)
    gl, gh = (gl if which != "entropy" else None), (gh if which != "logp" else None)
    want = ref.logprobs(x, y, 0, gl, gh)
    ref.close(dx, (want["dx"], dx_bound(x, y, gl, gh, want)), "dx")
    assert not r.top_logp.requires_grad


def test_logprobs_backward_views_masks_and_bad_tokens(ops):  # noqa: F811
    big = rnd(6, 700, seed=1, dtype=torch.float32)
    big[:, 100:200] = -torch.inf                                    # masked entries
    y = torch.tensor([3, -1, 99, 250, 400, 0], device=DEV)
    gl, gh = rnd(6, seed=1, dtype=torch.float32), rnd(6, seed=2, dtype=torch.float32)
    for a in range(5):                                              # every alignment of input rows against output rows
        x = big[:, a:a + 515].detach().requires_grad_()
        r = ops.token_logprobs(x, y)
        dx, = torch.autograd.grad((r.logp, r.entropy), x, (gl, gh))
        want = ref.logprobs(x, y, 0, gl, gh)
        assert not dx[:, 100:195].any()
        ref.close(dx, (want["dx"], dx_bound(x, y, gl, gh, want)), f"offset {a}")
    x = torch.full((2, 40), torch.finfo(torch.float32).min, device=DEV).requires_grad_()
    dx, = torch.autograd.grad(ops.token_logprobs(x, y[[0, 1]]).logp.sum(), x)
    assert torch.allclose(dx[0, 4:], torch.full((36,), -1 / 40, device=DEV)) and not dx[1].any()
    x = rnd(2, 40, seed=3).requires_grad_()
    dx, = torch.autograd.grad(ops.token_logprobs(x, torch.tensor([40, 39], device=DEV)).logp.sum(), x)
    assert dx[0].isnan().all() and dx[1].isfinite().all()


def test_logprobs_captured(ops):  # noqa: F811
    x, y = rnd(9, 3001, seed=1), torch.arange(9, device=DEV)
    t = table(ops)
    gl = torch.ones(9, device=DEV)

    def step():
        lp, h, st, tl, ti = t.token_logprobs_fwd(x, y, 4)
        return lp, h, tl, ti, t.token_logprobs_bwd(x, y, st, h, gl, None)
    first = [a.clone() for a in step()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    graph.replay()
    for a, b in zip(first, held):
        assert torch.equal(a, b)


def test_score_a_packed_batch(ops):  # noqa: F811
    """The operators as they are used together: packed attention, a head, the scores, and the gradients back to q, k, v,
    against the same chain sequence by sequence in 64 bits from the kernel's own attention output."""
    T, h, d, V = 400, 4, 64, 700
    cu = cu_of(0, 37, 38, 250, 400)
    q, k, v = (rnd(T, h, d, seed=s).requires_grad_() for s in (1, 2, 3))
    w = rnd(h * d, V, seed=4, std=0.1)
    y = torch.randint(0, V, (T,), generator=torch.Generator().manual_seed(2)).to(DEV)
    y[cu[1:].long() - 1] = -1                                       # a sequence's last row has no next token
    o = ops.packed_attention(q, k, v, cu)
    logits = o.reshape(T, h * d) @ w
    r = ops.token_logprobs(logits, y, top=1)
    dq, dk, dv = torch.autograd.grad(r.logp.sum(), (q, k, v))
    want = ref.logprobs(logits, y, 1, torch.ones(T, device=DEV))
    ref.close(r.logp, (want["logp"], logp_bound(logits.detach(), V)), "logp")
    do = (want["dx"].to(torch.bfloat16) @ w.t()).view(T, h, d)      # as autograd forms it: bf16 logits' gradient, bf16 product
    full = ref.packed(q, k, v, cu, do=do)
    for got, name in ((dq, "dq"), (dk, "dk"), (dv, "dv")):
        value, bound = full[name]
        # a gradient of the logits next to a rounding border may fall to the other side: one step (2 u) of single terms of
        # the product that makes do; in the norm over all elements that stays below one rounding of each
        err = (got.double() - value).norm() / value.norm()
        assert err < 3 * ref.u_of(torch.bfloat16), (name, err)
