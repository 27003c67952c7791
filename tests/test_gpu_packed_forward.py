"""Packed attention (forward), single-token attention and token log probabilities: the kernels against 64-bit statements,
element by element within the bounds that their roundings allow."""

import pytest
import torch

import packed_oracles as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from dual_mod_public_b200 import ops as o
    return o


def table(ops):
    return ops.default_ops(torch.device(DEV))


def rnd(*shape, seed, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def cu_of(*edges):
    return torch.tensor(edges, dtype=torch.int32, device=DEV)


PACKS = [
    # rows, sequence edges
    (1, (0, 1)),
    (2, (0, 1, 2)),
    (127, (0, 127)),
    (128, (0, 0, 64, 128)),
    (129, (0, 129)),
    (256, (0, 256)),
    (257, (0, 1, 1, 130, 257)),
    (300, (0, 20, 21, 90, 128, 300)),
    (511, (0, 511)),
    (513, (0, 127, 255, 383, 513)),
    (640, (3, 100, 500)),                 # rows before the first and behind the last sequence
    (700, (0, 129)),                      # a tail of four whole tiles
    (900, (0,)),                          # no sequence at all
    (1537, (0, 700, 1537)),
]


@pytest.mark.parametrize("rows,edges", PACKS)
@pytest.mark.parametrize("hq,hkv,dim", [(2, 2, 64), (4, 1, 128), (3, 3, 32), (6, 2, 72), (2, 1, 8)])
def test_packed_forward(ops, rows, edges, hq, hkv, dim):
    q, k, v = (rnd(rows, h, dim, seed=s, std=w) for h, s, w in ((hq, 1, 1.5), (hkv, 2, 1.5), (hkv, 3, 1.0)))
    o = ops.packed_attention(q, k, v, cu_of(*edges))
    table(ops).tc_check()
    ref.close(o, ref.packed(q, k, v, cu_of(*edges))["o"], "o")


@pytest.mark.parametrize("window", [1, 2, 63, 128, 129, 500, 100000])
@pytest.mark.parametrize("dim", [64, 128])
def test_packed_forward_window(ops, window, dim):
    q, k, v = (rnd(900, 2, dim, seed=s) for s in (1, 2, 3))
    cu = cu_of(0, 10, 500, 890)
    ref.close(ops.packed_attention(q, k, v, cu, window=window), ref.packed(q, k, v, cu, window)["o"], "o")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [0.02, 1.0])
def test_packed_forward_types_and_large_scores(ops, dtype, scale):
    """Scores of some tens: the running maximum moves by many octaves between key blocks."""
    q, k, v = (rnd(1100, 2, 64, seed=s, std=w, dtype=dtype) for s, w in ((1, 2.0), (2, 2.0), (3, 1.0)))
    k[600:] *= 3.0                                     # later blocks outgrow the earlier ones
    cu = cu_of(0, 1100)
    o, lse = table(ops).packed_attn_fwd(q, k, v, cu, 0, scale)
    want = ref.packed(q, k, v, cu, scale=scale)
    ref.close(o, want["o"], "o")
    ref.close(lse, want["lse"], "lse")


def test_packed_forward_very_negative_first_block(ops):
    """The first visible score of a row far below zero, the later ones far above."""
    q, k, v = (rnd(400, 1, 64, seed=s) for s in (1, 2, 3))
    q[:, :, 0] = 30.0
    k[:, :, 0] = torch.linspace(-60, 60, 400, device=DEV).to(k.dtype)[:, None]
    cu = cu_of(0, 400)
    ref.close(ops.packed_attention(q, k, v, cu), ref.packed(q, k, v, cu)["o"], "o")


def test_packed_forward_views(ops):
    """q, k, v as slices of one projection, a transposed head layout, an offset that breaks 16 bytes, expanded heads."""
    T, h, d = 333, 4, 64
    qkv = rnd(T, 3, h, d, seed=5)
    cu = cu_of(0, 100, 333)
    want = ref.packed(qkv[:, 0], qkv[:, 1], qkv[:, 2], cu)["o"]
    ref.close(ops.packed_attention(qkv[:, 0], qkv[:, 1], qkv[:, 2], cu), want, "slices")
    hm = qkv.permute(1, 2, 0, 3).contiguous()          # [3, h, T, d]
    q, k, v = (hm[i].transpose(0, 1) for i in range(3))
    ref.close(ops.packed_attention(q, k, v, cu), want, "head-major")
    odd = torch.empty(T * h * d + 1, dtype=torch.bfloat16, device=DEV)[1:].view(T, h, d).copy_(qkv[:, 0])
    ref.close(ops.packed_attention(odd, k, v, cu), want, "odd base")
    one = qkv[:, 1, :1]
    ref.close(ops.packed_attention(q, one.expand(T, h, d), v, cu), ref.packed(q, one.expand(T, h, d), v, cu)["o"], "expanded")


def test_packed_padding_is_not_read(ops):
    """Rows of no sequence may hold anything; their outputs are zero."""
    q, k, v = (rnd(500, 2, 64, seed=s) for s in (1, 2, 3))
    cu = cu_of(2, 200, 450)
    want = ref.packed(q, k, v, cu)["o"]
    for x, bad in ((q, float("nan")), (k, float("inf")), (v, float("nan"))):
        x[:2] = bad
        x[450:] = bad
    o = ops.packed_attention(q, k, v, cu)
    assert not o[:2].any() and not o[450:].any()
    ref.close(o, want, "o")


def test_packed_nonfinite_score_stays_in_its_row(ops):
    """A NaN query makes its own row NaN and no other; a key behind a row (masked) does not reach it whatever it holds."""
    q, k, v = (rnd(200, 1, 64, seed=s) for s in (1, 2, 3))
    cu = cu_of(0, 200)
    base = ops.packed_attention(q, k, v, cu)
    q2, k2 = q.clone(), k.clone()
    q2[50] = float("nan")
    k2[150] = float("nan")
    o = ops.packed_attention(q2, k2, v, cu)
    assert o[50].isnan().all() and o[150:].isnan().all()
    keep = [i for i in range(150) if i != 50]
    assert torch.equal(o[keep], base[keep])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d, residual", [(64, False), (64, True), (128, False), (40, True)])
def test_packed_nonfinite_value_reaches_the_rows_that_see_it(ops, dtype, d, residual):
    """Infinite and NaN value rows: every row that does not see them is as without them, in its own sequence (before them, or
    behind their window) and in the others of the same block of rows."""
    q, k, v = (rnd(300, 4, d, seed=s).to(dtype) for s in (1, 2, 3))
    k, v = k[:, :2].contiguous(), v[:, :2].contiguous()
    cu = cu_of(0, 60, 200, 299)
    grad = residual                                      # a training call writes what the rounding left as well
    for window in (0, 25):
        want = ref.packed(q, k, v, cu, window=window)["o"]
        w = v.clone()
        w[30, 0, 3] = float("inf")
        w[100, 1, 5] = float("nan")
        w[299] = float("nan")                            # padding
        o = ops.packed_attention(q.clone().requires_grad_(grad), k, w, cu, window=window).detach()
        sees = torch.zeros(300, 4, d, dtype=torch.bool, device=DEV)
        sees[30:min(60, 30 + (window or 300)), :2, 3] = True
        sees[100:min(200, 100 + (window or 300)), 2:, 5] = True
        assert not o[sees].isfinite().any() and (o[30, 0, 3] == float("inf")) and o[100, 2, 5].isnan()
        assert o[~sees].isfinite().all()
        ref.close(torch.where(sees, want[0].to(dtype), o), want, f"o {window}")


def test_packed_wrong_table_reads_nothing_out_of_range(ops):
    """Tables that do not ascend or point outside the rows: any output, but the call ends and the next one is right."""
    q, k, v = (rnd(300, 2, 64, seed=s) for s in (1, 2, 3))
    for edges in ((0, 250, 100, 300), (0, 1 << 30), (-(1 << 30), 100, 300), (300, 0), (0, 100, 100000)):
        ops.packed_attention(q, k, v, cu_of(*edges))
    table(ops).tc_check()
    cu = cu_of(0, 300)
    ref.close(ops.packed_attention(q, k, v, cu), ref.packed(q, k, v, cu)["o"], "o")


def test_packed_empty(ops):
    for T, hq in ((0, 4),):
        q = torch.empty(T, hq, 64, dtype=torch.bfloat16, device=DEV)
        assert ops.packed_attention(q, q, q, cu_of(0)).shape == q.shape


# ---- single tokens -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("P,lengths", [(1, (1,)), (7, (0, 7, 3)), (16, (16, 15, 17, -3)), (100, (100, 64, 65, 1, 16)),
                                       (129, (128, 129)), (1000, (1000, 513, 0, 255)), (5000, (5000, 1, 4097))])
@pytest.mark.parametrize("hq,hkv,dim", [(1, 1, 64), (4, 2, 128), (15, 15, 64), (16, 1, 128), (40, 2, 64), (3, 1, 24), (5, 1, 104)])
def test_cached(ops, P, lengths, hq, hkv, dim):
    B = len(lengths)
    q, k, v = rnd(B, hq, dim, seed=1, std=1.5), rnd(B, P, hkv, dim, seed=2, std=1.5), rnd(B, P, hkv, dim, seed=3)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    want = ref.cached(q, k, v, n)
    for b, m in enumerate(lengths):                    # what lies behind the live rows is not read
        k[b, max(0, m):] = float("nan")
        v[b, max(0, m):] = float("inf")
    ref.close(ops.cached_attention(q, k, v, n), want, "o")


@pytest.mark.parametrize("window", [1, 15, 16, 17, 300, 4000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_cached_window_and_types(ops, window, dtype):
    q, k, v = (rnd(*s, seed=i, dtype=dtype) for i, s in enumerate([(4, 8, 64), (4, 2100, 2, 64), (4, 2100, 2, 64)]))
    n = torch.tensor([2100, 0, 5, 1234], dtype=torch.int32, device=DEV)
    ref.close(ops.cached_attention(q, k, v, n, window=window), ref.cached(q, k, v, n, window), "o")


def test_cached_views(ops):
    """A head-major cache, a slice of a larger cache, a query slice of a projection."""
    B, P, h, d = 3, 260, 4, 64
    kv = rnd(2, B, h, P, d, seed=1).transpose(2, 3)
    qkv = rnd(B, 3, h, d, seed=2)
    n = torch.tensor([260, 17, 200], dtype=torch.int32, device=DEV)
    ref.close(ops.cached_attention(qkv[:, 1], kv[0], kv[1], n), ref.cached(qkv[:, 1], kv[0], kv[1], n), "head-major")
    ref.close(ops.cached_attention(qkv[:, 1], kv[0][:, 5:], kv[1][:, 5:], n), ref.cached(qkv[:, 1], kv[0][:, 5:], kv[1][:, 5:], n), "slice")


def test_cached_agrees_with_packed(ops):
    """The last row of each packed sequence is the single-token read of its cache."""
    lens, h, d = (1, 130, 257, 64), 4, 128
    cu = cu_of(0, *torch.tensor(lens).cumsum(0).tolist())
    T = sum(lens)
    q, k, v = (rnd(T, h, d, seed=s) for s in (1, 2, 3))
    P = 300
    kc, vc = (torch.zeros(4, P, h, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    edges = cu.tolist()
    for b, (a, e) in enumerate(zip(edges, edges[1:])):
        kc[b, :e - a], vc[b, :e - a] = k[a:e], v[a:e]
    last = (cu[1:] - 1).long()
    one = ops.cached_attention(q[last], kc, vc, torch.tensor(lens, dtype=torch.int32, device=DEV))
    want, bound = ref.packed(q, k, v, cu)["o"]
    ref.close(one, (want[last], bound[last]), "o")


# ---- scores ------------------------------------------------------------------------------------------------------------
# A log probability is a difference of two fp32 values of the row: each operation's rounding is 2^-24 of values of at most
# R = max - min of the finite entries + log V; a sum of V positive terms in fp32 along a tree of at most V / 256 + 16
# additions adds that many 2^-24 to its logarithm, the exponentials 2 ulp each.
def logp_bound(x, V):
    xf = x.double()
    fin = torch.isfinite(xf)
    hi = torch.where(fin, xf, -torch.inf).amax(-1)
    lo = torch.where(fin, xf, torch.inf).amin(-1)
    r = torch.where(fin.any(-1), (hi - lo).clamp(0, 1e5), 0.0) + 12
    return (r * 8 + V / 256 + 20) * 2.0 ** -24


@pytest.mark.parametrize("V", [1, 2, 7, 8, 31, 255, 256, 259, 2047, 2049, 32000, 50257])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
def test_logprobs_forward(ops, V, dtype, top):
    top = min(top, V)
    N = 13
    x = rnd(N, V, seed=V, dtype=dtype, std=3.0)
    y = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(1)).to(DEV)
    y[3] = -1
    r = ops.token_logprobs(x, y, top=top)
    want, b = ref.logprobs(x, y, top), logp_bound(x, V)
    ref.close(r.logp, (want["logp"], b), "logp")
    ref.close(r.entropy, (want["entropy"], 4 * b), "entropy")      # log S - E: the sum E has terms of up to 1 / e each
    if top:
        assert torch.equal(r.top_ids, want["top_ids"])
        ref.close(r.top_logp, (want["top_logp"], b[:, None]), "top_logp")
    else:
        assert r.top_logp is None and r.top_ids is None


def test_logprobs_ties_and_masks(ops):
    """Constant rows, rows masked down to fewer entries than are asked for, the type's lowest value as a mask, ties."""
    V = 4001
    x = torch.zeros(9, V, device=DEV)
    x[1] = torch.finfo(torch.float32).min                                    # all the lowest value: uniform
    x[2] = -torch.inf
    x[2, [7, 4000, 100]] = torch.tensor([1.0, 2.0, 1.0], device=DEV)         # three entries
    x[3] = torch.finfo(torch.float32).min
    x[3, 17] = 5.0
    x[4] = -torch.inf                                                        # nothing: NaN
    x[5, 9] = torch.nan
    x[6, ::2] = 1.0                                                          # more ties than a list holds
    x[7] = torch.arange(V, device=DEV).flip(0).float()
    x[8, [3, 5]] = torch.finfo(torch.float32).max
    y = torch.tensor([0, 3, 4000, 17, 1, 2, 2, 0, 5], device=DEV)
    r = ops.token_logprobs(x, y, top=8)
    live = [0, 1, 2, 3, 6, 7, 8]
    want = ref.logprobs(x[live], y[live], 8)
    b = logp_bound(x[live], V)
    ref.close(r.logp[live], (want["logp"], b), "logp")
    ref.close(r.entropy[live], (want["entropy"], 4 * b), "entropy")
    assert torch.equal(r.top_ids[live], want["top_ids"])
    for i in (4, 5):
        assert r.logp[i].isnan() and r.entropy[i].isnan()
    assert ((r.top_ids >= 0) & (r.top_ids < V)).all()


def test_logprobs_tokens_outside(ops):
    x = rnd(4, 100, seed=1)
    r = ops.token_logprobs(x, torch.tensor([-1, -100, 100, 1 << 40], device=DEV))
    assert r.logp[0] == 0 and r.logp[1] == 0 and r.logp[2:].isnan().all() and r.entropy.isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logprobs_views(ops, dtype):
    """Rows of a wider matrix at every alignment, columns with a stride, leading dims."""
    big = rnd(6, 700, seed=1, dtype=dtype)
    y = torch.arange(6, device=DEV) * 11
    for a in range(9):
        x = big[:, a:a + 515]
        r, want = ops.token_logprobs(x, y, top=3), ref.logprobs(x, y, 3)
        ref.close(r.logp, (want["logp"], logp_bound(x, 515)), f"offset {a}")
        assert torch.equal(r.top_ids, want["top_ids"])
    x = rnd(700, 6, seed=2, dtype=dtype).t()
    ref.close(ops.token_logprobs(x, y).logp, (ref.logprobs(x, y, 0)["logp"], logp_bound(x, 700)), "transposed")
    x = rnd(2, 3, 100, seed=3, dtype=dtype)
    r = ops.token_logprobs(x, y.view(2, 3) % 100, top=2)
    assert r.logp.shape == (2, 3) and r.top_ids.shape == (2, 3, 2)
    assert ops.token_logprobs(x[:0], y.view(2, 3)[:0], top=2).top_logp.shape == (0, 3, 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows, V", [(20, 1000), (9, 1), (300, 17), (20, 5001), (300, 40001), (2500, 3001), (5000, 2503)])
def test_greedy_entry_is_the_first_of_equals(ops, dtype, rows, V):
    """Coarse entries: many equals, in the vectors and before and behind them (rows start at any alignment)."""
    g = torch.Generator(device=DEV).manual_seed(V)
    x = torch.randint(-6, 7, (rows, V), generator=g, device=DEV).to(dtype)
    x[1] = float("-inf")
    x[2, : V // 2] = float("-inf")
    x[3] = 0
    x[4, : V - 1] = float("nan")
    y = torch.zeros(rows, dtype=torch.int64, device=DEV)
    r = ops.token_logprobs(x, y, top=1)
    key = x.float().nan_to_num(nan=float("-inf"), neginf=float("-inf"), posinf=float("inf"))
    first = (key == key.amax(-1, keepdim=True)).int().argmax(-1)
    assert torch.equal(r.top_ids[:, 0], first)
    keep = torch.arange(rows, device=DEV) > 4
    at = ops.token_logprobs(x, first).logp
    assert torch.equal(r.top_logp[keep, 0], at[keep])
    assert r.top_logp[1].isnan().all() and r.top_logp[4].isnan().all() or V == 1
