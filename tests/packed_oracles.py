"""64-bit statements of the operators on packed sequences, sequence by sequence, with bounds on what the kernels' roundings
can do to each output element.

u = eps / 2 of the element type is the relative error of one rounding.  The kernels round the weights p (relative u) before
the product with v, ds (relative u) before the products with k and q, o (relative u), and each gradient (relative u); the
backward forms delta = do . o from the rounded o.  Scores are fp32 sums of D exact products: an absolute error of at most
(D + 8) 2^-24 times scale sum |q_d k_d|, the 8 for scaling, subtracting the maximum and the exponential's own 2 ulp;
twice that, relative, in a normalised weight, and as much again for the fp32 sums over keys.  `F32` times the weight bounds
all of it."""

import math

import torch


def u_of(dtype):
    return torch.finfo(dtype).eps / 2


def packed(q, k, v, cu, window=0, scale=None, do=None):
    """dict of name -> (value, bound) in 64 bits; q / k / v / do in the dtype the operator is given."""
    T, Hq, D = q.shape
    g = Hq // k.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    u = u_of(q.dtype)
    qd, kd, vd = (x.detach().double() for x in (q, k, v))
    dd = None if do is None else do.double()
    z = lambda x: torch.zeros_like(x)
    o, bo, lse, bl = z(qd), z(qd), torch.full((Hq, T), -math.inf, dtype=torch.float64, device=q.device), None
    bl = torch.zeros_like(lse)
    dq, bq, dk, bk, dv, bv = z(qd), z(qd), z(kd), z(kd), z(vd), z(vd)
    edges = cu.tolist()
    for a, b in zip(edges, edges[1:]):
        n = b - a
        if n <= 0:
            continue
        i = torch.arange(n, device=q.device)
        seen = i[None, :] <= i[:, None]
        if window:
            seen &= i[None, :] > i[:, None] - window
        for h in range(Hq):
            c = h // g
            Q, K, V = qd[a:b, h], kd[a:b, c], vd[a:b, c]
            s = torch.where(seen, Q @ K.T * scale, -math.inf)
            p = torch.softmax(s, -1)
            f32 = 4 * (D + 8) * 2.0 ** -24 * scale * (Q.abs() @ K.abs().T).max().item() + 2.0 ** -20
            e = u + f32                                              # relative error of a rounded weight
            pa = p @ V.abs()
            o[a:b, h] = p @ V
            bo[a:b, h] = e * pa + u * o[a:b, h].abs()
            lse[h, a:b] = torch.logsumexp(s, -1)
            bl[h, a:b] = f32 * (1 + lse[h, a:b].abs())
            if dd is None:
                continue
            G = dd[a:b, h]
            dp = G @ V.T
            delta = (G * o[a:b, h]).sum(-1, keepdim=True)
            ds = p * (dp - delta) * scale
            e_delta = (G.abs() * bo[a:b, h]).sum(-1, keepdim=True) + f32 * (G.abs() @ V.abs().T).amax(-1, keepdim=True)
            e_ds = (u + f32) * ds.abs() + (1 + u) * p * scale * e_delta
            dv[a:b, c] += p.T @ G
            bv[a:b, c] += e * (p.T @ G.abs())
            dq[a:b, h] = ds @ K
            bq[a:b, h] = e_ds @ K.abs() + f32 * (ds.abs() @ K.abs())
            dk[a:b, c] += ds.T @ Q
            bk[a:b, c] += e_ds.T @ Q.abs() + f32 * (ds.abs().T @ Q.abs())
    tiny = 1e-30
    out = {"o": (o, bo * (1 + u) + tiny), "lse": (lse, bl)}
    if dd is not None:
        for name, x, bx in (("dq", dq, bq), ("dk", dk, bk), ("dv", dv, bv)):
            out[name] = (x, bx * (1 + u) + u * x.abs() + tiny)
    return out


def cached(q, k, v, lengths, window=0, scale=None):
    """(value, bound): one query per sequence; only live rows are looked at."""
    B, Hq, D = q.shape
    g = Hq // k.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    u = u_of(q.dtype)
    o = torch.zeros(B, Hq, D, dtype=torch.float64, device=q.device)
    bo = torch.zeros_like(o)
    for b, n in enumerate(lengths.tolist()):
        n = min(max(n, 0), k.shape[1])
        lo = max(0, n - window) if window else 0
        if n <= lo:
            continue
        K = k[b, lo:n].double().repeat_interleave(g, 1).transpose(0, 1)
        V = v[b, lo:n].double().repeat_interleave(g, 1).transpose(0, 1)
        Q = q[b].double()[:, None]
        p = torch.softmax(Q @ K.transpose(1, 2) * scale, -1)
        f32 = 4 * (D + 8) * 2.0 ** -24 * scale * (Q.abs() @ K.abs().transpose(1, 2)).max().item() + 2.0 ** -20
        o[b] = (p @ V)[:, 0]
        bo[b] = (u + f32) * (p @ V.abs())[:, 0] + u * o[b].abs()
    return o, bo * (1 + u) + 1e-30


def logprobs(x, y, top, g_lp=None, g_h=None):
    """dict of name -> value in 64 bits; rows without target have logp 0."""
    xd = x.detach().double()
    lp = torch.log_softmax(xd, -1)
    p = lp.exp()
    h = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    has = y >= 0
    out = {"logp": torch.where(has, lp.gather(-1, y.clamp_min(0)[:, None])[:, 0], 0.0), "entropy": h}
    order = xd.sort(dim=-1, descending=True, stable=True).indices[:, :top]
    out |= {"top_ids": order, "top_logp": lp.gather(-1, order)}
    if g_lp is not None or g_h is not None:
        gl = torch.zeros_like(h) if g_lp is None else g_lp.double() * has
        gh = torch.zeros_like(h) if g_h is None else g_h.double()
        hot = torch.zeros_like(p).scatter_(-1, y.clamp_min(0)[:, None], 1.0)
        out["dx"] = gl[:, None] * (hot - p) - gh[:, None] * torch.where(p > 0, p * (lp + h[:, None]), 0.0)
    return out


def close(got, want, what):
    """Every element within its bound; non-finite values equal."""
    value, bound = want
    got = got.detach().double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    fine = torch.isfinite(value)
    assert torch.equal(torch.isfinite(got), fine) and torch.equal(got[~fine & ~value.isnan()], value[~fine & ~value.isnan()]), what
    off = ((got - value).abs() / bound.clamp_min(1e-300))[fine]
    worst = off.max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} of the bound"
    return worst
