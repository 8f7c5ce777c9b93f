"""64-bit references of the rotary, score-attention and gradient-clip operators with the error bounds their arithmetic allows, in plain
torch on the CPU.  A bound is an array beside the value: |kernel - value| <= bound, element by element."""
import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}       # a rounding is off by at most half a step


def rotary_ref(x, pos, axes, base=10000.0, interleaved=False, shared=False, inverse=False):
    """-> (value, bound).  Bound: the angle's fraction of a revolution is rounded to fp32 (half a step of a number <= 1/2: 2^-26 rev, twice
    that after the doubling) and formed from 53-bit factors; sine and cosine are good to 2 units in the last place of a number <= 1
    (2^-23); two products and a sum in fp32 add three half steps; then the output's own rounding."""
    P = sum(axes)
    n = [k for k in axes for _ in range(k)]
    i = [j for k in axes for j in range(k)]
    ax = torch.tensor([a for a, k in enumerate(axes) for _ in range(k)])
    f = torch.tensor([base ** (-p / P) if shared else base ** (-i[p] / n[p]) for p in range(P)], dtype=torch.float64)
    ps = pos.double().cpu()
    if ps.dim() == 2:
        ps = ps[None]
    th = (ps[..., ax] * f)[:, :, None, :] * (-1.0 if inverse else 1.0)
    z = x.detach().double().cpu()
    y, b = z.clone(), z.abs() * 0
    lo = slice(0, 2 * P, 2) if interleaved else slice(0, P)
    hi = slice(1, 2 * P, 2) if interleaved else slice(P, 2 * P)
    c, s = torch.cos(th), torch.sin(th)
    y[..., lo], y[..., hi] = z[..., lo] * c - z[..., hi] * s, z[..., lo] * s + z[..., hi] * c
    ang = 2 * math.pi * 2.0 ** -25 + th.abs() * 2.0 ** -50
    e = (ang + 2.0 ** -23 + 3 * 2.0 ** -24) * (z[..., lo].abs() + z[..., hi].abs())
    b[..., lo], b[..., hi] = e, e
    return y, b + (y.abs() + b) * HALF[x.dtype] + 1e-30


def visible(B, Sq, Sk, causal=False, prefix=None, q_start=None, q_doc=None, k_doc=None):
    p = torch.arange(Sq)[None, :] + (torch.full((B, 1), Sk - Sq) if q_start is None else q_start.cpu().long()[:, None])
    j = torch.arange(Sk)
    vis = torch.ones(B, Sq, Sk, dtype=torch.bool)
    if causal:
        vis = j[None, None, :] <= p[:, :, None]
        if prefix is not None:
            vis = vis | (j[None, None, :] < prefix.cpu()[:, None, None])
    if q_doc is not None:
        vis = vis & (q_doc.cpu()[:, :, None] == k_doc.cpu()[:, None, :]) & (k_doc.cpu()[:, None, :] >= 0)
    return vis, (p[:, :, None] - j[None, None, :]).abs().double()


def attention_ref(q, k, v, go=None, scale=None, softcap=0.0, slopes=None, causal=False, prefix=None, q_start=None, q_doc=None, k_doc=None):
    """-> {name: (value, bound)} for out and, with ``go``, dq, dk, dv, dslopes.

    Bounds (u = half a step of the tensors' type, w = 2^-24): a score carries the rounding of its D fp32 products and of the few fp32
    operations behind it, and the tanh's absolute error (2^-20 of the cap); e = what that and the exponential (2 units) do to a
    probability relative to itself, twice (numerator and sum).  P and dS enter the next product rounded to the tensors' type (u each);
    delta is formed from the rounded output (u sum |go| |o|); every fp32 sum of n terms may lose n w of the terms' absolute sum."""
    dt = q.dtype
    u, w = HALF[dt], 2.0 ** -24
    keep = None
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    vis, dist = visible(B, Sq, Sk, causal, prefix, q_start, q_doc, k_doc)
    clean = lambda t, dead: t.detach().double().cpu().masked_fill(dead[:, :, None, None], 0.0)      # rows nobody may use: whatever they hold
    dead_q = (q_doc.cpu() < 0) if q_doc is not None else torch.zeros(B, Sq, dtype=torch.bool)
    dead_k = ~vis.any(dim=1)
    qd = clean(q, dead_q).permute(0, 2, 1, 3)
    G = H // Hk
    kd = clean(k, dead_k).permute(0, 2, 1, 3).repeat_interleave(G, dim=1)
    vd = clean(v, dead_k).permute(0, 2, 1, 3).repeat_interleave(G, dim=1)
    t = scale * (qd @ kd.transpose(-1, -2))
    ta = abs(scale) * (qd.abs() @ kd.abs().transpose(-1, -2))
    es = (D + 4) * w * ta
    th = torch.zeros_like(t)
    if softcap > 0:
        th = torch.tanh(t / softcap)
        t = softcap * th
        es = es + softcap * 2.0 ** -20
    if slopes is not None:
        sl = slopes.detach().double().cpu()[None, :, None, None]
        t = t - sl * dist[:, None]
        es = es + 4 * w * (sl * dist[:, None]).abs()
    es = es + 4 * w * t.abs()
    vis = vis[:, None]
    t = t.masked_fill(~vis, -math.inf)
    mx = t.amax(dim=-1, keepdim=True) if Sk else torch.zeros(B, H, Sq, 1, dtype=torch.float64)
    mx = torch.where(torch.isinf(mx), torch.zeros_like(mx), mx)
    e = torch.exp(t - mx)
    l = e.sum(dim=-1, keepdim=True)
    P = e / torch.where(l > 0, l, torch.ones_like(l))
    esm = torch.where(vis, es, torch.zeros_like(es)).amax(dim=-1, keepdim=True) if Sk else mx * 0
    rel = 2 * (esm + 2.0 ** -21) + (Sk + 64) * w                      # of one probability
    o = P @ vd
    A = P @ vd.abs()
    pu = 0.0 if dt == torch.float32 else u                            # rounding of P and dS between the products
    res = {}
    ob = o.abs() * u + (pu + rel + Sk * w) * A
    back = lambda x: x.permute(0, 2, 1, 3)
    res["out"] = (back(o), back(ob) + 1e-30)
    if go is None:
        return res
    gd = clean(go, dead_q).permute(0, 2, 1, 3)
    dP = gd @ vd.transpose(-1, -2)
    dPa = gd.abs() @ vd.abs().transpose(-1, -2)
    delta = (gd * o).sum(-1, keepdim=True)
    # delta is formed from the stored output: its whole error (rounding included) times |go|
    ed = (gd.abs() * (ob + D * w * o.abs())).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    eS = rel * P * (dP - delta).abs() + P * (D * w * dPa + ed) + 4 * w * P * (dPa + delta.abs())
    cd = 1 - th * th
    ec = (4 * es / softcap + 2.0 ** -19) if softcap > 0 else 0.0      # of the cap's derivative, absolute
    dT = dS * cd
    eT = eS * cd + (dS.abs() + eS) * ec
    group = lambda x: x.view(B, Hk, G, Sk, D).sum(2)
    n = Sq * G
    eT = eT + pu * (dT.abs() + eT)
    dq, eq = scale * (dT @ kd), abs(scale) * ((eT + Sk * w * dT.abs()) @ kd.abs())
    dk, ek = scale * group(dT.transpose(-1, -2) @ qd), abs(scale) * group((eT + n * w * dT.abs()).transpose(-1, -2) @ qd.abs())
    eP = (pu + rel + n * w) * P
    dv, ev = group(P.transpose(-1, -2) @ gd), group(eP.transpose(-1, -2) @ gd.abs())
    for name, x, ex in (("dq", dq, eq), ("dk", dk, ek), ("dv", dv, ev)):
        res[name] = (back(x), back(ex + (x.abs() + ex) * u) + 1e-30)
    if slopes is not None:
        ds = -(dS * dist[:, None]).sum(dim=(0, 2, 3))
        eds = ((eS + (Sk + 8) * w * dS.abs()) * dist[:, None]).sum(dim=(0, 2, 3))
        res["dslopes"] = (ds, eds + ds.abs() * w + 1e-30)
    return res


def check(name, got, want):
    value, bound = want
    got = got.detach().double().cpu()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    assert torch.isfinite(got).all() or not torch.isfinite(value).all(), f"{name}: not finite"
    bad = (got - value).abs() > bound
    if bad.any():
        i = ((got - value).abs() / bound).argmax()
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} beyond the bound; worst at {i.item()}: got {got.flatten()[i].item():.8g}, "
                             f"want {value.flatten()[i].item():.8g} +- {bound.flatten()[i].item():.3g}")
