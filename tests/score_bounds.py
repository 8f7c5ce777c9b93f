"""Attention with changed scores in 64 bits, with bounds that follow the SCORES: what the cap's tanh may be off by is a part of the capped score
(not of the cap), and a distance counts from the nearest position inside the keys (a shift that all keys of a row share changes nothing).
|kernel - value| <= bound, element by element; plain torch on the CPU."""
import math

import torch

from operator_refs import HALF, visible


def capped(s, es, cap):
    """cap tanh(s / cap), what it may be off by for a score off by es, its derivative and what that may be off by.  The kernels' tanh is good
    to 2^-20 of its value (a fit of 7e-7 with its roundings in bf16, tanhf in fp32); the derivative 1 - tanh^2 doubles that and adds two roundings;
    an inner error moves both within the interval [|s| - es, |s| + es], where they are monotonous."""
    if cap == 0:
        return s, es, torch.ones_like(s), torch.zeros_like(s)
    lo, hi = (s.abs() - es).clamp_min(0) / cap, (s.abs() + es) / cap
    sech2 = lambda y: 1.0 / torch.cosh(y.clamp_max(300.0)) ** 2
    t = cap * torch.tanh(s / cap)
    et = torch.maximum(cap * torch.tanh(hi) - t.abs(), t.abs() - cap * torch.tanh(lo)) + 2.0 ** -20 * t.abs()
    d = sech2(s.abs() / cap)
    ed = torch.maximum(sech2(lo) - d, d - sech2(hi)) + 2.0 ** -19 * (t / cap) ** 2 + 2.0 ** -23
    return t, et, d, ed


def attention_bounds(q, k, v, go=None, scale=None, softcap=0.0, slopes=None, causal=False, prefix=None, q_start=None, q_doc=None, k_doc=None):
    """-> {"out", "dq", "dk", "dv", "dslopes"}: (value, bound).  u = half a step of the tensors' type, w = 2^-24.  A score: D products and their
    sums (D w of the absolute sum), the scale and the change to base 2 (4 w), the cap (above), the distance and its subtraction (4 w).  A
    probability is off by the factor e^(2 e), e = the largest such error among its row's visible scores, 2^-21 for the exponential and the
    row's fp32 sum.  P and dS are rounded to the tensors' type between the products; delta comes from the output (in bf16 with its rounding's
    residual, itself rounded); a sum of n terms may lose n w of their absolute sum."""
    u, w = HALF[q.dtype], 2.0 ** -24
    pu = 0.0 if q.dtype == torch.float32 else u
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    vis, _ = visible(B, Sq, Sk, causal, prefix, q_start, q_doc, k_doc)
    p = torch.arange(Sq)[None] + (torch.full((B, 1), Sk - Sq) if q_start is None else q_start.cpu().long()[:, None])
    dist = (p.clamp(0, Sk - 1)[:, :, None] - torch.arange(Sk)).abs().double()[:, None]
    heads = lambda t, n: t.detach().double().cpu().permute(0, 2, 1, 3).repeat_interleave(n, dim=1)
    back = lambda t: t.permute(0, 2, 1, 3)
    group = lambda t: t.view(B, Hk, G, Sk, D).sum(2)
    qd, kd, vd = heads(q, 1), heads(k, G), heads(v, G)
    vis = vis[:, None]
    s = scale * (qd @ kd.transpose(-1, -2))
    t, es, cd, ec = capped(s, (D + 4) * w * abs(scale) * (qd.abs() @ kd.abs().transpose(-1, -2)), softcap)
    es = es + 4 * w * t.abs()
    if slopes is not None:
        bias = slopes.detach().double().cpu()[None, :, None, None] * dist
        t, es = t - bias, es + 4 * w * bias.abs()
    t = t.masked_fill(~vis, -math.inf)
    top = t.amax(-1, keepdim=True)
    e = torch.exp(t - torch.where(top == -math.inf, 0.0, top))
    P = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
    worst = es.masked_fill(~vis, 0.0).amax(-1, keepdim=True)
    rel = torch.expm1((2 * (worst + 2.0 ** -21) + (Sk + 64) * w).clamp_max(50.0))
    eP = torch.minimum(rel * P, torch.ones_like(P))
    o = P @ vd
    eo = (eP + (pu + Sk * w) * P) @ vd.abs()
    res = {"out": (back(o), back(eo + u * (o.abs() + eo)) + 1e-30)}
    if go is None:
        return res
    gd = heads(go, 1)
    dP, dPa = gd @ vd.transpose(-1, -2), gd.abs() @ vd.abs().transpose(-1, -2)
    delta = (gd * o).sum(-1, keepdim=True)
    ed = (gd.abs() * (eo + (u * u + 2 * D * w) * o.abs())).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    eS = eP * (dP - delta).abs() + (P + eP) * (D * w * dPa + ed + 4 * w * (dPa + delta.abs()))
    dT = dS * cd
    eT = eS * cd + (dS.abs() + eS) * ec
    eT = eT + pu * (dT.abs() + eT)
    n = Sq * G
    grads = {"dq": (scale * (dT @ kd), abs(scale) * ((eT + Sk * w * dT.abs()) @ kd.abs())),
             "dk": (scale * group(dT.transpose(-1, -2) @ qd), abs(scale) * group((eT + n * w * dT.abs()).transpose(-1, -2) @ qd.abs())),
             "dv": (group(P.transpose(-1, -2) @ gd), group((eP + (pu + n * w) * P).transpose(-1, -2) @ gd.abs()))}
    for name, (x, ex) in grads.items():
        res[name] = (back(x), back(ex + u * (x.abs() + ex)) + 1e-30)
    if slopes is not None:
        x, ex = -(dS * dist).sum((0, 2, 3)), ((eS + (Sk + 8) * w * dS.abs()) * dist).sum((0, 2, 3))
        res["dslopes"] = (x, ex + x.abs() * w + 1e-30)
    return res
