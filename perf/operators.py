"""Measured cases of three operators of this package's training step: rotary positions with several axes (``rotary``), attention
whose scores are capped, biased by distance and masked by documents and prefixes (``attention``), and the global gradient norm over
many tensors with clipping (``clip``).

With ``own`` false ``run`` computes each operator's plain form out of elementary torch operations in 32 bits (64 for the angles of the
rotary positions and the long sum of the norm); with ``own`` true it makes the calls a user makes:

    attention_ops.RotaryPlan(head_dim, axes, ...)      attention_ops.rotary(q, k, pos, plan)
    attention_ops.score_attention(q, k, v, scale=, softcap=, slopes=, causal=, prefix=, q_doc=, k_doc=, q_start=)
    optim.clip_grad_norm_(params, max_norm, norm_type=)
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp32": 4}


# ---------------------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------------------
def _rot(name, B, S, H, Hk, D, axes, dtype="bf16", train=True, interleaved=False, fractional=False, start=0, packed=False):
    return {"name": name, "op": "rotary", "B": B, "S": S, "H": H, "Hk": Hk, "D": D, "nt": axes[0], "nh": axes[1], "nw": axes[2],
            "dtype": dtype, "train": train, "interleaved": interleaved, "fractional": fractional, "start": start, "packed": packed}


def _att(name, B, Sq, Sk, H, Hk, D, dtype="bf16", train=True, mask="full", cap=0.0, slopes=False, docs=0, pad=False, packed=False):
    return {"name": name, "op": "attention", "B": B, "Sq": Sq, "Sk": Sk, "H": H, "Hk": Hk, "D": D, "dtype": dtype, "train": train,
            "mask": mask, "cap": cap, "slopes": slopes, "docs": docs, "pad": pad, "packed": packed}


def _clip(name, d, layers, levels, dtype="fp32", norm="2", max_norm=1.0, odd=False):
    return {"name": name, "op": "clip", "d": d, "layers": layers, "levels": levels, "dtype": dtype, "norm": norm, "max_norm": max_norm,
            "odd": odd}


def listed():
    return [
        # one new token of each of four sequences, at positions an hour of video reaches: a launch and little else
        _rot("rotary_token", 4, 1, 16, 4, 128, (16, 24, 24), train=False, start=262144),
        # the benchmark encoder's tokens (196 patches + 512 words, four heads of 192), Q and K as thirds of one packed projection
        _rot("rotary_fusion_step", 32, 708, 4, 4, 192, (32, 32, 32), packed=True),
        # fp32, an odd number of tokens, patch positions of a coarse level on the fine level's grid, channels that are not rotated
        _rot("rotary_fp32_levels", 3, 917, 6, 2, 88, (9, 13, 13), dtype="fp32", interleaved=True, fractional=True),
        # next-token attention of a small batch over a long context, shared key heads: the bytes of the keys and values
        _att("attention_token", 4, 1, 16411, 16, 4, 128, train=False, mask="causal", cap=30.0, slopes=True),
        # the smallest call: one query each over a short caption
        _att("attention_short", 2, 1, 77, 4, 4, 64, train=False, mask="causal", slopes=True),
        # the benchmark encoder's layer with the visual tokens as a bidirectional prefix and padded captions, forward and backward
        _att("attention_fusion_step", 32, 708, 708, 4, 4, 192, mask="prefix", cap=50.0, pad=True, packed=True),
        # packed documents of ragged lengths, shared key heads, capped scores: long-sequence training
        _att("attention_documents", 1, 8192, 8192, 16, 4, 64, mask="causal", cap=50.0, docs=11),
        # the longest forward: a causal prompt with distance bias
        _att("attention_prompt", 1, 16384, 16384, 8, 2, 128, train=False, mask="causal", slopes=True),
        # fp32 training, odd sizes, learned distance slopes
        _att("attention_fp32", 2, 355, 417, 6, 3, 88, dtype="fp32", mask="prefix", slopes=True, pad=True),
        # gradients of a one-layer encoder: latency
        _clip("clip_small", 64, 1, 1, odd=True),
        # the four encoders of the feature levels, 208 tensors
        _clip("clip_levels", 768, 4, 4),
        # bf16 weights with fp32 biases and norms, the largest set
        _clip("clip_mixed_large", 1792, 12, 1, dtype="mixed", odd=True),
    ]


_HEADS = [(1, 1), (2, 1), (4, 4), (4, 2), (6, 2), (8, 2), (8, 8), (12, 4), (16, 4), (14, 2)]
_DIMS = [16, 24, 32, 40, 64, 72, 88, 96, 128, 160, 176, 192, 224, 256]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_any(rng):
    op = rng.choice(["rotary", "rotary", "attention", "attention", "attention", "clip"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    H, Hk = rng.choice(_HEADS)
    D = rng.choice(_DIMS)
    if op == "rotary":
        total = rng.randint(3, D // 2) if rng.random() < 0.5 else D // 2
        nt = rng.randint(0, total - 2)
        nh = rng.randint(1, total - nt - 1)
        return _rot("", rng.randint(1, 32), _log(rng, 1, 4096), H, Hk, D, (nt, nh, total - nt - nh), dtype=dtype, train=rng.random() < 0.6,
                    interleaved=rng.random() < 0.5, fractional=rng.random() < 0.3, start=_log(rng, 1, 1000000) - 1, packed=rng.random() < 0.5)
    if op == "attention":
        kind = rng.random()
        Sk = _log(rng, 1, 16384)
        if kind < 0.3:
            Sq, train = rng.randint(1, min(4, Sk)), False
        elif kind < 0.45:
            Sq, train = _log(rng, 1, Sk), rng.random() < 0.5
        else:
            Sq, train = Sk, rng.random() < 0.7
        docs = rng.randint(2, 12) if (Sq == Sk and rng.random() < 0.35) else 0
        return _att("", _log(rng, 1, 32), Sq, Sk, H, Hk, D, dtype=dtype, train=train, mask=rng.choice(["full", "causal", "prefix"]),
                    cap=rng.choice([0.0, 0.0, 30.0, 50.0]), slopes=rng.random() < 0.4, docs=docs, pad=docs == 0 and rng.random() < 0.4,
                    packed=Sq == Sk and rng.random() < 0.4)
    return _clip("", 8 * _log(rng, 8, 224), rng.randint(1, 12), rng.randint(1, 4), dtype=rng.choice(["fp32", "bf16", "mixed"]),
                 norm=rng.choice(["2", "2", "inf"]), max_norm=rng.choice([0.5, 1.0, 1e6]), odd=rng.random() < 0.5)


def draw(rng):
    """A case no costlier than the largest listed one of its operator; attention's plain form holds B * H * Sq * Sk scores, so those
    are bounded too."""
    cap = {}
    for c in listed():
        w = work(c)
        size = c["B"] * c["H"] * c["Sq"] * c["Sk"] * (2 if c["train"] else 1) if c["op"] == "attention" else 0
        old = cap.get(c["op"], (0, 0, 0))
        cap[c["op"]] = (max(old[0], w["bytes"]), max(old[1], w["flops"]), max(old[2], size))
    while True:
        c = _draw_any(rng)
        w = work(c)
        size = c["B"] * c["H"] * c["Sq"] * c["Sk"] * (2 if c["train"] else 1) if c["op"] == "attention" else 0
        lim = cap[c["op"]]
        # an fp32 product costs sixteen bf16 ones on the matrix units
        if w["bytes"] <= lim[0] and w["flops"] * (16 if c.get("dtype") == "fp32" else 1) <= lim[1] and size <= lim[2]:
            del c["name"]
            return c


# ---------------------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda:0").manual_seed(seed)


def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda:0") * scale).to(dtype)


def _grid_positions(case, seed):
    """[B, S, 3] (time, height, width): frames of a patch grid over the first tokens, text behind them that counts on from the largest
    coordinate on every axis; every sample's video starts at a frame of its own."""
    B, S = case["B"], case["S"]
    side = 14 if S >= 250 else 4
    n_vis = min(S * 3 // 4, max(1, S // 3) // (side * side) * side * side + side * side) if S > 1 else 0
    i = np.arange(n_vis)
    vis = np.stack([i // (side * side), i // side % side, i % side], axis=1).astype(np.float64)
    if case["fractional"]:
        vis[:, 1:] = (vis[:, 1:] + 0.5) * (28.0 / side) - 0.5        # a coarse level's patch centres on the finest level's grid
    last = math.floor(vis.max()) + 1 if n_vis else 0
    txt = np.repeat(last + np.arange(S - n_vis, dtype=np.float64)[:, None], 3, axis=1)
    pos = np.concatenate([vis, txt], axis=0)[None].repeat(B, axis=0)
    pos[:, :, 0] += case["start"] + (seed * 7 + np.arange(B) * 13)[:, None] % 97
    return torch.from_numpy(pos.astype(np.float32 if case["fractional"] else np.int32)).to("cuda:0")


def _doc_lengths(case, b):
    """Document lengths of sample b (they add up to <= Sk; what is left is padding): a function of the case, so that ``work`` knows
    the visible pairs."""
    Sk = case["Sk"]
    rng = random.Random(Sk * 131 + case["docs"] * 17 + b)
    if case["docs"] == 0:
        return [Sk - (rng.randint(0, (Sk - 1) // 2) if case["pad"] else 0)]
    n = min(case["docs"], Sk)
    cuts = sorted(rng.sample(range(1, Sk), n - 1)) if n > 1 else []
    return [e - s for s, e in zip([0] + cuts, cuts + [Sk])]


def _first_token(case, n):
    """Padding follows the tokens of a whole sequence and precedes those of a cache that its last queries read."""
    return case["Sk"] - n if case["pad"] and case["Sq"] < case["Sk"] else 0


def _has_docs(case):
    return case["docs"] > 0 or case["pad"]


def _prefix_of(case, b):
    return (case["Sk"] * 196 // 708 if case["Sk"] >= 708 else case["Sk"] // 3) - b % 3 if case["mask"] == "prefix" else 0


def _visible_pairs(case):
    """Number of (query, key) pairs of one head over the batch that take part."""
    total = 0
    Sq, Sk = case["Sq"], case["Sk"]
    for b in range(case["B"]):
        p = np.arange(Sk - Sq, Sk)
        lengths = _doc_lengths(case, b)
        a = _first_token(case, sum(lengths))
        for n in lengths:
            q = p[(p >= a) & (p < a + n)]
            if case["mask"] == "full":
                total += len(q) * n
            else:
                hi = np.minimum(np.maximum(q + 1, max(0, _prefix_of(case, b))), a + n)
                total += int(np.maximum(hi - a, 0).sum())
            a += n
    return total


def _clip_shapes(case):
    d = case["d"]
    ff = 2 * d
    enc = []
    for _ in range(case["layers"]):
        enc += [(3 * d, d), (3 * d,), (d, d), (d,), (ff, d), (ff,), (d, ff), (d,), (d,), (d,), (d,), (d,)]
    enc += [(1, d), (1, d), (d,), (d,)]
    shapes = enc * case["levels"]
    if case["odd"]:                              # class heads: 87 nouns, 74 verbs, one time
        shapes = shapes + [(87, d), (87,), (74, d), (74,), (1, d), (1,)]
    return shapes


def _clip_dtype(case, shape):
    if case["dtype"] == "mixed":
        return torch.bfloat16 if len(shape) == 2 else torch.float32
    return _DT[case["dtype"]]


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "rotary":
        B, S, H, Hk, D = (case[k] for k in ("B", "S", "H", "Hk", "D"))
        dt = _DT[case["dtype"]]
        if case["packed"]:
            qkv = _randn(g, (B, S, H + 2 * Hk, D), dt)
            q, k = qkv[:, :, :H], qkv[:, :, H:H + Hk]
        else:
            q, k = _randn(g, (B, S, H, D), dt), _randn(g, (B, S, Hk, D), dt)
        st = {"case": case, "q": q.requires_grad_(case["train"]), "k": k.requires_grad_(case["train"]), "pos": _grid_positions(case, seed)}
        if case["train"]:
            st["gq"], st["gk"] = _randn(g, (B, S, H, D), dt), _randn(g, (B, S, Hk, D), dt)
        axes = (case["nt"], case["nh"], case["nw"])
        if own:
            from transfusion_amd import attention_ops
            st["plan"] = attention_ops.RotaryPlan(D, axes, base=10000.0, interleaved=case["interleaved"], device="cuda:0")
        else:
            inv = [10000.0 ** (-i / n) for n in axes for i in range(n)]
            st["inv"] = torch.tensor(inv, dtype=torch.float64, device="cuda:0")
            st["axis"] = torch.tensor([a for a, n in enumerate(axes) for _ in range(n)], device="cuda:0")
        return st
    if case["op"] == "attention":
        B, Sq, Sk, H, Hk, D = (case[k] for k in ("B", "Sq", "Sk", "H", "Hk", "D"))
        dt = _DT[case["dtype"]]
        if case["packed"]:                       # the layout of a fused projection: Q | K | V side by side in one row
            qkv = _randn(g, (B, Sk, H + 2 * Hk, D), dt)
            q, k, v = qkv[:, :, :H], qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:]
        else:
            q, k, v = _randn(g, (B, Sq, H, D), dt), _randn(g, (B, Sk, Hk, D), dt), _randn(g, (B, Sk, Hk, D), dt)
        st = {"case": case, "q": q, "k": k, "v": v, "slopes": None, "prefix": None, "q_doc": None, "k_doc": None,
              "scale": 1.0 / math.sqrt(D)}
        if case["slopes"]:
            st["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device="cuda:0") * (1.0 + 0.01 * (seed % 7))
        if case["mask"] == "prefix":
            st["prefix"] = torch.tensor([max(0, _prefix_of(case, b)) for b in range(B)], dtype=torch.int32, device="cuda:0")
        if _has_docs(case):
            doc = np.full((B, Sk), -1, np.int32)
            for b in range(B):
                lengths = _doc_lengths(case, b)
                a = _first_token(case, sum(lengths))
                for i, n in enumerate(lengths):
                    doc[b, a:a + n] = i
                    a += n
            st["k_doc"] = torch.from_numpy(doc).to("cuda:0")
            st["q_doc"] = st["k_doc"][:, Sk - Sq:].contiguous()
        if case["train"]:
            st["go"] = _randn(g, (B, Sq, H, D), dt)
            for name in ("q", "k", "v", "slopes"):
                if st[name] is not None:
                    st[name].requires_grad_(True)
        return st
    # the gradients are slices of one buffer per type, as this package's training step keeps them (slices start at multiples of 16
    # bytes, or, with odd sizes, wherever the one before ends); the buffers are what run returns
    shapes = _clip_shapes(case)
    place, length = [], {}
    for shape in shapes:
        dt, n = _clip_dtype(case, shape), math.prod(shape)
        place.append((dt, length.get(dt, 0), n))
        length[dt] = length.get(dt, 0) + (n if case["odd"] else (n + 7) // 8 * 8)
    flat = {dt: _randn(g, (n,), dt, 0.02 * (1.0 + 0.1 * (seed % 5))) for dt, n in length.items()}
    params = []
    for shape, (dt, a, n) in zip(shapes, place):
        p = torch.empty(shape, dtype=dt, device="cuda:0").requires_grad_(True)
        p.grad = flat[dt][a:a + n].view(shape)
        params.append(p)
    return {"case": case, "params": params, "flat": list(flat.values())}


# ---------------------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------------------
def _rotate_plain(x, cos, sin, interleaved):
    P = cos.shape[-1]
    xf = x.float()
    c, s = cos[:, :, None, :], sin[:, :, None, :]
    if interleaved:
        a, b = xf[..., 0:2 * P:2], xf[..., 1:2 * P:2]
        rot = torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2)
    else:
        a, b = xf[..., :P], xf[..., P:2 * P]
        rot = torch.cat((a * c - b * s, a * s + b * c), dim=-1)
    return torch.cat((rot, xf[..., 2 * P:]), dim=-1).to(x.dtype)


def _mask_plain(st):
    """[B, 1, Sq, Sk] truth values: which keys a query attends; None when it is all of them."""
    c = st["case"]
    Sq, Sk = c["Sq"], c["Sk"]
    vis = None
    if c["mask"] != "full":
        p = torch.arange(Sk - Sq, Sk, device="cuda:0")
        j = torch.arange(Sk, device="cuda:0")
        vis = (j[None, :] <= p[:, None])[None]
        if st["prefix"] is not None:
            vis = vis | (j[None, None, :] < st["prefix"][:, None, None])
        vis = vis[:, None]
    if st["k_doc"] is not None:
        same = (st["q_doc"][:, :, None] == st["k_doc"][:, None, :]) & (st["k_doc"][:, None, :] >= 0)
        vis = same[:, None] if vis is None else vis & same[:, None]
    return vis


def _attention_plain(st):
    c = st["case"]
    B, Sq, Sk, H, Hk, D = (c[k] for k in ("B", "Sq", "Sk", "H", "Hk", "D"))
    q = st["q"].float().transpose(1, 2)
    k = st["k"].float().transpose(1, 2).repeat_interleave(H // Hk, dim=1)
    v = st["v"].float().transpose(1, 2).repeat_interleave(H // Hk, dim=1)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * st["scale"]
    if c["cap"] > 0:
        s = c["cap"] * torch.tanh(s / c["cap"])
    if st["slopes"] is not None:
        p = torch.arange(Sk - Sq, Sk, device="cuda:0")
        dist = (p[:, None] - torch.arange(Sk, device="cuda:0")[None, :]).abs().float()
        s = s - st["slopes"][:, None, None] * dist
    vis = _mask_plain(st)
    if vis is not None:
        s = s.masked_fill(~vis, -math.inf)
    m = s.detach().amax(dim=-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = torch.exp(s - m)
    l = e.sum(dim=-1, keepdim=True)
    l = torch.where(l == 0, torch.ones_like(l), l)
    return torch.matmul(e / l, v).transpose(1, 2).to(st["q"].dtype)


def _clip_plain(params, max_norm, norm):
    grads = [p.grad for p in params]
    if norm == "inf":
        total = torch.stack([g.float().abs().amax() for g in grads]).amax()
    else:
        total = torch.stack([(g.float() ** 2).sum(dtype=torch.float64) for g in grads]).sum().sqrt().float()
    coef = torch.clamp(max_norm / (total + 1e-6), max=1.0)
    for g in grads:
        g.copy_(g.float() * coef)
    return total


def run(state):
    c = state["case"]
    if c["op"] == "rotary":
        q, k = state["q"], state["k"]
        with torch.set_grad_enabled(c["train"]):
            if own:
                from transfusion_amd import attention_ops
                qr, kr = attention_ops.rotary(q, k, state["pos"], state["plan"])
            else:
                ang = state["pos"].double()[..., state["axis"]] * state["inv"]
                cos, sin = ang.cos().float(), ang.sin().float()
                qr, kr = _rotate_plain(q, cos, sin, c["interleaved"]), _rotate_plain(k, cos, sin, c["interleaved"])
        if not c["train"]:
            return qr, kr
        gq, gk = torch.autograd.grad((qr, kr), (q, k), (state["gq"], state["gk"]))
        return qr, kr, gq, gk
    if c["op"] == "attention":
        with torch.set_grad_enabled(c["train"]):
            if own:
                from transfusion_amd import attention_ops
                out = attention_ops.score_attention(state["q"], state["k"], state["v"], scale=state["scale"], softcap=c["cap"],
                                                    slopes=state["slopes"], causal=c["mask"] != "full", prefix=state["prefix"],
                                                    q_doc=state["q_doc"], k_doc=state["k_doc"])
            else:
                out = _attention_plain(state)
        if not c["train"]:
            return (out,)
        wrt = [state[n] for n in ("q", "k", "v", "slopes") if state[n] is not None]
        return (out,) + torch.autograd.grad(out, wrt, state["go"])
    params = state["params"]
    if own:
        from transfusion_amd import optim
        total = optim.clip_grad_norm_(params, c["max_norm"], norm_type=math.inf if c["norm"] == "inf" else 2.0)
    else:
        total = _clip_plain(params, c["max_norm"], c["norm"])
    return (total,) + tuple(state["flat"])


# ---------------------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "rotary":
        rot = 2 * (case["nt"] + case["nh"] + case["nw"])
        rows = case["B"] * case["S"]
        passes = 2 if case["train"] else 1
        n = rows * (case["H"] + case["Hk"])
        return {"bytes": passes * 2 * n * case["D"] * _SIZE[case["dtype"]] + rows * 12, "flops": passes * n * rot * 3}
    if case["op"] == "attention":
        B, Sq, Sk, H, Hk, D = (case[k] for k in ("B", "Sq", "Sk", "H", "Hk", "D"))
        pairs = _visible_pairs(case) * H
        e = _SIZE[case["dtype"]]
        qo, kv = B * Sq * H * D * e, B * Sk * Hk * D * e
        nbytes = 2 * qo + 2 * kv
        if case["train"]:                        # backward: dO and dQ, dK, dV
            nbytes += 2 * qo + 2 * kv
        return {"bytes": nbytes + (4 * B * (Sq + Sk) if _has_docs(case) else 0), "flops": (14 if case["train"] else 4) * D * pairs}
    n = b = 0
    for shape in _clip_shapes(case):
        k = math.prod(shape)
        n += k
        b += k * (2 if _clip_dtype(case, shape) == torch.bfloat16 else 4)
    return {"bytes": 3 * b if case["max_norm"] < 1e3 else b, "flops": 3 * n}


# ---------------------------------------------------------------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------------------------------------------------------------
def _exact_rotate(x, theta, interleaved, inverse):
    """Complex multiplication of the channel pairs by exp(+-i theta)."""
    P = theta.shape[-1]
    z = x.detach().double()
    pairs = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if interleaved else (slice(0, P), slice(P, 2 * P))
    w = torch.complex(z[..., pairs[0]], z[..., pairs[1]]) * torch.polar(torch.ones_like(theta), -theta if inverse else theta)[:, :, None, :]
    y = z.clone()
    y[..., pairs[0]], y[..., pairs[1]] = w.real, w.imag
    return y


def _exact_attention(case, st):
    """Head by head, with the gradients of the definition written out."""
    B, Sq, Sk, H, Hk, D = (case[k] for k in ("B", "Sq", "Sk", "H", "Hk", "D"))
    f = lambda t: t.detach().double()
    cap, scale, train = case["cap"], st["scale"], case["train"]
    out = torch.zeros(B, Sq, H, D, dtype=torch.float64, device="cuda:0")
    dq, dk, dv = torch.zeros_like(out), *(torch.zeros(B, Sk, Hk, D, dtype=torch.float64, device="cuda:0") for _ in range(2))
    dslope = torch.zeros(H, dtype=torch.float64, device="cuda:0")
    row = torch.arange(Sq, device="cuda:0")[:, None] + (Sk - Sq)
    col = torch.arange(Sk, device="cuda:0")[None, :]
    dist = (row - col).abs().double()
    for b in range(B):
        hidden = torch.zeros(Sq, Sk, dtype=torch.bool, device="cuda:0")
        if case["mask"] != "full":
            hidden |= col > row
            if st["prefix"] is not None:
                hidden &= col >= int(st["prefix"][b])
        if st["k_doc"] is not None:
            hidden |= (st["q_doc"][b][:, None] != st["k_doc"][b][None, :]) | (st["k_doc"][b] < 0)[None, :]
        for h in range(H):
            g = h // (H // Hk)
            qh, kh, vh = f(st["q"][b, :, h]), f(st["k"][b, :, g]), f(st["v"][b, :, g])
            t = qh @ kh.T * scale
            th = torch.tanh(t / cap) if cap > 0 else None
            if cap > 0:
                t = cap * th
            if st["slopes"] is not None:
                t = t - f(st["slopes"])[h] * dist
            t[hidden] = -math.inf
            top = t.max(dim=1, keepdim=True).values.clamp_min(-1e300)
            w = torch.exp(t - top)
            z = w.sum(dim=1, keepdim=True)
            w /= torch.where(z > 0, z, torch.ones_like(z))
            o = w @ vh
            out[b, :, h] = o
            if not train:
                continue
            go = f(st["go"][b, :, h])
            dv[b, :, g] += w.T @ go
            ds = w * (go @ vh.T - (go * o).sum(dim=1, keepdim=True))
            dslope[h] -= (ds * dist).sum()
            if cap > 0:
                ds *= 1 - th * th
            dq[b, :, h] = ds @ kh * scale
            dk[b, :, g] += ds.T @ qh * scale
    if not train:
        return (out,)
    return (out, dq, dk, dv) + ((dslope,) if st["slopes"] is not None else ())


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rotary":
        axes = (case["nt"], case["nh"], case["nw"])
        theta = torch.cat([st["pos"][..., a:a + 1].double() * torch.tensor([10000.0 ** (-i / n) for i in range(n)], dtype=torch.float64,
                                                                            device="cuda:0") for a, n in enumerate(axes)], dim=-1)
        outs = [_exact_rotate(st["q"], theta, case["interleaved"], False), _exact_rotate(st["k"], theta, case["interleaved"], False)]
        if case["train"]:
            outs += [_exact_rotate(st["gq"], theta, case["interleaved"], True), _exact_rotate(st["gk"], theta, case["interleaved"], True)]
        return tuple(outs)
    if case["op"] == "attention":
        return _exact_attention(case, st)
    grads = [f.double() for f in st["flat"]]
    if case["norm"] == "inf":
        total = max(float(g.abs().max()) for g in grads)
    else:
        total = math.sqrt(sum(float(torch.dot(g.flatten(), g.flatten())) for g in grads))
    coef = min(1.0, case["max_norm"] / (total + 1e-6))
    return (torch.tensor(total, dtype=torch.float64, device="cuda:0"),) + tuple(g * coef for g in grads)
