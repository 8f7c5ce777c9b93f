"""Rotary positions with several axes, attention with changed scores, norm and clip over many tensors: the HIP kernels through the public
entry points against 64-bit references with derived bounds (tests/operator_refs.py)."""
import math

import pytest
import torch

from operator_refs import HALF, attention_ref, check, rotary_ref, visible

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    from transfusion_amd import _lib
    _lib.load()
    return torch.device("cuda:0")


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------------------------------------------
# rotary
# ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,S,H,Hk,D,axes,inter,shared,kind,start", [
    (1, 1, 1, 1, 8, (4,), False, False, torch.int32, 0),                  # one token, one axis, nothing passes through
    (4, 1, 16, 4, 128, (16, 24, 24), False, False, torch.int32, 262144),  # single tokens far out
    (2, 77, 4, 2, 192, (32, 32, 32), False, True, torch.int64, 3),
    (3, 37, 6, 2, 88, (9, 13, 13), True, False, torch.float32, 0),        # a pair count that no vector divides
    (3, 37, 6, 2, 88, (9, 13, 13), False, False, torch.int32, 1 << 20),
    (2, 19, 3, 3, 72, (0, 20, 12), False, False, torch.int32, 5),         # an axis without pairs, channels behind the pairs
    (2, 5, 14, 2, 22, (3, 4, 4), False, False, torch.int32, 1000),        # head width that no vector divides
    (1, 9, 2, 1, 22, (11,), True, True, torch.int64, 1 << 33),            # positions beyond 32 bits
    (2, 300, 4, 4, 256, (40, 44, 44), True, False, torch.int32, 17),
])
def test_rotary(dev, guard, dtype, B, S, H, Hk, D, axes, inter, shared, kind, start):
    from transfusion_amd import attention_ops as A
    g = gen(S * D + B)
    q, k = (guard(torch.randn(B, S, h, D, generator=g).to(dtype)).requires_grad_(True) for h in (H, Hk))
    pos = torch.randint(0, 50, (B, S, len(axes)), generator=g)
    pos = (pos.double() + 0.25 * torch.randint(0, 4, pos.shape, generator=g)).float() if kind == torch.float32 else (pos + start).to(kind)
    plan = A.RotaryPlan(D, axes, interleaved=inter, shared=shared, device=dev)
    pd = guard(pos)
    qr, kr = A.rotary(q, k, pd, plan)
    assert qr.is_contiguous() and kr.is_contiguous() and qr.dtype == dtype
    check("q", qr, rotary_ref(q, pos, axes, interleaved=inter, shared=shared))
    check("k", kr, rotary_ref(k, pos, axes, interleaved=inter, shared=shared))
    gq, gk = (guard(torch.randn(t.shape, generator=g).to(dtype)) for t in (q, k))
    dq, dk = torch.autograd.grad((qr, kr), (q, k), (gq, gk))
    check("dq", dq, rotary_ref(gq, pos, axes, interleaved=inter, shared=shared, inverse=True))
    check("dk", dk, rotary_ref(gk, pos, axes, interleaved=inter, shared=shared, inverse=True))
    # without keys, positions shared by the samples, no graph: the same rows
    with torch.no_grad():
        alone = A.rotary(q, None, guard(pos[0].contiguous()), plan)
    assert torch.equal(alone[0], qr[0].detach())


def test_rotary_views_and_partial_gradients(dev):
    """Thirds of a packed projection, transposed heads, a broadcast sample, rows off 16 bytes; only one of q / k with a gradient."""
    from transfusion_amd import attention_ops as A
    g = gen(5)
    plan = A.RotaryPlan(64, (8, 12, 12), device=dev)
    pos = torch.randint(0, 99, (31, 3), generator=g, dtype=torch.int32)
    pd = pos.to(dev)
    base = torch.randn(2, 31, 12, 64, generator=g).to(BF).to(dev)
    views = {"packed": base[:, :, 4:8], "heads first": base.transpose(1, 2).contiguous().transpose(1, 2)[:, :, :4],
             "broadcast": base[:1, :, :4].expand(2, -1, -1, -1), "shifted": torch.randn(2 * 31 * 4 * 64 + 1, device=dev).to(BF)[1:].view(2, 31, 4, 64),
             "channels apart": base[:, :, :4].transpose(2, 3).contiguous().transpose(2, 3)}
    for name, x in views.items():
        check(name, A.rotary(x, None, pd, plan), rotary_ref(x, pos, (8, 12, 12)))
    q, k = base[:, :, :4].clone().requires_grad_(True), base[:, :, 4:6].clone()
    qr, kr = A.rotary(q, k, pd, plan)
    (dq,) = torch.autograd.grad((qr.float() * 2).sum() + kr.float().sum(), q)
    check("dq", dq, rotary_ref(torch.full(q.shape, 2.0, dtype=BF), pos, (8, 12, 12), inverse=True))
    k.requires_grad_(True)
    qr, kr = A.rotary(q, k, pd, plan)
    (dk,) = torch.autograd.grad(kr, k, torch.ones_like(kr))
    check("dk", dk, rotary_ref(torch.ones(k.shape, dtype=BF), pos, (8, 12, 12), inverse=True))


def test_rotary_gradient_against_differences(dev):
    """Directional derivative of the 64-bit formula by central differences (the map is linear: exact up to rounding)."""
    from transfusion_amd import attention_ops as A
    g = gen(6)
    axes, eps = (5, 3), 1e-3
    q = torch.randn(2, 7, 2, 24, generator=g)
    pos = torch.randint(0, 999, (2, 7, 2), generator=g, dtype=torch.int32)
    go, u = torch.randn(q.shape, generator=g), torch.randn(q.shape, generator=g)
    qd = q.to(dev).requires_grad_(True)
    (dq,) = torch.autograd.grad(A.rotary(qd, None, pos.to(dev), A.RotaryPlan(24, axes, device=dev)), qd, go.to(dev))
    f = lambda x: (rotary_ref(x, pos, axes)[0] * go.double()).sum()
    # (q in 64 bits: rotary_ref's bound is for fp32, its value is what is used here)
    HALF[torch.float64] = 0.0
    diff = (f(q.double() + eps * u.double()) - f(q.double() - eps * u.double())) / (2 * eps)
    bound = (rotary_ref(go, pos, axes, inverse=True)[1] * u.double().abs()).sum()
    assert abs((dq.double().cpu() * u.double()).sum() - diff) <= bound + 1e-9 * abs(diff)


def test_rotary_sizes_of_nothing(dev):
    from transfusion_amd import attention_ops as A
    plan = A.RotaryPlan(16, (8,), device=dev)
    for B, S, H, Hk in ((0, 3, 2, 1), (2, 0, 2, 1), (2, 3, 0, 1)):
        q = torch.empty(B, S, H, 16, device=dev, requires_grad=True)
        k = torch.empty(B, S, Hk, 16, device=dev).normal_().requires_grad_(True)
        qr, kr = A.rotary(q, k, torch.zeros(S, 1, dtype=torch.int32, device=dev), plan)
        assert qr.shape == q.shape and torch.equal(kr, k)
        torch.autograd.grad((qr.sum() + kr.sum()), (q, k))


# ------------------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------------------
CASES = {
    # name: (B, Sq, Sk, H, Hk, D, options)
    "one key": (1, 1, 1, 1, 1, 8, {}),
    "one query": (2, 1, 77, 4, 4, 64, {"causal": 1, "slopes": 1}),
    "plain": (2, 130, 130, 2, 2, 64, {}),
    "causal": (2, 130, 130, 4, 2, 64, {"causal": 1}),
    "causal cap": (1, 257, 257, 3, 1, 40, {"causal": 1, "cap": 2.0}),
    "prefix pad": (3, 97, 97, 4, 4, 192, {"causal": 1, "prefix": 1, "pad": 1, "cap": 5.0}),
    "documents": (2, 321, 321, 4, 2, 96, {"causal": 1, "docs": 5, "slopes": 1}),
    "documents all ways": (1, 200, 200, 2, 1, 32, {"docs": 4, "cap": 3.0}),
    "scattered documents": (2, 150, 150, 2, 2, 24, {"docs": -3}),
    "slopes both sides": (2, 66, 130, 4, 4, 16, {"slopes": 1}),
    "more keys": (2, 33, 417, 6, 3, 88, {"causal": 1, "prefix": 1, "slopes": 1, "pad": 1}),
    "more queries": (2, 150, 40, 2, 2, 72, {"causal": 1}),               # the first 110 rows see nothing
    "wide": (1, 140, 140, 2, 1, 256, {"causal": 1, "cap": 4.0, "slopes": 1}),
    "wide 224": (2, 65, 65, 2, 2, 224, {"prefix": 1, "causal": 1}),
    "starts": (3, 5, 300, 4, 2, 128, {"causal": 1, "start": 1, "slopes": 1}),
    "tile edges": (1, 128, 128, 2, 2, 128, {"causal": 1}),
    "tile edges plus": (1, 129, 193, 2, 2, 128, {"causal": 1, "docs": 3}),
    "far slopes": (1, 64, 1100, 2, 2, 64, {"causal": 1, "slopes": 30}),  # steep: far keys vanish
    "long split": (1, 3, 1500, 8, 2, 64, {"causal": 1, "cap": 10.0}),
    "group rows": (2, 7, 513, 14, 2, 64, {"causal": 1, "slopes": 1, "pad": 1}),
    "token documents": (3, 1, 700, 6, 2, 40, {"docs": -3, "slopes": 1}),
    "token behind padding": (3, 2, 900, 8, 1, 192, {"causal": 1, "pad": 1, "cap": 6.0}),
    "token wide": (2, 1, 333, 4, 4, 256, {"causal": 1, "slopes": 1}),
    "token wide padding": (2, 3, 260, 4, 2, 256, {"causal": 1, "pad": 1}),
    "token caches": (4, 1, 1000, 8, 2, 96, {"causal": 1, "start": 1, "prefix": 1}),
    "32 rows": (2, 4, 222, 8, 1, 128, {"causal": 1}),
    "33 rows": (2, 33, 222, 1, 1, 32, {"causal": 1}),
    "cap tiny": (1, 70, 70, 2, 1, 64, {"cap": 1e-10, "causal": 1}),
    "cap huge": (1, 70, 70, 2, 1, 64, {"cap": 1e10, "causal": 1}),
    "sets of eight": (8, 150, 150, 2, 1, 32, {"causal": 1}),             # every way in which causal blocks are dealt
    "eight heads": (2, 150, 150, 4, 2, 32, {"causal": 1, "pad": 1}),
    "eight parts": (1, 700, 700, 2, 2, 24, {"causal": 1}),
    "odd halves": (1, 353, 290, 2, 1, 64, {"causal": 1, "slopes": 1}),   # parts of a loop that begin inside a tile
    "odd halves documents": (1, 419, 419, 2, 2, 192, {"causal": 1, "docs": 3, "pad": 1}),
    "odd halves wide": (1, 290, 353, 3, 3, 128, {"docs": 2, "pad": 1}),
    "many rows": (3, 500, 500, 2, 1, 16, {"causal": 1, "slopes": 1}),    # more rows than one workgroup adds up
    "documents of one": (2, 70, 70, 2, 1, 64, {"docs": 70, "causal": 1}),
    "few rows split": (1, 40, 2100, 2, 1, 64, {"causal": 1, "slopes": 1, "pad": 1}),
}


def make(name, dtype, place=lambda t: t):
    B, Sq, Sk, H, Hk, D, o = CASES[name]
    g = gen(sum(map(ord, name)))
    q, k, v = (place(torch.randn(B, s, h, D, generator=g).to(dtype)) for s, h in ((Sq, H), (Sk, Hk), (Sk, Hk)))
    opt = {"causal": bool(o.get("causal"))}
    if "cap" in o:
        opt["softcap"] = o["cap"]
    if "slopes" in o:
        opt["slopes"] = place(o["slopes"] * torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)]))
    if "prefix" in o:
        opt["prefix"] = place(torch.tensor([(Sk // 3 + 11 * b) % (Sk + 5) for b in range(B)], dtype=torch.int32))
    if "start" in o:
        opt["q_start"] = place(torch.tensor([(0, 40, 296, -2)[b % 4] for b in range(B)], dtype=torch.int32))
    if "docs" in o or "pad" in o:
        n = o.get("docs", 1)
        doc = torch.randint(-1, -n, (B, Sk), generator=g) if n < 0 else (torch.arange(Sk) * n // Sk).expand(B, Sk).clone()
        if "pad" in o:
            for b in range(B):
                cut = Sk - 1 - (b * 29) % (Sk // 2)
                if Sq == Sk:
                    doc[b, cut:] = -1
                else:
                    doc[b, :Sk - cut] = -1
        doc = doc.to(torch.int32)
        opt["k_doc"] = place(doc)
        opt["q_doc"] = place(doc[:, Sk - Sq:].contiguous())
    go = place(torch.randn(B, Sq, H, D, generator=g).to(dtype))
    return q, k, v, go, opt


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("name", list(CASES))
def test_attention(dev, guard, name, dtype):
    from transfusion_amd import attention_ops as A
    q, k, v, go, opt = make(name, dtype, guard)
    want = attention_ref(q, k, v, go, **opt)
    with torch.no_grad():
        check("inference", A.score_attention(q, k, v, **opt), want["out"])
    leaves = {"dq": q.requires_grad_(True), "dk": k.requires_grad_(True), "dv": v.requires_grad_(True)}
    if "slopes" in opt:
        leaves["dslopes"] = opt["slopes"].requires_grad_(True)
    out = A.score_attention(q, k, v, **opt)
    check("out", out, want["out"])
    for n, gr in zip(leaves, torch.autograd.grad(out, list(leaves.values()), go)):
        check(n, gr, want[n])


@pytest.mark.parametrize("name", [n for n, c in CASES.items() if "slopes" in c[6]])
def test_attention_slopes_gradient_of_bf16_is_exact_to_fp32(dev, name):
    """It is an fp32 tensor: no rounding of P, dS or the output to bf16 may reach it, so it has to keep the bounds that the same inputs held in
    fp32 have."""
    from transfusion_amd import attention_ops as A
    q, k, v, go, opt = make(name, BF, lambda t: t.to(dev))
    want = attention_ref(q.float(), k.float(), v.float(), go.float(), **opt)
    out = A.score_attention(q, k, v, **{**opt, "slopes": opt["slopes"].requires_grad_(True)})
    check("dslopes", torch.autograd.grad(out, opt["slopes"], go)[0], want["dslopes"])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("S,H,Hk,D,cap", [(1, 2, 1, 64, 0.0), (70, 2, 1, 64, 0.0), (130, 4, 4, 192, 5.0), (200, 3, 1, 128, 0.0), (90, 2, 2, 256, 3.0), (40, 2, 1, 24, 0.0)])
def test_rows_that_see_one_key_have_no_gradient_behind_the_softmax(dev, dtype, S, H, Hk, D, cap):
    """P = 1 whatever the score is: the output is the value itself and dq, dk and dslopes are 0, not what rounding leaves of dP - delta."""
    from transfusion_amd import attention_ops as A
    g = gen(S + D)
    q, k, v, go = (torch.randn(2, S, h, D, generator=g).to(dtype).to(dev).requires_grad_(True) for h in (H, Hk, Hk, H))
    sl = torch.ones(H, device=dev, requires_grad=True)
    doc = torch.arange(S, dtype=torch.int32, device=dev).expand(2, -1).contiguous()
    out = A.score_attention(q, k, v, softcap=cap, slopes=sl, causal=True, q_doc=doc, k_doc=doc)
    assert torch.equal(out, v.repeat_interleave(H // Hk, dim=2))
    dq, dk, dsl = torch.autograd.grad(out, (q, k, sl), go.detach())
    assert not dq.any() and not dk.any() and not dsl.any()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_reads_views(dev, dtype):
    """A packed projection's thirds, heads before tokens, broadcast keys (their gradient is summed by autograd), rows off 16 bytes."""
    from transfusion_amd import attention_ops as A
    g = gen(11)
    S, D = 90, 48
    packed = torch.randn(2, S, 8, D, generator=g).to(dtype).to(dev).requires_grad_(True)
    go = torch.randn(2, S, 4, D, generator=g).to(dtype).to(dev)
    want = attention_ref(packed[:, :, :4], packed[:, :, 4:6], packed[:, :, 6:], go, causal=True)
    out = A.score_attention(packed[:, :, :4], packed[:, :, 4:6], packed[:, :, 6:], causal=True)
    check("packed", out, want["out"])
    (gp,) = torch.autograd.grad(out, packed, go)
    for n, sl in (("dq", slice(0, 4)), ("dk", slice(4, 6)), ("dv", slice(6, 8))):
        check(n, gp[:, :, sl], want[n])
    hf = packed.detach().transpose(1, 2).contiguous().transpose(1, 2)
    check("heads first", A.score_attention(hf[:, :, :4], hf[:, :, 4:6], hf[:, :, 6:], causal=True), want["out"])
    off = torch.empty(packed.numel() + 1, dtype=dtype, device=dev)[1:].view(packed.shape).copy_(packed.detach())
    check("off 16 bytes", A.score_attention(off[:, :, :4], off[:, :, 4:6], off[:, :, 6:], causal=True), want["out"])
    kb = packed.detach()[:1, :, 4:6].clone().requires_grad_(True)
    vb = packed.detach()[:1, :, 6:].clone().requires_grad_(True)
    want = attention_ref(packed[:, :, :4], kb.expand(2, -1, -1, -1), vb.expand(2, -1, -1, -1), go)
    out = A.score_attention(packed.detach()[:, :, :4], kb.expand(2, -1, -1, -1), vb.expand(2, -1, -1, -1))
    check("broadcast", out, want["out"])
    dk, dv = torch.autograd.grad(out, (kb, vb), go)
    for n, got in (("dk", dk), ("dv", dv)):
        val, bound = want[n]
        # autograd adds the two samples in the tensors' type: one more rounding of the sum
        check(n, got, (val.sum(0, keepdim=True), bound.sum(0, keepdim=True) * 1.01 + val.sum(0, keepdim=True).abs() * HALF[dtype]))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_never_uses_hidden_rows(dev, dtype):
    """NaN and infinity in padded rows of every operand, and in the rows of a cache beyond its last written token."""
    from transfusion_amd import attention_ops as A
    q, k, v, go, opt = make("prefix pad", dtype, lambda t: t.to(dev))
    want = attention_ref(q, k, v, go, **opt)
    dead = opt["k_doc"] < 0
    for t, val in ((q, math.nan), (k, math.nan), (v, math.inf), (go, math.nan)):
        t[dead] = val
    out = A.score_attention(q.requires_grad_(True), k.requires_grad_(True), v.requires_grad_(True), **opt)
    check("out", out, want["out"])
    for n, gr in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), go)):
        check(n, gr, want[n])
        if n == "dq":
            assert (gr[dead] == 0).all()
    q, k, v, go, opt = make("starts", dtype, lambda t: t.to(dev))
    want = attention_ref(q, k, v, go, **opt)
    for b, s in enumerate(opt["q_start"].tolist()):
        k[b, max(0, s + q.shape[1]):], v[b, max(0, s + q.shape[1]):] = math.nan, math.inf
    out = A.score_attention(q.requires_grad_(True), k.requires_grad_(True), v.requires_grad_(True), **opt)
    check("cache", out, want["out"])
    for n, gr in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), go)):
        check(n, gr, want[n])


def test_attention_propagates_what_is_visible(dev):
    """A NaN in a visible key reaches the rows that see it and no row of another sample."""
    from transfusion_amd import attention_ops as A
    q, k, v, go, opt = make("causal", BF, lambda t: t.to(dev))
    ref = A.score_attention(q, k, v, **opt)
    k[0, 100] = math.nan
    out = A.score_attention(q, k, v, **opt)
    assert torch.isnan(out[0, 100:]).all() and torch.equal(out[1], ref[1]) and torch.equal(out[0, :64], ref[0, :64])


def test_attention_sizes_of_nothing(dev):
    from transfusion_amd import attention_ops as A
    for B, Sq, Sk in ((0, 4, 4), (2, 0, 5), (2, 5, 0)):
        q = torch.randn(B, Sq, 4, 16, device=dev, requires_grad=True)
        k = torch.randn(B, Sk, 2, 16, device=dev, requires_grad=True)
        v = torch.randn(B, Sk, 2, 16, device=dev, requires_grad=True)
        sl = torch.ones(4, device=dev, requires_grad=True)
        out = A.score_attention(q, k, v, slopes=sl, causal=True)
        assert out.shape == q.shape and (out == 0).all()
        for t, gr in zip((q, k, v, sl), torch.autograd.grad(out, (q, k, v, sl), torch.ones_like(out))):
            assert gr.shape == t.shape and (gr == 0).all()


def test_attention_gradient_against_differences(dev):
    """Central differences of the 64-bit formula along random directions; truncation ~ eps^2 times a third derivative of order 10."""
    from transfusion_amd import attention_ops as A
    HALF[torch.float64] = 0.0
    q, k, v, go, opt = make("causal cap", F32)
    opt["slopes"] = torch.tensor([0.3, 0.01, -0.05])
    want = attention_ref(q, k, v, go, **opt)
    dv_ = lambda t: t.to(dev).requires_grad_(True)
    ins = {"dq": dv_(q), "dk": dv_(k), "dv": dv_(v), "dslopes": dv_(opt["slopes"])}
    o2 = dict(opt, slopes=ins["dslopes"])
    grads = dict(zip(ins, torch.autograd.grad(A.score_attention(ins["dq"], ins["dk"], ins["dv"], **o2), list(ins.values()), go.to(dev))))
    host = {"dq": q.double(), "dk": k.double(), "dv": v.double(), "dslopes": opt["slopes"].double()}
    f = lambda h: (attention_ref(h["dq"], h["dk"], h["dv"], **dict(opt, slopes=h["dslopes"]))["out"][0] * go.double()).sum()
    eps = 1e-4
    for n in ins:
        u = torch.randn(host[n].shape, generator=gen(3)).double()
        diff = (f({**host, n: host[n] + eps * u}) - f({**host, n: host[n] - eps * u})) / (2 * eps)
        bound = (want[n][1] * u.abs()).sum()
        assert abs((grads[n].double().cpu() * u).sum() - diff) <= bound + 1e-6 * (1 + abs(diff)), n


def test_attention_offsets_beyond_32_bits(dev):
    """A cache whose rows lie 64 KiB apart: the last keys start beyond 4 GiB."""
    from transfusion_amd import attention_ops as A
    Sk, D, row = 70000, 64, 32768
    buf = torch.empty(Sk * row, dtype=BF, device=dev).view(1, Sk, row)
    k, v = buf[:, :, :2 * D].view(1, Sk, 2, D), buf[:, :, 1024:1024 + 2 * D].view(1, Sk, 2, D)
    g = gen(4)
    k.copy_(torch.randn(1, Sk, 2, D, generator=g))
    v.copy_(torch.randn(1, Sk, 2, D, generator=g))
    for Sq in (1, 130):
        q = torch.randn(1, Sq, 4, D, generator=g).to(BF).to(dev)
        check(f"Sq {Sq}", A.score_attention(q, k, v, causal=True), attention_ref(q, k, v, causal=True)["out"])
    del buf, k, v
    torch.cuda.empty_cache()


def test_attention_is_deterministic_and_stream_safe(dev):
    from transfusion_amd import attention_ops as A
    q, k, v, go, opt = make("group rows", BF, lambda t: t.to(dev))

    def both():
        a, b, c = (t.detach().requires_grad_(True) for t in (q, k, v))
        out = A.score_attention(a, b, c, **opt)
        return [out.detach()] + list(torch.autograd.grad(out, (a, b, c), go))
    ref = both()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for st in streams:
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(both())
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
        for gs in got:
            for x, y in zip(ref, gs):
                assert torch.equal(x, y)


# ------------------------------------------------------------------------------------------------------
# norm and clip
# ------------------------------------------------------------------------------------------------------
def clip_ref(grads, max_norm, norm_type):
    gs = [g.detach().double().cpu() for g in grads]
    total = max([float(g.abs().max()) for g in gs if g.numel()] or [0.0]) if norm_type == math.inf else math.sqrt(sum(float((g * g).sum()) for g in gs))
    return total, min(1.0, max_norm / (total + 1e-6)), gs


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("case", ["one", "few", "mixed", "hundreds", "large", "no clip"])
def test_clip(dev, guard, case, norm_type):
    """Total: 64-bit sums, rounded once to fp32 (+ the root's).  Gradients: the coefficient carries the norm's, the sum's and the
    quotient's rounding (4 half steps of fp32), the product one more, then the type's own."""
    from transfusion_amd import optim
    g = gen(len(case))
    sizes = {"one": [1], "few": [5, 0, 64, 3, 1000], "mixed": [7, 4096, 33, 20000, 1], "hundreds": [1 + (i * 37) % 500 for i in range(431)],
             "large": [3000001, 17, 40000], "no clip": [100, 200]}[case]
    dts = [F32 if case in ("one", "hundreds") or i % 2 else BF for i in range(len(sizes))]
    place = guard if case != "hundreds" else (lambda t: t.to(dev))
    params = []
    for n, dt in zip(sizes, dts):
        p = torch.zeros(n, dtype=dt, device=dev, requires_grad=True)
        p.grad = place(torch.randn(n, generator=g).to(dt))
        params.append(p)
    max_norm = 1e9 if case == "no clip" else 0.7
    total, coef, gs = clip_ref([p.grad for p in params], max_norm, norm_type)
    before = [p.grad.clone() for p in params]
    versions = [p.grad._version for p in params]
    measured = optim.clip_grad_norm_(params, math.inf, norm_type=norm_type)
    assert all(torch.equal(p.grad, b) for p, b in zip(params, before))
    got = optim.clip_grad_norm_(params, max_norm, norm_type=norm_type)
    assert got.shape == () and got.dtype == F32 and torch.equal(got, measured)
    assert abs(float(got) - total) <= 2 * 2.0 ** -24 * total
    for p, w, b, ver in zip(params, gs, before, versions):
        if coef == 1.0:
            assert torch.equal(p.grad, b)
        check("grad", p.grad, (w * coef, (w * coef).abs() * (6 * 2.0 ** -24 + HALF[p.grad.dtype] * (1 + 2.0 ** -20)) + 1e-38))
        assert p.grad._version > ver


def test_clip_order_of_axes_unaligned_slices_and_repeats(dev):
    from transfusion_amd import optim
    flat = torch.randn(1000, device=dev)
    half = torch.randn(1001, device=dev).to(BF)
    ps = []
    for gr in (flat[1:1 + 35].view(5, 7), flat[36:36 + 3], flat[100:100 + 600].view(20, 30).t(), half[1:400], half[400:401],
               torch.randn(2, 3, 4, 5, device=dev).to(memory_format=torch.channels_last)):
        p = torch.zeros(gr.shape, dtype=gr.dtype, device=dev, requires_grad=True)
        p.grad = gr
        ps.append(p)
    none = torch.zeros(3, device=dev, requires_grad=True)
    keep_f, keep_h = flat.clone(), half.clone()
    total, coef, gs = clip_ref([p.grad for p in ps], 1.0, 2.0)
    got = optim.clip_grad_norm_(ps + [none, ps[0], ps[2]], 1.0)                 # repeated parameters count and scale once
    assert abs(float(got) - total) <= 2 * 2.0 ** -24 * total
    for p, w in zip(ps, gs):
        check("grad", p.grad, (w * coef, (w * coef).abs() * (6 * 2.0 ** -24 + HALF[p.grad.dtype] * (1 + 2.0 ** -20)) + 1e-38))
    for t, old, used in ((flat, keep_f, ((1, 39), (100, 700))), (half, keep_h, ((1, 401),))):      # what lies between the slices stays
        mask = torch.ones_like(t, dtype=torch.bool)
        for a, b in used:
            mask[a:b] = False
        assert torch.equal(t[mask], old[mask])


def test_clip_not_finite(dev):
    """As torch: infinite norm -> finite gradients go to zero, infinite ones to NaN; a NaN spreads; squares beyond fp32 do not overflow."""
    from transfusion_amd import optim

    def run(vals, norm_type=2.0):
        p = torch.zeros(len(vals), device=dev, requires_grad=True)
        p.grad = torch.tensor(vals, device=dev)
        return optim.clip_grad_norm_([p], 1.0, norm_type=norm_type), p.grad
    for nt in (2.0, math.inf):
        n, g = run([1.0, math.inf], nt)
        assert math.isinf(float(n)) and float(g[0]) == 0.0 and math.isnan(float(g[1]))
        n, g = run([1.0, math.nan, math.inf], nt)
        assert math.isnan(float(n)) and torch.isnan(g).all()
    n, g = run([3e30, 4e30])
    assert abs(float(n) - 5e30) < 1e24 and abs(float(g[0]) - 0.6) < 1e-6


def test_clip_nothing(dev):
    from transfusion_amd import optim
    assert float(optim.clip_grad_norm_([], 1.0)) == 0.0
    p = torch.zeros(0, device=dev, requires_grad=True)
    p.grad = torch.zeros(0, device=dev)
    assert float(optim.clip_grad_norm_(p, 1.0)) == 0.0


# ------------------------------------------------------------------------------------------------------
# graphs, and a step of the three together
# ------------------------------------------------------------------------------------------------------
def test_captured_and_replayed(dev):
    """Forward, backward and clip captured once, replayed with new inputs between eager work: every replay has the eager bits."""
    from transfusion_amd import attention_ops as A, optim
    plan = A.RotaryPlan(64, (8, 12, 12), device=dev)
    static = {n: torch.zeros(2, 200, h, 64, dtype=BF, device=dev) for n, h in (("q", 4), ("k", 2), ("v", 2), ("go", 4))}
    pos = torch.zeros(2, 200, 3, dtype=torch.int32, device=dev)
    doc = torch.zeros(2, 200, dtype=torch.int32, device=dev)
    tail = static["q"][:, -1:].clone()

    def step():
        q, k, v = (static[n].detach().requires_grad_(True) for n in ("q", "k", "v"))
        qr, kr = A.rotary(q, k, pos, plan)
        out = A.score_attention(qr, kr, v, causal=True, softcap=20.0, q_doc=doc, k_doc=doc)
        for t, gr in zip((q, k, v), torch.autograd.grad(out, (q, k, v), static["go"])):
            t.grad = gr
        norm = optim.clip_grad_norm_([q, k, v], 0.5)
        with torch.no_grad():
            one = A.score_attention(tail, kr, v, causal=True)
        return [out.detach(), q.grad, k.grad, v.grad, norm, one]

    def fill(seed):
        g = gen(seed)
        for t in static.values():
            t.copy_(torch.randn(t.shape, generator=g))
        tail.copy_(torch.randn(tail.shape, generator=g))
        pos.copy_(torch.randint(0, 500, pos.shape, generator=g))
        doc.copy_((torch.arange(200)[None] * (seed + 2) // 200).expand(2, -1))
    fill(0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(1, 5):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        for x, y in zip(got, step()):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_training_step_of_the_operators(dev, dtype):
    """Projection -> rotary -> attention -> projection, the gradients' norm and clip, and the optimiser, against the same step in 64-bit
    torch on the CPU (weights rounded as the kernels see them).  Tolerances: relative L2 of a chain of five rounded products."""
    from transfusion_amd import attention_ops as A, ops, optim
    B, S, H, Hk, D, d = 2, 70, 4, 2, 32, 128
    g = gen(8)
    axes = (4, 6, 6)
    x = torch.randn(B, S, d, generator=g).to(dtype)
    w1 = (torch.randn((H + 2 * Hk) * D, d, generator=g) / math.sqrt(d)).to(BF).float()
    w2 = (torch.randn(d, H * D, generator=g) / math.sqrt(H * D)).to(BF).float()
    sl = torch.tensor([0.5, 0.25, 0.1, 0.05])
    pos = torch.randint(0, 40, (S, 3), generator=g, dtype=torch.int32)
    doc = (torch.arange(S) * 2 // S).expand(B, S).clone().to(torch.int32)
    doc[1, 60:] = -1
    prefix = torch.tensor([10, 20], dtype=torch.int32)
    go = torch.randn(B, S, d, generator=g)
    go[1, 60:] = 0

    P = [torch.nn.Parameter(t.to(dev)) for t in (w1, w2, sl)]
    prec = "bf16" if dtype == BF else "fp32"
    qkv = ops.linear(x.to(dev), P[0], precision=prec).view(B, S, H + 2 * Hk, D)
    qr, kr = A.rotary(qkv[:, :, :H], qkv[:, :, H:H + Hk], pos.to(dev), A.RotaryPlan(D, axes, device=dev))
    o = A.score_attention(qr, kr, qkv[:, :, H + Hk:], softcap=15.0, slopes=P[2], causal=True, prefix=prefix.to(dev), q_doc=doc.to(dev), k_doc=doc.to(dev))
    y = ops.linear(o.reshape(B, S, H * D), P[1], precision=prec)
    y.float().backward(go.to(dev))
    norm = optim.clip_grad_norm_(P, 1.0)

    R = [t.double().requires_grad_(True) for t in (w1, w2, sl)]
    z = (x.double() @ R[0].T).view(B, S, H + 2 * Hk, D)
    ax = torch.tensor([a for a, n in enumerate(axes) for _ in range(n)])
    th = (pos.double()[:, ax] * torch.tensor([10000.0 ** (-i / n) for n in axes for i in range(n)], dtype=torch.float64))[None, :, None]
    def turn(t):
        a, b = t[..., :16], t[..., 16:]
        return torch.cat((a * th.cos() - b * th.sin(), a * th.sin() + b * th.cos()), -1)
    qh, kh, vh = (t.permute(0, 2, 1, 3) for t in (turn(z[:, :, :H]), turn(z[:, :, H:H + Hk]), z[:, :, H + Hk:]))
    kh, vh = kh.repeat_interleave(2, 1), vh.repeat_interleave(2, 1)
    vis, dist = visible(B, S, S, True, prefix, None, doc, doc)
    s = 15 * torch.tanh(qh @ kh.transpose(-1, -2) / math.sqrt(D) / 15) - R[2][:, None, None] * dist[:, None]
    s = s.masked_fill(~vis[:, None], -1e30)
    a = torch.softmax(s, -1) * vis[:, None].any(-1, keepdim=True)
    yr = (a @ vh).permute(0, 2, 1, 3).reshape(B, S, H * D) @ R[1].T
    yr.backward(go.double())
    tol = 2e-2 if dtype == BF else 2e-4
    rel = lambda u, w: ((u.detach().double().cpu() - w).norm() / w.norm()).item()
    assert rel(y, yr.detach()) < tol
    tn = math.sqrt(sum(float((r.grad ** 2).sum()) for r in R))
    assert abs(float(norm) - tn) < tol * tn
    for p, r in zip(P, R):
        assert rel(p.grad, r.grad * min(1.0, 1.0 / (tn + 1e-6))) < tol, p.shape
    before = [p.detach().clone() for p in P]
    optim.FusedRAdam(P, lr=1e-2).step()
    optim.FusedRAdam(P, lr=1e-2, degenerated_to_sgd=True).step()
    assert all(torch.isfinite(p).all() for p in P) and any(not torch.equal(p, b) for p, b in zip(P, before))


# ------------------------------------------------------------------------------------------------------
# refusals that need device tensors
# ------------------------------------------------------------------------------------------------------
def test_refusals(dev):
    from transfusion_amd import _lib as L, attention_ops as A, optim
    q, k = torch.zeros(2, 5, 4, 16, device=dev), torch.zeros(2, 7, 2, 16, device=dev)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)
    for args, kw in [((q, k, k[:, :6]), {}), ((q, k[:1], k[:1]), {}), ((q[0], k, k), {}), ((q, k.to(BF), k.to(BF)), {}), ((q.half(), k.half(), k.half()), {}),
                     ((q[:, :, :3], k, k), {}), ((q[..., :12], k[..., :12], k[..., :12]), {}), ((q, k.cpu(), k), {}), ((q, k, k), {"softcap": -1.0}),
                     ((q, k, k), {"softcap": math.inf}), ((q, k, k), {"softcap": 1e-11}), ((q, k, k), {"softcap": 1e11}), ((q, k, k), {"scale": 1e11}), ((q, k, k), {"scale": math.nan}), ((q, k, k), {"slopes": torch.zeros(2, device=dev)}),
                     ((q, k, k), {"slopes": torch.zeros(4)}), ((q, k, k), {"slopes": torch.zeros(4, dtype=BF, device=dev)}), ((q, k, k), {"prefix": i(2)}),
                     ((q, k, k), {"causal": True, "prefix": i(3)}), ((q, k, k), {"causal": True, "prefix": torch.zeros(2, dtype=torch.int64, device=dev)}),
                     ((q, k, k), {"causal": True, "q_start": 3}), ((q, k, k), {"q_doc": i(2, 5)}), ((q, k, k), {"q_doc": i(2, 5), "k_doc": i(2, 5)})]:
        with pytest.raises(L.TfError):
            A.score_attention(*args, **kw)
    plan = A.RotaryPlan(16, (4, 4), device=dev)
    p = i(2, 5, 2)
    for args in [(q, k, p, plan), (q, q, i(2, 5, 3), plan), (q, q, i(5), plan), (q, q, p.to(torch.int16), plan), (q, q, p.cpu(), plan), (q, q, p, None),
                 (q[..., :8], None, p, plan), (q.half(), None, p, plan), (q, q.to(BF), p, plan), (q, None, p.float().requires_grad_(True), plan)]:
        with pytest.raises(L.TfError):
            A.rotary(*args)
    for gr in (torch.zeros(3, dtype=torch.float16, device=dev), torch.zeros(6, device=dev)[::2], torch.zeros(1, device=dev).expand(4)):
        t = torch.zeros(gr.shape, dtype=gr.dtype, device=dev, requires_grad=True)
        t.grad = gr
        with pytest.raises(L.TfError):
            optim.clip_grad_norm_([t], 1.0)
    flat = torch.zeros(10, device=dev)
    a, b = (torch.zeros(6, device=dev, requires_grad=True) for _ in range(2))
    a.grad, b.grad = flat[:6], flat[4:]
    with pytest.raises(L.TfError):
        optim.clip_grad_norm_([a, b], 1.0)
