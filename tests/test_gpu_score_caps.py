"""Caps of every accepted size in attention with changed scores: a capped score may be off by a part of ITSELF, whatever the cap is, in every
kernel (few rows, prompt, both backward kernels) and beside scores of any size."""
import pytest
import torch

from operator_refs import check
from score_bounds import attention_bounds

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    from transfusion_amd import _lib
    _lib.load()
    return torch.device("cuda:0")


def inputs(seed, B, Sq, Sk, H, Hk, D, dtype):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(B, s, h, D, generator=g).to(dtype) for s, h in ((Sq, H), (Sk, Hk), (Sk, Hk), (Sq, H))]


def compare(dev, tensors, **opt):
    from transfusion_amd import attention_ops as A
    q, k, v, go = (t.to(dev) for t in tensors)
    want = attention_bounds(q, k, v, go, **opt)
    opt = {n: x.to(dev) if isinstance(x, torch.Tensor) else x for n, x in opt.items()}
    with torch.no_grad():
        check("inference", A.score_attention(q, k, v, **opt), want["out"])
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    out = A.score_attention(q, k, v, **opt)
    check("out", out, want["out"])
    for n, gr in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), go)):
        check(n, gr, want[n])


SHAPES = [(1, 1, 77, 1, 1, 64), (2, 1, 300, 4, 2, 64), (2, 4, 513, 8, 1, 128), (1, 3, 260, 2, 2, 256),       # few rows
          (1, 70, 70, 2, 1, 64), (1, 200, 333, 2, 2, 192)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cap", [1e-10, 1e-3, 1.0, 30.0, 1e3, 1e4, 1e6, 1e8, 1e10])
@pytest.mark.parametrize("shape", SHAPES)
def test_every_cap(dev, shape, cap, dtype):
    compare(dev, inputs(sum(shape), *shape, dtype), softcap=cap, causal=True)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cap", [1e3, 1e6])
@pytest.mark.parametrize("shape", [(1, 4, 128, 2, 1, 64), (1, 96, 96, 2, 2, 64), (1, 160, 160, 2, 1, 128)])
@pytest.mark.parametrize("kind", ["query", "hidden key"])
def test_scores_beside_much_larger_ones(dev, kind, shape, cap, dtype):
    """One query whose scores reach the cap, or a last key that only the last query sees and whose scores do: the other rows of the tile keep
    their own precision."""
    t = inputs(sum(shape) + 1, *shape, dtype)
    if kind == "query":
        t[0][:, 1] *= cap
    else:
        t[1][:, -1] *= cap
    compare(dev, t, softcap=cap, causal=True)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("scale,cap", [(9e5, 1.0), (1e10, 1e5), (1e10, 1e10), (1e10, 1e-10), (-9e5, 1.0), (1e-3, 1e10), (1e-20, 1e10), (0.0, 1.0)])
@pytest.mark.parametrize("shape", [(1, 2, 90, 2, 1, 64), (1, 70, 70, 2, 1, 64)])
def test_scores_of_zero(dev, shape, scale, cap, dtype):
    """A query of zeros attends every key alike, whatever scale and cap make of other scores."""
    t = inputs(sum(shape) + 2, *shape, dtype)
    t[0].zero_()
    compare(dev, t, scale=scale, softcap=cap)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("docs", [False, True])
@pytest.mark.parametrize("slope", [None, 0.0, 0.25, 1e9])
@pytest.mark.parametrize("scale,cap", [(1e4, 0.0), (1e7, 0.0), (1e10, 0.0), (1e4, 1e10), (1e7, 1e10)])
@pytest.mark.parametrize("shape", [(1, 2, 90, 2, 1, 64), (2, 70, 70, 2, 1, 64), (1, 150, 333, 2, 2, 128)])
def test_scores_beyond_all_measure(dev, shape, scale, cap, slope, docs, dtype):
    """Scores far apart: every row takes one value whole, and its gradient is that value's.  Query i is the unit vector of channel i % D, the keys hold
    whole numbers, so that scores are exact up to the scale's (and the cap's) rounding, and the winner is ahead by more than that."""
    from transfusion_amd import attention_ops as A
    q, k, v, go = inputs(sum(shape) + 4, *shape, dtype)
    B, Sq, Sk, H, Hk, D = shape
    q.zero_()
    q[:, torch.arange(Sq), :, torch.arange(Sq) % D] = 1.0
    g = torch.Generator().manual_seed(5)
    k = torch.stack([torch.randperm(Sk, generator=g) for _ in range(B * Hk * D)]).view(B, Hk, D, Sk).permute(0, 3, 1, 2).remainder(256).to(dtype)
    slopes = None if slope is None else torch.full((H,), slope)
    t = torch.einsum("bihd,bjhd->bhij", q.double(), k.double().repeat_interleave(H // Hk, dim=2)) * scale
    t = cap * torch.tanh(t / cap) if cap else t
    p, j = torch.arange(Sk - Sq, Sk), torch.arange(Sk)
    if slope:
        t = t - slope * (p[:, None] - j).abs().double()
    t = t.masked_fill(j > p[:, None], -float("inf"))
    top = t.topk(2, dim=-1)
    sure = (top.values[..., 0] - top.values[..., 1]) > 64 + 2.0 ** -18 * top.values.abs().amax(-1)       # [B, H, Sq]
    assert sure.float().mean() > 0.3
    go = go * sure.permute(0, 2, 1)[..., None]
    best = top.indices[..., 0]
    vh = v.repeat_interleave(H // Hk, dim=2).permute(0, 2, 1, 3)
    want = torch.gather(vh, 2, best[..., None].expand(-1, -1, -1, D))
    dv = torch.zeros(B, H, Sk, D, dtype=torch.float64).scatter_add_(2, best[..., None].expand(-1, -1, -1, D), go.double().permute(0, 2, 1, 3))
    dv = dv.view(B, Hk, H // Hk, Sk, D).sum(2).permute(0, 2, 1, 3)
    leaves = [x.to(dev).requires_grad_(True) for x in (q, k, v)]
    doc = {n: torch.full((B, S), 7, dtype=torch.int32, device=dev) for n, S in (("q_doc", Sq), ("k_doc", Sk))} if docs else {}
    out = A.score_attention(*leaves, scale=scale, softcap=cap, slopes=None if slopes is None else slopes.to(dev), causal=True, **doc)
    got = out.detach().cpu().permute(0, 2, 1, 3)
    assert torch.isfinite(got).all() and torch.equal(got[sure], want[sure])
    dq, dk, dv_ = torch.autograd.grad(out, leaves, go.to(dev))
    assert torch.isfinite(dq).all() and torch.isfinite(dk).all()
    # sums of up to Sq H / Hk terms in fp32, rounded to the type
    check("dv", dv_, (dv, dv.abs() * 2.0 ** (-8 if dtype == BF else -24) + Sq * H * 2.0 ** -24 * 8 + 1e-30))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-6, 3.0])
@pytest.mark.parametrize("shape", [(1, 3, 130, 2, 1, 64), (2, 150, 150, 2, 1, 96)])
def test_scales_of_either_sign(dev, shape, scale, cap, dtype):
    compare(dev, inputs(sum(shape) + 6, *shape, dtype), scale=scale, softcap=cap, causal=True)
