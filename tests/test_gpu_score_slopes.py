"""Slopes of attention with changed scores: gradients where values are not finite (what a row sees reaches them, what is hidden does not), and
queries far from the keys."""
import math

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


def inputs(seed, B, Sq, Sk, H, Hk, D, dtype, dev):
    g = torch.Generator().manual_seed(seed)
    q, k, v, go = (torch.randn(B, s, h, D, generator=g).to(dtype).to(dev) for s, h in ((Sq, H), (Sk, Hk), (Sk, Hk), (Sq, H)))
    return q, k, v, go, torch.tensor([0.7 ** h for h in range(H)], device=dev)


def gradients(q, k, v, go, sl, **opt):
    from transfusion_amd import attention_ops as A
    q, k, v, sl = (t.detach().clone().requires_grad_(True) for t in (q, k, v, sl))
    out = A.score_attention(q, k, v, slopes=sl, **opt)
    return (out.detach(),) + torch.autograd.grad(out, (q, k, v, sl), go)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [(1, 2, 90, 4, 2, 64), (2, 130, 130, 4, 2, 64), (3, 500, 500, 2, 2, 16)])
@pytest.mark.parametrize("where", ["key", "query", "value", "dout"])
def test_what_is_visible_reaches_the_slopes(dev, where, shape, dtype):
    q, k, v, go, sl = inputs(sum(shape), *shape, dtype, dev)
    G = shape[3] // shape[4]
    {"key": k, "query": q, "value": v, "dout": go}[where][0, 0, 0, 3] = math.nan     # of the first head (of keys)
    ds = gradients(q, k, v, go, sl, causal=True)[4]
    n = G if where in ("key", "value") else 1
    assert torch.isnan(ds[:n]).all() and torch.isfinite(ds[n:]).all(), ds


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Sq,Sk", [(2, 90), (130, 130), (70, 300)])
def test_what_is_hidden_does_not(dev, Sq, Sk, dtype):
    """NaN and infinities in padded rows of every operand (queries, keys, values, output gradients)."""
    q, k, v, go, sl = inputs(Sq, 2, Sq, Sk, 4, 2, 64, dtype, dev)
    k_doc = torch.zeros(2, Sk, dtype=torch.int32, device=dev)
    k_doc[0, :Sk // 3], k_doc[1, Sk - 1:] = -1, -1
    q_doc = k_doc[:, Sk - Sq:].contiguous()
    opt = {"causal": True, "q_doc": q_doc, "k_doc": k_doc, "softcap": 9.0}
    clean = [t.clone() for t in (q, k, v, go)]
    for t, dead in zip(clean, (q_doc, k_doc, k_doc, q_doc)):
        t[dead < 0] = 0
    want = attention_bounds(*clean, slopes=sl, **opt)
    for t, dead, x in ((q, q_doc, math.nan), (k, k_doc, math.nan), (v, k_doc, math.inf), (go, q_doc, -math.inf)):
        t[dead < 0] = x
    for n, got in zip(("out", "dq", "dk", "dv", "dslopes"), gradients(q, k, v, go, sl, **opt)):
        check(n, got, want[n])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", [(4, 2, 300, 4, 2, 64), (4, 70, 70, 2, 1, 32), (4, 140, 200, 2, 2, 128)])
def test_queries_far_from_the_keys(dev, shape, causal, dtype):
    """Queries behind the last key, before the first, across either end, up to the largest number: a shift of all distances of a row changes neither
    the softmax nor a gradient, so no precision may be lost to it."""
    q, k, v, go, sl = inputs(sum(shape) + 3, *shape, dtype, dev)
    for starts in ((1000000, 200, 2 ** 31 - 1, 65), (-3, -1000000, -2 ** 31, 280)):
        start = torch.tensor(starts, dtype=torch.int32, device=dev)
        opt = {"causal": causal, "q_start": start, "softcap": 20.0}
        want = attention_bounds(q, k, v, go, slopes=sl, **opt)
        for n, got in zip(("out", "dq", "dk", "dv", "dslopes"), gradients(q, k, v, go, sl, **opt)):
            check(f"{n} {starts}", got, want[n])
