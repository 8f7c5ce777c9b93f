"""Forward-mode derivatives of the rotary and score-attention operators are refused, as for every operator of the package: a result without its
tangent would pass for a constant."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def calls():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    from transfusion_amd import attention_ops as A
    dev = torch.device("cuda:0")
    plan = A.RotaryPlan(16, (4, 4), device=dev)
    pos = torch.arange(20, dtype=torch.int32, device=dev).view(10, 2)
    x = torch.randn(2, 10, 4, 16, generator=torch.Generator().manual_seed(1)).to(dev)
    sl = torch.ones(4, device=dev)
    return x, {"rotary q": lambda t: A.rotary(t, None, pos, plan), "rotary k": lambda t: A.rotary(x, t, pos, plan)[1],
               "attention q": lambda t: A.score_attention(t, x, x), "attention k": lambda t: A.score_attention(x, t, x, causal=True),
               "attention v": lambda t: A.score_attention(x, x, t), "attention slopes": lambda t: A.score_attention(x, x, x, slopes=sl * t.mean())}


@pytest.mark.parametrize("name", ["rotary q", "rotary k", "attention q", "attention k", "attention v", "attention slopes"])
@pytest.mark.parametrize("grad", [True, False])
def test_dual_tensors_are_refused(calls, name, grad):
    x, fns = calls
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x.clone().requires_grad_(grad), torch.ones_like(x))
        with pytest.raises(NotImplementedError):
            fns[name](d)
        with torch.no_grad(), pytest.raises(NotImplementedError):
            fns[name](d)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(fns[name], (x,), (torch.ones_like(x),))


@pytest.mark.parametrize("name", ["rotary q", "rotary k", "attention q", "attention k"])
def test_plain_tensors_inside_a_level_give_the_same(calls, name):
    x, fns = calls
    want = fns[name](x)
    with forward_ad.dual_level():
        assert torch.equal(fns[name](x), want)
