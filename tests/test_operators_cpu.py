"""Refusals of the rotary, score-attention and gradient-clip entries: argument errors come back before anything is launched, so the C
entries are called here without a GPU; the Python entry points refuse CPU tensors."""
import ctypes as C
import math

import pytest
import torch

from transfusion_amd import _lib as L, attention_ops, optim

PTR = 1 << 20          # a 16-byte aligned number in place of an address: nothing reads it, every call below is refused first


@pytest.fixture(scope="module")
def lib():
    import os
    from transfusion_amd import build
    if not os.path.exists(L.LIB_PATH):
        build.build_lib()
    return L.load()


def rotary_args(**kw):
    a = dict(q=PTR, q_sb=640, q_ss=64, q_sh=16, k=PTR, k_sb=640, k_ss=64, k_sh=16, q_out=PTR, k_out=PTR, B=1, S=10, H=4, Hk=4, D=16, is_f32=0,
             pos=PTR, pos_type=0, n_axes=2, inv_freq=PTR, axis=PTR, pairs=8)
    a.update(kw)
    return L.TfRotaryArgs(**a)


@pytest.mark.parametrize("kw", [dict(pairs=0), dict(pairs=9), dict(D=0), dict(B=-1), dict(S=-2), dict(H=-1), dict(pos_type=3), dict(n_axes=0), dict(pos=0),
                                dict(inv_freq=0), dict(axis=0), dict(q=0), dict(k_out=0), dict(pairs=257, D=1024)])
def test_rotary_entry_refuses(lib, kw):
    a = rotary_args(**kw)
    assert lib.tf_rotary(C.byref(a), None) < 0
    assert b"tf_rotary" in lib.tf_last_error()


def attn_args(**kw):
    a = dict(q=PTR, q_sb=640, q_ss=64, q_sh=16, k=PTR, k_sb=640, k_ss=64, k_sh=16, v=PTR, v_sb=640, v_ss=64, v_sh=16, out=PTR, lse=PTR, B=1, Sq=10, Sk=10,
             H=4, Hk=4, D=16, is_f32=0, scale=0.25, dout=PTR, do_sb=640, do_ss=64, do_sh=16, dq=PTR, dk=PTR, dv=PTR, delta=PTR)
    a.update(kw)
    return L.TfScoreAttnArgs(**a)


BOTH = [dict(H=0), dict(Hk=0), dict(Hk=3), dict(D=0), dict(D=12), dict(D=264), dict(B=-1), dict(Sq=-1), dict(Sk=-1), dict(softcap=-1.0),
        dict(softcap=math.inf), dict(softcap=1e-11), dict(softcap=1e11), dict(scale=math.inf), dict(scale=math.nan), dict(scale=-1e11),
        dict(softcap=math.nan), dict(q_doc=PTR), dict(k_doc=PTR), dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(q=PTR + 8), dict(k_ss=60), dict(v_sh=4),
        dict(q_sb=4), dict(B=1 << 20, Sq=1 << 10), dict(Sk=1 << 30)]


@pytest.mark.parametrize("kw", BOTH + [dict(B=1, H=1, Hk=1, Sq=1, Sk=1 << 16, work_bytes=16, work=PTR)])
def test_score_attn_fwd_entry_refuses(lib, kw):
    a = attn_args(**kw)
    assert lib.tf_score_attn_fwd(C.byref(a), None) < 0
    assert b"tf_score_attn_fwd" in lib.tf_last_error()


@pytest.mark.parametrize("kw", BOTH + [dict(lse=0), dict(delta=0), dict(dout=0), dict(dq=0), dict(dk=0), dict(dv=0), dict(do_ss=4), dict(dk=PTR + 4),
                                       dict(dslopes=PTR), dict(dslopes=PTR, slopes=PTR), dict(Hk=1, Sq=900, work=PTR, work_bytes=64), dict(out_lo=PTR + 8)])
def test_score_attn_bwd_entry_refuses(lib, kw):
    a = attn_args(**kw)
    assert lib.tf_score_attn_bwd(C.byref(a), None) < 0
    assert b"tf_score_attn_bwd" in lib.tf_last_error()


def clip_args(ptrs, lens, bf, **kw):
    n = len(ptrs)
    p, l, b = (C.c_void_p * n)(*ptrs), (C.c_longlong * n)(*lens), (C.c_int * n)(*bf)
    a = dict(grads=C.addressof(p), n=C.addressof(l), is_bf16=C.addressof(b), count=n, norm_type=0, clip=1, max_norm=1.0, norm=PTR, work=PTR, parts=1 << 20)
    a.update(kw)
    return L.TfGradClipArgs(**a), (p, l, b)


@pytest.mark.parametrize("kw", [dict(count=-1), dict(norm_type=2), dict(work=0), dict(norm=0), dict(parts=1), dict(n=0), dict(grads=0), dict(is_bf16=0)])
def test_grad_clip_entry_refuses(lib, kw):
    a, keep = clip_args([PTR, PTR + (1 << 18)], [40000, 40000], [0, 0], **kw)
    assert lib.tf_grad_clip(C.byref(a), None) < 0
    assert b"tf_grad_clip" in lib.tf_last_error()


@pytest.mark.parametrize("ptrs,lens,bf", [([PTR, PTR], [8, 8], [0, 0]), ([PTR, PTR + 28], [8, 8], [0, 0]), ([PTR + 15, PTR], [8, 8], [1, 1]), ([0], [4], [0]),
                                          ([PTR + 2], [4], [0]), ([PTR + 1], [4], [1]), ([PTR], [-1], [0]), ([PTR], [1 << 50], [0])])
def test_grad_clip_refuses_overlaps_and_bad_tensors(lib, ptrs, lens, bf):
    a, keep = clip_args(ptrs, lens, bf)
    assert lib.tf_grad_clip(C.byref(a), None) < 0


def test_null_arguments(lib):
    for f in ("tf_rotary", "tf_score_attn_fwd", "tf_score_attn_bwd", "tf_grad_clip"):
        assert getattr(lib, f)(None, None) == -1
    assert lib.tf_grad_clip_parts(None, 3) < 0 and lib.tf_grad_clip_parts(None, 0) == 1


def test_cpu_tensors_are_refused():
    q = torch.randn(1, 2, 2, 16)
    with pytest.raises(L.TfError):
        attention_ops.score_attention(q, q, q)
    with pytest.raises(L.TfError):
        attention_ops.rotary(q, q, torch.zeros(2, 1, dtype=torch.int32), None)
    with pytest.raises(L.TfError):
        attention_ops.RotaryPlan(16, (8,), device="cpu")
    p = torch.zeros(3, requires_grad=True)
    p.grad = torch.ones(3)
    with pytest.raises(L.TfError):
        optim.clip_grad_norm_([p], 1.0)


@pytest.mark.parametrize("kw", [dict(axes=(5, 4)), dict(axes=()), dict(axes=(0, 0)), dict(axes=(-1, 3)), dict(axes=(4,), base=0.0), dict(axes=(4,), base=math.inf)])
def test_rotary_plan_refuses(kw):
    with pytest.raises(L.TfError):
        attention_ops.RotaryPlan(16, device="cuda", **kw)


def test_clip_refuses():
    for kw in (dict(norm_type=1.0), dict(max_norm=-1.0), dict(max_norm=math.nan)):
        with pytest.raises(L.TfError):
            optim.clip_grad_norm_([], **{"max_norm": 1.0, **kw})
