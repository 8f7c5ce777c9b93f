"""Rotary positions with several axes and attention with changed scores (capped, biased by distance, masked by documents, a causal
horizon and a bidirectional prefix), over the C ABI (``tf_rotary``, ``tf_score_attn_*``; include/tfusion.h).  bf16 or fp32 tensors
[B, tokens, heads, head_dim] of any batch / token / head strides: the thirds of a packed projection go in as they are.  Both run under
autograd, on the current stream of their tensors' device; CPU tensors raise -- there is no CPU path.

    plan = RotaryPlan(192, axes=(32, 32, 32), device=dev)             # time, height, width: 32 channel pairs each
    q, k = rotary(q, k, pos, plan)                                    # pos [B, S, 3] or [S, 3]
    o = score_attention(q, k, v, softcap=50.0, causal=True, prefix=n_visual, q_doc=doc, k_doc=doc)
"""
from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from transfusion_amd import _lib as L
from transfusion_amd import ops

_POS_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}


def _heads(name, t, like=None):
    """A bf16 or fp32 [B, S, H, D] device tensor, of the type and on the device of ``like``."""
    if not t.is_cuda:
        ops._require_cuda(t)
    if t.dim() != 4:
        raise L.TfError(f"{name}: [batch, tokens, heads, head_dim] expected, got {tuple(t.shape)}")
    if like is None:
        ops._is_f32(t)
    elif t.dtype != like.dtype or t.device != like.device:
        raise L.TfError(f"{name}: {t.dtype} on {t.device}, the queries are {like.dtype} on {like.device}")


def _rows(t):
    """(tensor, batch stride, token stride, head stride): ``t`` itself if its channels are contiguous, every row starts on 16 bytes and the rows
    lie within 16 MiB of each other (64 of them are addressed with 32-bit offsets), else a contiguous copy.  Strides in elements, 0 for
    an axis of length 1 (torch leaves any number there)."""
    B, S, H, D = t.shape
    sb, ss, sh, sd = t.stride()
    if B == 1:
        sb = 0
    if S == 1:
        ss = 0
    if H == 1:
        sh = 0
    n = 16 // t.element_size()
    if (sd == 1 or D == 1) and not (sb | ss | sh) & (n - 1) and not t.data_ptr() & 15 and ss < n << 20:
        return t, sb, ss, sh
    if D % n == 0 or sd != 1:            # (channel counts that no 16 bytes divide: rotary takes such rows element by element, as they are)
        t = t.clone(memory_format=torch.contiguous_format)
        sb, ss, sh = S * H * D, H * D, D
    return t, sb, ss, sh


def _ints(name, t, shape, dev):
    """An int32 device tensor of exactly ``shape``, contiguous."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
        raise L.TfError(f"{name}: an int32 tensor expected")
    ops._require_cuda(t)
    if t.device != dev or tuple(t.shape) != tuple(shape):
        raise L.TfError(f"{name}: {tuple(t.shape)} on {t.device}, expected {tuple(shape)} on {dev}")
    return t.contiguous()


def _keep(dev, *tensors):
    """Saved tensors may come from another stream's pool: the allocator must not hand their memory on before this stream has read it
    (autograd drops them as soon as the backward is enqueued)."""
    st = torch.cuda.current_stream(dev)
    for t in tensors:
        if t is not None and t.numel():
            t.record_stream(st)


def _recorded(*tensors):
    """Does autograd have to see this call?  (inside a forward-mode level always: it refuses dual tensors there, which have no tangent behind a
    kernel called directly)"""
    return forward_ad._current_level >= 0 or torch.is_grad_enabled() and any([t is not None and t.requires_grad for t in tensors])


# ------------------------------------------------------------------------------------------------------
# rotary positions
# ------------------------------------------------------------------------------------------------------
class RotaryPlan:
    """Which channel pair turns with which axis, and how fast: ``axes[a]`` pairs turn with axis ``a`` (in that order; a count of 0 leaves the
    axis out).  Pair i of n on an axis has the frequency ``base ** (-i / n)``; with ``shared`` pair p of all P has ``base ** (-p / P)``
    whatever its axis.  Pairs are the channels (p, P + p), or (2p, 2p + 1) with ``interleaved``; channels from 2 P on are not turned.
    Holds two small device tensors; make it once a model, not once a call."""

    def __init__(self, head_dim: int, axes, base: float = 10000.0, interleaved: bool = False, shared: bool = False, device="cuda"):
        axes = tuple(int(n) for n in axes)
        P = sum(axes)
        if not axes or min(axes) < 0 or P == 0 or 2 * P > head_dim or P > 256:
            raise L.TfError(f"RotaryPlan: {axes} channel pairs do not fit a head of {head_dim} channels (at most 256 pairs)")
        if not (base > 0.0 and math.isfinite(base)):
            raise L.TfError(f"RotaryPlan: base {base} must be positive and finite")
        self.head_dim, self.axes, self.base, self.pairs = int(head_dim), axes, float(base), P
        self.interleaved, self.shared = bool(interleaved), bool(shared)
        if shared:
            freq = [base ** (-p / P) for p in range(P)]
        else:
            freq = [base ** (-i / n) for n in axes for i in range(n)]
        dev = torch.device(device)
        if dev.type != "cuda":
            raise L.TfError("transfusion_amd kernels need device tensors on an MI355X (gfx950); there is no CPU fallback")
        self.freq_rev = torch.tensor([f / (2.0 * math.pi) for f in freq], dtype=torch.float64).to(dev)
        self.axis = torch.tensor([a for a, n in enumerate(axes) for _ in range(n)], dtype=torch.int32).to(dev)


_pack_rotary = L.packer("TfRotaryArgs")
_pack_score = L.packer("TfScoreAttnArgs")


def _rotary_call(q, k, pos, plan, inverse):
    dev = q.device
    q, qb, qs, qh = _rows(q)
    B, S, H, D = q.shape
    qo = torch.empty(B, S, H, D, dtype=q.dtype, device=dev)
    if k is None:
        kp = kb = ks = kh = Hk = kop = 0
        ko = None
    else:
        k, kb, ks, kh = _rows(k)
        Hk = k.shape[2]
        ko = torch.empty(B, S, Hk, D, dtype=q.dtype, device=dev)
        kp, kop = k.data_ptr(), ko.data_ptr()
    a = _pack_rotary(q.data_ptr(), qb, qs, qh, kp, kb, ks, kh, qo.data_ptr(), kop, B, S, H, Hk, D, ops._is_f32(q),
                     pos.data_ptr(), _POS_TYPES[pos.dtype], pos.dim() == 3, len(plan.axes), plan.freq_rev.data_ptr(), plan.axis.data_ptr(),
                     plan.pairs, plan.interleaved, inverse)
    with ops.on_device(dev):
        L.call_packed("tf_rotary", a, ops._stream())
    return qo, ko


class _RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, pos, plan):
        ctx.save_for_backward(pos)
        ctx.plan, ctx.shapes, ctx.dtype = plan, (q.shape, None if k is None else k.shape), q.dtype
        if any(ctx.needs_input_grad[:2]):
            _keep(q.device, pos)
        ctx.set_materialize_grads(False)
        qo, ko = _rotary_call(q, k, pos, plan, False)
        return qo if k is None else (qo, ko)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        (pos,) = ctx.saved_tensors
        live = [(i, g) for i, g in enumerate(grads) if g is not None and ctx.needs_input_grad[i]]
        out = [None, None]
        if live:
            outs = _rotary_call(live[0][1], live[1][1] if len(live) > 1 else None, pos, ctx.plan, True)
            for (i, _), g in zip(live, outs):
                out[i] = g
        return out[0], out[1], None, None


def rotary(q, k, pos, plan: RotaryPlan):
    """Turns the channel pairs of ``q`` [B, S, H, D] and ``k`` [B, S, Hk, D] (or None) by their tokens' positions -> new contiguous tensors
    (a pair, or the turned ``q`` alone).  ``pos``: [B, S, len(axes)] or [S, len(axes)] int32, int64 or fp32 (fractional positions: a
    coarse level's patches on a finer grid).  Positions take no gradient."""
    _heads("rotary q", q)
    if k is not None:
        _heads("rotary k", k, like=q)
        if k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3]:
            raise L.TfError(f"rotary: k {tuple(k.shape)} does not match q {tuple(q.shape)}")
    if not isinstance(plan, RotaryPlan) or plan.head_dim != q.shape[3] or plan.freq_rev.device != q.device:
        raise L.TfError(f"rotary: a RotaryPlan of head_dim {q.shape[3]} on {q.device} expected")
    ops._require_cuda(pos)
    if pos.dtype not in _POS_TYPES or pos.device != q.device or pos.requires_grad:
        raise L.TfError("rotary: positions are int32, int64 or fp32 tensors on the queries' device, without a gradient")
    B, S = q.shape[:2]
    if tuple(pos.shape) not in ((B, S, len(plan.axes)), (S, len(plan.axes))):
        raise L.TfError(f"rotary: positions {tuple(pos.shape)}, expected {(B, S, len(plan.axes))} or {(S, len(plan.axes))}")
    pos = pos.contiguous()
    if _recorded(q, k):
        return _RotaryFn.apply(q, k, pos, plan)
    qo, ko = _rotary_call(q, k, pos, plan, False)
    return qo if k is None else (qo, ko)


# ------------------------------------------------------------------------------------------------------
# attention with changed scores
# ------------------------------------------------------------------------------------------------------
def _score_fwd(q, k, v, opt, want_lse):
    scale, softcap, slopes, causal, prefix, q_start, q_doc, k_doc = opt
    q, qb, qs, qh = _rows(q)
    k, kb, ks, kh = _rows(k)
    v, vb, vs, vh = _rows(v)
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    dev = q.device
    out = torch.empty(B, Sq, H, D, dtype=q.dtype, device=dev)
    p = L.ptr
    f32 = ops._is_f32(q)
    lse = out_lo = None
    if want_lse:                          # for the backward: the log-sum-exps, and what the rounding of a bf16 output took
        lse = torch.empty(B, H, Sq, dtype=torch.float32, device=dev)
        out_lo = None if f32 else torch.empty_like(out)
    need = L.load().tf_score_attn_work(B, Sq, Sk, H, Hk, D, f32)
    work = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    a = _pack_score(q.data_ptr(), qb, qs, qh, k.data_ptr(), kb, ks, kh, v.data_ptr(), vb, vs, vh, out.data_ptr(), p(lse), B, Sq, Sk, H, Hk, D, f32,
                    scale, softcap, p(slopes), causal, p(prefix), p(q_start), p(q_doc), p(k_doc), p(work), need, p(out_lo),
                    0, 0, 0, 0, 0, 0, 0, 0, 0)
    with ops.on_device(dev):
        L.call_packed("tf_score_attn_fwd", a, ops._stream())
    return q, k, v, out, lse, out_lo


class _ScoreAttnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, slopes, scale, softcap, causal, prefix, q_start, q_doc, k_doc):
        opt = (scale, softcap, slopes, causal, prefix, q_start, q_doc, k_doc)
        q, k, v, out, lse, out_lo = _score_fwd(q, k, v, opt, True)
        _keep(q.device, q, k, v, slopes, prefix, q_start, q_doc, k_doc)
        ctx.save_for_backward(q, k, v, slopes, out, lse, out_lo, prefix, q_start, q_doc, k_doc)
        ctx.opt = (scale, softcap, causal)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, go):
        q, k, v, slopes, out, lse, out_lo, prefix, q_start, q_doc, k_doc = ctx.saved_tensors
        scale, softcap, causal = ctx.opt
        dev, p = q.device, L.ptr
        q, qb, qs, qh = _rows(q)
        k, kb, ks, kh = _rows(k)
        v, vb, vs, vh = _rows(v)
        go, gb, gs, gh = _rows(go)
        B, Sq, H, D = q.shape
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k, v))
        delta = torch.empty(B, H, Sq, dtype=torch.float32, device=dev)
        ds = torch.empty(H, dtype=torch.float32, device=dev) if slopes is not None and ctx.needs_input_grad[3] else None
        f32 = ops._is_f32(q)
        need = L.load().tf_score_attn_bwd_work(B, Sq, k.shape[1], H, k.shape[2], D, f32, ds is not None)
        work = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        a = _pack_score(q.data_ptr(), qb, qs, qh, k.data_ptr(), kb, ks, kh, v.data_ptr(), vb, vs, vh, out.data_ptr(), lse.data_ptr(),
                        B, Sq, k.shape[1], H, k.shape[2], D, f32, scale, softcap, p(slopes), causal, p(prefix), p(q_start), p(q_doc),
                        p(k_doc), p(work), need, p(out_lo), go.data_ptr(), gb, gs, gh, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), delta.data_ptr(), p(ds))
        with ops.on_device(dev):
            L.call_packed("tf_score_attn_bwd", a, ops._stream())
        return dq, dk, dv, ds, None, None, None, None, None, None, None


def score_attention(q, k, v, scale: float = None, softcap: float = 0.0, slopes=None, causal: bool = False, prefix=None, q_start=None,
                    q_doc=None, k_doc=None):
    """softmax(change(scale q k^T)) v -> [B, Sq, H, D], differentiable in ``q`` [B, Sq, H, D], ``k`` / ``v`` [B, Sk, Hk, D] (H a multiple of
    Hk: consecutive heads share) and ``slopes``.  A query at position p = ``q_start[b]`` + i (default: the queries are the last Sq of the
    Sk tokens) sees key j with the score

        s = scale q.k;   softcap tanh(s / softcap) if softcap > 0;   - slopes[h] |p - j|   (slopes: fp32 [H])

    unless it is hidden: ``causal`` hides j > p except the first ``prefix[b]`` keys (int32 [B]); ``q_doc`` / ``k_doc`` (int32 [B, Sq] /
    [B, Sk]) hide keys of other documents, and a negative document is padding: attends nothing, is attended by nobody, and whatever its
    rows hold is not used.  A query that sees nothing gets zeros.  (A NaN or an infinity in a key or value that some query sees may reach queries beside
    it that do not: 0 times it is not 0.)  Scores are fp32 numbers: what lies below the last place of a row's largest one, 2^-24 of it, is lost to
    probabilities and gradients.  ``scale`` (within 1e10) defaults to 1 / sqrt(D);
    ``softcap`` is 0 or between 1e-10 and 1e10.  D <= 256, a multiple of 8."""
    _heads("score_attention q", q)
    _heads("score_attention k", k, like=q)
    _heads("score_attention v", v, like=q)
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D:
        raise L.TfError(f"score_attention: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not belong together")
    if H == 0 or Hk == 0 or H % Hk:
        raise L.TfError(f"score_attention: {H} query heads cannot share {Hk} key heads")
    if D == 0 or D > 256 or D % 8:
        raise L.TfError(f"score_attention: head_dim {D} must be a multiple of 8, at most 256")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    softcap = float(softcap)
    if not abs(scale) <= 1e10 or not (softcap == 0.0 or 1e-10 <= softcap <= 1e10):
        raise L.TfError(f"score_attention: scale {scale} must lie within 1e10 of 0, softcap {softcap} be 0 (none) or between 1e-10 and 1e10")
    dev = q.device
    if slopes is not None:
        ops._require_cuda(slopes)
        if slopes.dtype != torch.float32 or tuple(slopes.shape) != (H,) or slopes.device != dev:
            raise L.TfError(f"score_attention: slopes must be fp32 [{H}] on {dev}")
        slopes = slopes.contiguous()
    if prefix is not None:
        if not causal:
            raise L.TfError("score_attention: a prefix needs causal=True (without it every key is visible)")
        prefix = _ints("score_attention prefix", prefix, (B,), dev)
    if q_start is not None:
        q_start = _ints("score_attention q_start", q_start, (B,), dev)
    if (q_doc is None) != (k_doc is None):
        raise L.TfError("score_attention: q_doc and k_doc come together")
    if q_doc is not None:
        q_doc = _ints("score_attention q_doc", q_doc, (B, Sq), dev)
        k_doc = _ints("score_attention k_doc", k_doc, (B, Sk), dev)
    if _recorded(q, k, v, slopes):
        return _ScoreAttnFn.apply(q, k, v, slopes, scale, softcap, int(bool(causal)), prefix, q_start, q_doc, k_doc)
    return _score_fwd(q, k, v, (scale, softcap, slopes, int(bool(causal)), prefix, q_start, q_doc, k_doc), False)[3]
