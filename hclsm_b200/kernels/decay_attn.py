"""Linear attention whose state forgets at a rate of each head: a memory of constant size.

Beside the selective scan, whose state is a few numbers a channel, this state is
a matrix a head: ``S_t = g S_{t-1} + k_t^T v_t`` is read by ``o_t = scale q_t S_t``,
with ``g = exp(log_decay)`` of the head.  ``decay_attention`` runs whole
histories in chunks on the tensor cores, forward and backward;
``decay_attention_step`` takes one token through the state.
"""
from __future__ import annotations

import math

import torch

from .. import _lib

__all__ = ["decay_attention", "decay_attention_step"]


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _args(q, k, v, decay, s0, lens, scale, o=None, s1=None, do=None, dq=None, dk=None, dv=None, ds1=None, ds0=None):
    B, L, H, D = q.shape
    return _lib.DECAY_ARGS.pack(
        *_lib.view_args(q), *_lib.view_args(k), *_lib.view_args(v),
        *((0, 0, 0, 0) if do is None else _lib.view_args(do)), _ptr(o), _ptr(dq), _ptr(dk), _ptr(dv), decay.data_ptr(),
        _ptr(s0), _ptr(s1), _ptr(ds1), _ptr(ds0), _ptr(lens), B, L, H, D, v.shape[3], _lib.dtype_code(q.dtype), scale)


def _workspace(q, n):
    return q.new_empty(n, dtype=torch.uint8) if n else None


def _forward(q, k, v, decay, s0, lens, scale, want_state):
    B, L, H, D = q.shape
    o = _lib.empty_like(v)
    s1 = q.new_empty((B, H, D, v.shape[3]), dtype=torch.float32) if want_state else None
    a = _args(q, k, v, decay, s0, lens, scale, o, s1)
    lib = _lib.load()
    n = lib.hclsm_decay_attn_fwd_workspace_size(a)
    ws = _workspace(q, n)
    _lib.check(lib.hclsm_decay_attn_fwd(a, _lib.ptr(ws), n, _lib.stream_ptr(q.device)), "hclsm_decay_attn_fwd")
    return o, s1


def _backward(q, k, v, decay, s0, lens, scale, do, ds1, want_ds0):
    do = _lib.dense_last(do)
    dq, dk, dv = _lib.empty_like(q), _lib.empty_like(k), _lib.empty_like(v)
    ds0 = torch.empty_like(s0) if want_ds0 else None
    if ds1 is not None:
        ds1 = ds1.contiguous()
    a = _args(q, k, v, decay, s0, lens, scale, None, None, do, dq, dk, dv, ds1, ds0)
    lib = _lib.load()
    n = lib.hclsm_decay_attn_bwd_workspace_size(a)
    ws = _workspace(q, n)
    _lib.check(lib.hclsm_decay_attn_bwd(a, _lib.ptr(ws), n, _lib.stream_ptr(q.device)), "hclsm_decay_attn_bwd")
    return dq, dk, dv, ds0


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, decay, s0, lens, scale, want_state):
        o, s1 = _forward(q, k, v, decay, s0, lens, scale, want_state)
        ctx.save_for_backward(q, k, v, decay, s0, lens)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, s1

    @staticmethod
    def backward(ctx, do, ds1):
        _lib.no_double_backward()
        q, k, v, decay, s0, lens = ctx.saved_tensors
        if do is None:
            if ds1 is None:
                return (None,) * 8
            do = torch.zeros_like(v)
        dq, dk, dv, ds0 = _backward(q, k, v, decay, s0, lens, ctx.scale, do, ds1, ctx.needs_input_grad[4])
        return dq, dk, dv, None, ds0, None, None, None


def _check_decay(decay, H):
    if decay.shape != (H,) or decay.dtype != torch.float32:
        raise ValueError(f"log_decay must be ({H},) float32, got {tuple(decay.shape)} {decay.dtype}")
    if decay.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("decay_attention has no gradient of log_decay: detach it")
    return decay if decay.is_contiguous() else decay.contiguous()


def _check_scale(scale, D):
    scale = D ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    return scale


def _check_state(state, shape, name="state"):
    if state.shape != shape or state.dtype != torch.float32:
        raise ValueError(f"{name} must be {shape} float32, got {tuple(state.shape)} {state.dtype}")


def _prepare(q, k, v, log_decay, state, lens, scale):
    """The checked arguments of the kernels."""
    if _lib.in_dual_level():
        _lib.no_tangents(q, k, v, log_decay, state)
    dev = _lib.require_cuda(q, k, v, log_decay, state, lens)
    if q.dim() != 4 or k.shape != q.shape or v.dim() != 4 or v.shape[:3] != q.shape[:3]:
        raise ValueError(f"q and k must be (B, L, H, D), v (B, L, H, Dv), got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    B, _, H, D = q.shape
    Dv = v.shape[3]
    if H < 1 or not 1 <= D <= 128 or not 1 <= Dv <= 128:
        raise ValueError(f"head dims must be 1 to 128, got {D} and {Dv} of {H} heads")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"q, k and v must share one dtype, got {q.dtype}, {k.dtype}, {v.dtype}")
    _lib.dtype_code(q.dtype)
    log_decay = _check_decay(log_decay, H)
    if state is not None:
        _check_state(state, (B, H, D, Dv))
        state = state.contiguous()
    return (_lib.dense_last(q), _lib.dense_last(k), _lib.dense_last(v), log_decay, state,
            _lib.index32(lens, (B,), "lens", dev), _check_scale(scale, D))


def decay_fwd(q, k, v, log_decay, state, lens, scale):
    """(o, final state) without autograd."""
    return _forward(*_prepare(q, k, v, log_decay, state, lens, scale), True)


def decay_bwd(q, k, v, log_decay, state, lens, scale, do, dstate):
    """(dq, dk, dv, gradient of the first state or None); dstate: of the final state, or None."""
    args = _prepare(q, k, v, log_decay, state, lens, scale)
    do = _lib.like(do, v.shape, q.dtype, "do", q.device)
    if dstate is not None:
        dstate = _lib.like(dstate, (q.shape[0], q.shape[2], q.shape[3], v.shape[3]), torch.float32, "dstate", q.device)
    return _backward(*args, do, dstate, state is not None)


def decay_attention(q, k, v, log_decay, *, state=None, lens=None, scale=None, return_state: bool = False):
    """o (B, L, H, Dv) of q, k (B, L, H, D) and v (B, L, H, Dv): token t reads the state with its own token in it.

    ``log_decay`` (H,) fp32: logarithm of each head's factor a token, at most 0 (above counts as 0;
    -inf forgets all).  ``state`` (B, H, D, Dv) fp32: the state before the first token, default zeros;
    with ``return_state`` the result is (o, the state behind the last token).  ``lens`` (B,) int: entry
    b's first lens[b] tokens count (clamped to [0, L]); the others may hold anything, NaN included, and their
    outputs and gradients are zeros.  A token that counts and is not finite spreads to the
    tokens of its chunk (128; 64 in fp32), the earlier ones too.  ``scale`` > 0, default D ** -0.5.  float32 or bfloat16, head dims up to
    128; sums and states in fp32.  bfloat16 runs on the tensor cores where dims, strides and addresses are
    whole 16 bytes and no dim of more than one is expanded (in the backward those of o's gradient too), else on the
    much slower FMA pipe.  Differentiable in q, k, v and state, not in log_decay; bit-reproducible.
    """
    args = _prepare(q, k, v, log_decay, state, lens, scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or (state is not None and state.requires_grad)):
        o, s1 = _DecayAttention.apply(*args, return_state)
    else:
        o, s1 = _forward(*args, return_state)
    return (o, s1) if return_state else o


def decay_attention_step(q, k, v, log_decay, state, *, out=None, active=None, scale=None):
    """One token: o (B, H, Dv) of q, k (B, H, D) and v (B, H, Dv); ``state`` (B, H, D, Dv) fp32 takes it in, in place, or
    ``out`` gets the new state and ``state`` stays.  ``active`` (B,) bool: an entry that is not keeps its state and gives
    zeros.  The state is rounded to fp32 once a token: a head that forgets less than 2^-25 of it a token keeps a value to which
    nothing is added.  No gradients."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad
                                    or (out is not None and out.requires_grad)):
        raise NotImplementedError("decay_attention_step has no gradients: call it under torch.no_grad()")
    if _lib.in_dual_level():
        _lib.no_tangents(q, k, v, log_decay, state)
    dev, index = _lib.require_cuda(q), q.get_device()
    if (k.get_device() != index or v.get_device() != index or log_decay.get_device() != index
            or state.get_device() != index or (out is not None and out.get_device() != index)
            or (active is not None and active.get_device() != index)):
        raise ValueError(f"all tensors must be on {dev}")
    shape_q, shape_v = q.shape, v.shape
    if len(shape_q) != 3 or k.shape != shape_q or len(shape_v) != 3 or shape_v[:2] != shape_q[:2]:
        raise ValueError(f"q and k must be (B, H, D), v (B, H, Dv), got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    B, H, D = shape_q
    Dv = shape_v[2]
    if H < 1 or not 1 <= D <= 128 or not 1 <= Dv <= 128:
        raise ValueError(f"head dims must be 1 to 128, got {D} and {Dv} of {H} heads")
    dtype = q.dtype
    if k.dtype != dtype or v.dtype != dtype:
        raise TypeError(f"q, k and v must share one dtype, got {q.dtype}, {k.dtype}, {v.dtype}")
    log_decay = _check_decay(log_decay, H)
    shape = (B, H, D, Dv)
    _check_state(state, shape)
    if out is None:
        out = state
    elif out is not state:
        _check_state(out, shape, "out")
        far = out.data_ptr() - state.data_ptr()
        if far and abs(far) < 4 * state.numel():
            raise ValueError("out overlaps state without being it")
    if not state.is_contiguous() or not out.is_contiguous():
        raise ValueError("state and out must be contiguous")
    if active is not None:
        if active.dtype != torch.bool or active.shape != (B,):
            raise ValueError(f"active must be ({B},) bool")
        active = active.contiguous()
    q, k, v = _lib.dense_last(q), _lib.dense_last(k), _lib.dense_last(v)
    o = _lib.empty_like(v)
    qb, qh, _ = q.stride()
    kb, kh, _ = k.stride()
    vb, vh, _ = v.stride()
    a = _lib.DECAY_ARGS.pack(
        q.data_ptr(), qb, 0, qh, k.data_ptr(), kb, 0, kh, v.data_ptr(), vb, 0, vh, 0, 0, 0, 0, o.data_ptr(), 0, 0, 0,
        log_decay.data_ptr(), state.data_ptr(), out.data_ptr(), 0, 0, 0, B, 1, H, D, Dv, _lib.dtype_code(dtype),
        _check_scale(scale, D))
    _lib.check(_lib.load().hclsm_decay_attn_step(a, _lib.ptr(active), _lib.stream_ptr(dev)), "hclsm_decay_attn_step")
    _lib.changed(out)
    return o
