"""Cross attention: queries over another set of states, of another length.

The goal transformer of the reference (hclsm/dynamics/level2_goal.py:88-141)
lets a few queries attend to a video's states; slots attend to patch tokens and
rollout steps to their history in the same way.  ``cross_attention(q, k, v)``
takes ragged state counts and a mask of dead slots, shares key heads between
query heads, and is differentiable in q, k and v (bit-reproducible gradients).
"""
from __future__ import annotations

import math

import torch

from .. import _lib

__all__ = ["cross_attention"]


def _args(q, k, v, o, lse, lo, lens, mask, scale, do=None, dq=None, dk=None, dv=None):
    B, Lq, H, D = q.shape
    qb, qt, qh, _ = q.stride()
    kb, kt, kh, _ = k.stride()
    vb, vt, vh, _ = v.stride()
    gp = gb = gt = gh = dqp = dkp = dvp = 0
    if do is not None:
        gp, gb, gt, gh = _lib.view_args(do)
        dqp, dkp, dvp = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    return _lib.XATTN_ARGS.pack(
        q.data_ptr(), qb, qt, qh, k.data_ptr(), kb, kt, kh, v.data_ptr(), vb, vt, vh, gp, gb, gt, gh, o.data_ptr(),
        dqp, dkp, dvp, 0 if lse is None else lse.data_ptr(), 0 if lo is None else lo.data_ptr(),
        0 if lens is None else lens.data_ptr(),
        0 if mask is None else mask.data_ptr(), 0 if mask is None else mask.stride(0), B, Lq, k.shape[1], H, k.shape[2],
        D, _lib.dtype_code(q.dtype), scale)


def _forward(q, k, v, lens, mask, scale, keep):
    o = q.new_empty(q.shape)
    lse = lo = None
    if keep:
        B, Lq, H, _ = q.shape
        lse = q.new_empty((B, H, Lq), dtype=torch.float32)
        if q.dtype == torch.bfloat16:
            lo = q.new_empty(q.shape)  # what rounding takes from o: the backward's row sums do . o are then fp32's
    a = _args(q, k, v, o, lse, lo, lens, mask, scale)
    lib, ws = _lib.load(), None
    n = lib.hclsm_xattn_fwd_workspace_size(a)
    if n:
        ws = q.new_empty(n, dtype=torch.uint8)
    _lib.check(lib.hclsm_xattn_fwd(a, None if ws is None else ws.data_ptr(), n, _lib.stream_ptr(q.device)),
               "hclsm_xattn_fwd")
    return o, lse, lo


def _backward(q, k, v, o, lse, lo, lens, mask, scale, do):
    do = _lib.dense_last(do)
    dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
    a = _args(q, k, v, o, lse, lo, lens, mask, scale, do, dq, dk, dv)
    lib = _lib.load()
    n = lib.hclsm_xattn_bwd_workspace_size(a)
    ws = q.new_empty(n, dtype=torch.uint8)
    _lib.check(lib.hclsm_xattn_bwd(a, ws.data_ptr(), n, _lib.stream_ptr(q.device)), "hclsm_xattn_bwd")
    return dq, dk, dv


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lens, mask, scale):
        o, lse, lo = _forward(q, k, v, lens, mask, scale, True)
        ctx.save_for_backward(q, k, v, o, lse, lo, lens, mask)
        ctx.scale = scale
        return o

    @staticmethod
    def backward(ctx, do):
        _lib.no_double_backward()
        return (*_backward(*ctx.saved_tensors, ctx.scale, do), None, None, None)


def _prepare(q, k, v, kv_lens, key_mask, scale):
    """The checked arguments of the kernels."""
    if _lib.in_dual_level():
        _lib.no_tangents(q, k, v)
    dev = _lib.require_cuda(q, k, v, kv_lens, key_mask)
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape:
        raise ValueError("q must be (B, Lq, H, D); k and v (B, Lk, Hkv, D)")
    B, _, H, D = q.shape
    if k.shape[0] != B or k.shape[3] != D:
        raise ValueError(f"k and v must share q's batch and head_dim {(B, D)}, got {tuple(k.shape)}")
    if k.shape[2] < 1 or H < 1 or H % k.shape[2]:
        raise ValueError(f"query heads ({H}) must be a multiple of key heads ({k.shape[2]})")
    if not 1 <= D <= 128:
        raise ValueError(f"head_dim must be 1 to 128, got {D}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"q, k and v must share one dtype, got {q.dtype}, {k.dtype}, {v.dtype}")
    _lib.dtype_code(q.dtype)
    scale = D ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    lens = _lib.index32(kv_lens, (B,), "kv_lens", dev)
    if key_mask is not None:
        if key_mask.dtype != torch.bool or tuple(key_mask.shape) != (B, k.shape[1]):
            raise ValueError(f"key_mask must be {(B, k.shape[1])} bool")
        key_mask = _lib.dense_last(key_mask)
    return _lib.dense_last(q), _lib.dense_last(k), _lib.dense_last(v), lens, key_mask, scale


def attention_fwd(q, k, v, kv_lens, key_mask, scale):
    """(o, lse2, lo): the forward and what its backward needs (lo: None in fp32), without autograd."""
    return _forward(*_prepare(q, k, v, kv_lens, key_mask, scale), True)


def attention_bwd(q, k, v, o, lse, lo, do, kv_lens, key_mask, scale):
    """(dq, dk, dv) from attention_fwd's results."""
    q, k, v, lens, key_mask, scale = _prepare(q, k, v, kv_lens, key_mask, scale)
    o, do = (_lib.like(t, q.shape, q.dtype, n, q.device) for t, n in ((o, "o"), (do, "do")))
    lse = _lib.like(lse, (q.shape[0], q.shape[2], q.shape[1]), torch.float32, "lse", q.device)
    if lo is not None:
        if q.dtype != torch.bfloat16:
            raise TypeError("lo goes with bfloat16")
        lo = _lib.like(lo, q.shape, q.dtype, "lo", q.device)
    return _backward(q, k, v, o, lse, lo, lens, key_mask, scale, do)


def cross_attention(q, k, v, *, kv_lens=None, key_mask=None, scale=None):
    """softmax(scale q k^T) v for q (B, Lq, H, D) and k, v (B, Lk, Hkv, D).

    H is a multiple of Hkv: query head h reads key head h // (H // Hkv).
    ``kv_lens`` (B,) int: entry b's first kv_lens[b] states count (clamped to
    [0, Lk]); ``key_mask`` (B, Lk) bool: False states do not count.  What does not
    count is never read as an operand (it may be NaN), and its gradients are zero;
    a query with no state gives zeros.  ``scale`` > 0, default D ** -0.5.
    float32 or bfloat16, head_dim up to 128; softmax and sums in fp32.  Heads are
    dense, the other strides are free.
    """
    q, k, v, lens, key_mask, scale = _prepare(q, k, v, kv_lens, key_mask, scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _CrossAttention.apply(q, k, v, lens, key_mask, scale)
    return _forward(q, k, v, lens, key_mask, scale, False)[0]
