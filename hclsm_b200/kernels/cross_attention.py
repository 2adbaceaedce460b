"""Cross attention: queries over another set of states, of another length.

The goal transformer of the reference (hclsm/dynamics/level2_goal.py:88-141)
lets a few queries attend to a video's states; slots attend to patch tokens and
rollout steps to their history in the same way.  ``cross_attention(q, k, v)``
takes ragged state counts and a mask of dead slots, shares key heads between
query heads, and is differentiable in q, k and v (bit-reproducible gradients).
"""
from __future__ import annotations

import ctypes
import math

import torch

from .. import _lib

__all__ = ["cross_attention"]


def _args(q, k, v, o, lse, lens, mask, scale):
    a = _lib.XattnArgs()
    a.q, a.k, a.v = _lib.view(q), _lib.view(k), _lib.view(v)
    a.o, a.lse2, a.lens = o.data_ptr(), _lib.ptr(lse), _lib.ptr(lens)
    if mask is not None:
        a.mask, a.mask_sb = mask.data_ptr(), mask.stride(0)
    a.B, a.Lq, a.H, a.D = q.shape
    a.Lk, a.Hkv = k.shape[1], k.shape[2]
    a.dtype, a.scale = _lib.dtype_code(q.dtype), scale
    return a


def _workspace(n, device):
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def _forward(q, k, v, lens, mask, scale, keep):
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    B, Lq, H, _ = q.shape
    lse = torch.empty(B, H, Lq, dtype=torch.float32, device=q.device) if keep else None
    a = _args(q, k, v, o, lse, lens, mask, scale)
    lib, at = _lib.load(), ctypes.addressof(a)
    n = lib.hclsm_xattn_fwd_workspace_size(at)
    ws = _workspace(n, q.device)
    _lib.check(lib.hclsm_xattn_fwd(at, _lib.ptr(ws), n, _lib.stream_ptr(q.device)), "hclsm_xattn_fwd")
    return o, lse


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lens, mask, scale):
        o, lse = _forward(q, k, v, lens, mask, scale, True)
        ctx.save_for_backward(q, k, v, o, lse, lens, mask)
        ctx.scale = scale
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse, lens, mask = ctx.saved_tensors
        do = _lib.dense_last(do.to(q.dtype))
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        a = _args(q, k, v, o, lse, lens, mask, ctx.scale)
        a.dout = _lib.view(do)
        a.dq, a.dk, a.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
        lib, at = _lib.load(), ctypes.addressof(a)
        n = lib.hclsm_xattn_bwd_workspace_size(at)
        ws = _workspace(n, q.device)
        _lib.check(lib.hclsm_xattn_bwd(at, _lib.ptr(ws), n, _lib.stream_ptr(q.device)), "hclsm_xattn_bwd")
        return dq, dk, dv, None, None, None


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
    q, k, v = _lib.dense_last(q), _lib.dense_last(k), _lib.dense_last(v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _CrossAttention.apply(q, k, v, lens, key_mask, scale)
    return _forward(q, k, v, lens, key_mask, scale, False)[0]
