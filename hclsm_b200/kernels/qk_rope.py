"""Per-head norm of queries and keys and their position rotation, one launch.

``qk_norm_rope(q, k, q_weight, k_weight, cos, sin)`` normalises every head of
q (B, Lq, H, D) and k (B, Lk, Hkv, D) by its root mean square, multiplies by the
weight and turns the first ``2 * cos.shape[1]`` dims by the angles of the token's
position; forward and backward are one pass over the data each (plus a short
reduction for the weights' gradients).  All arithmetic is fp32; outputs and
gradients have their inputs' dtypes (float32 or bfloat16; weights fp32).
"""
from __future__ import annotations

import torch

from .. import _lib

__all__ = ["qk_norm_rope", "rope_tables"]

_INTERLEAVED, _NO_NORM = 1, 2


def rope_tables(positions: int, dim: int, base: float = 10000.0, *, scale: float = 1.0, device="cuda"):
    """(cos, sin), each (positions, dim / 2) fp32: position p turns pair i by
    ``p / scale * base ** (-2 i / dim)``; ``scale`` > 1 stretches the angles of
    short training contexts over longer ones."""
    if dim < 2 or dim % 2 or positions < 0 or not scale > 0 or not base > 0:
        raise ValueError(f"rope_tables: positions {positions}, dim {dim}, base {base}, scale {scale}")
    freq = float(base) ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    ang = torch.arange(positions, dtype=torch.float64)[:, None] / float(scale) * freq
    return ang.cos().float().to(device), ang.sin().float().to(device)


def _dense16(t):
    if not t.is_contiguous():
        t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _check(q, k, q_weight, k_weight, cos, sin, eps):
    if _lib.in_dual_level():
        _lib.no_tangents(q, k, q_weight, k_weight, cos, sin)
    dev = _lib.require_cuda(q, k, q_weight, k_weight, cos, sin)
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError("q and k must be (batch, tokens, heads, head_dim)")
    B, D = q.shape[0], q.shape[3]
    if k is not None and (k.shape[0] != B or k.shape[3] != D):
        raise ValueError(f"k must share q's batch and head_dim {(B, D)}, got {tuple(k.shape)}")
    if k is not None and k.dtype != q.dtype:
        raise TypeError(f"q and k must share one dtype, got {q.dtype} and {k.dtype}")
    if k is None and k_weight is not None:
        raise ValueError("k_weight without k")
    _lib.dtype_code(q.dtype)
    if D % 8 or not 8 <= D <= 256:
        raise ValueError(f"head_dim must be a multiple of 8 up to 256, got {D}")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            continue
        if eps is None:
            raise ValueError(f"{name} without the norm (eps=None)")
        if w.shape != (D,) or w.dtype != torch.float32:
            raise ValueError(f"{name} must be ({D},) float32")
    if ((cos is not None and cos.requires_grad) or (sin is not None and sin.requires_grad)) and torch.is_grad_enabled():
        raise NotImplementedError("qk_norm_rope has no gradients of cos and sin: detach them")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    if cos is not None:
        if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
            raise ValueError("cos and sin must be (positions, rotary_dim / 2) float32")
    return dev


def _side(x, y, w, pos, dy=None, dw=None):
    sb, st, sh, _ = x.stride()
    B, L, H, _ = x.shape
    if (sb | st | sh) & 7:  # the library wants strides of whole 16 bytes; one of a dim of one is not used
        sb, st, sh = sb if B > 1 else 0, st if L > 1 else 0, sh if H > 1 else 0
    return _lib.ROPE_SIDE.pack(x.data_ptr(), 0 if dy is None else dy.data_ptr(), y.data_ptr(),
                               0 if w is None else w.data_ptr(), 0 if pos is None else pos.data_ptr(),
                               0 if dw is None else dw.data_ptr(), sb, st, sh, L, H)


def _tables(q, cos, sin, eps, interleaved):
    """The arguments after the two sides."""
    flags = (_INTERLEAVED if interleaved else 0) | (_NO_NORM if eps is None else 0)
    B, _, _, D = q.shape
    if cos is None:
        return None, None, 0, 0, B, D, eps or 0.0, _lib.dtype_code(q.dtype), flags
    P, half = cos.shape
    return cos.data_ptr(), sin.data_ptr(), P, 2 * half, B, D, eps or 0.0, _lib.dtype_code(q.dtype), flags


def _forward(q, k, qw, kw, cos, sin, q_pos, k_pos, eps, interleaved):
    q = _lib.rows16(q)
    yq = q.new_empty(q.shape)
    qs, ks, yk = _side(q, yq, qw, q_pos), None, None
    if k is not None:
        k = _lib.rows16(k)
        yk = k.new_empty(k.shape)
        ks = _side(k, yk, kw, k_pos)
    _lib.check(_lib.load().hclsm_qk_norm_rope(qs, ks, *_tables(q, cos, sin, eps, interleaved),
                                              _lib.stream_ptr(q.device)), "hclsm_qk_norm_rope")
    return q, k, yq, yk


def _dense_grad(g):
    return g if g.is_contiguous() and g.data_ptr() % 16 == 0 else g.clone(memory_format=torch.contiguous_format)


def _backward(q, k, qw, kw, cos, sin, q_pos, k_pos, eps, interleaved, gq, gk, want_qw, want_kw):
    dk = dqw = dkw = ks = ws = None
    gq, dq = _dense_grad(gq), q.new_empty(q.shape)
    if qw is not None and want_qw:
        dqw = qw.new_empty(qw.shape)
    qs = _side(q, dq, qw, q_pos, gq, dqw)
    if k is not None:
        gk, dk = _dense_grad(gk), k.new_empty(k.shape)
        if kw is not None and want_kw:
            dkw = kw.new_empty(kw.shape)
        ks = _side(k, dk, kw, k_pos, gk, dkw)
    lib, n = _lib.load(), 0
    if dqw is not None or dkw is not None:
        n = lib.hclsm_qk_norm_rope_bwd_workspace_size(q.shape[3])
        ws = q.new_empty(n, dtype=torch.uint8)
    _lib.check(lib.hclsm_qk_norm_rope_bwd(qs, ks, *_tables(q, cos, sin, eps, interleaved),
                                          None if ws is None else ws.data_ptr(), n, _lib.stream_ptr(q.device)),
               "hclsm_qk_norm_rope_bwd")
    return dq, dk, dqw, dkw


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, qw, kw, cos, sin, q_pos, k_pos, eps, interleaved):
        q, k, yq, yk = _forward(q, k, qw, kw, cos, sin, q_pos, k_pos, eps, interleaved)
        ctx.save_for_backward(q, k, qw, kw, cos, sin, q_pos, k_pos)
        ctx.eps, ctx.interleaved = eps, interleaved
        return yq, yk

    @staticmethod
    def backward(ctx, gq, gk):
        _lib.no_double_backward()
        want = ctx.needs_input_grad
        return (*_backward(*ctx.saved_tensors, ctx.eps, ctx.interleaved, gq, gk, want[2], want[3]), None, None, None,
                None, None, None)


def _prepare(q, k, q_weight, k_weight, cos, sin, q_pos, k_pos, eps, interleaved):
    """The checked arguments of the kernels."""
    dev = _check(q, k, q_weight, k_weight, cos, sin, eps)
    if cos is not None:
        cos, sin = _dense16(cos), _dense16(sin)
        rot = 2 * cos.shape[1]
        if rot > q.shape[3] or rot % (8 if interleaved else 16):
            raise ValueError(f"rotary_dim {rot} must be a multiple of {8 if interleaved else 16} up to head_dim")
    B, Lq = q.shape[:2]
    if cos is not None:
        q_pos = _lib.index32(q_pos, (B, Lq), "q_pos", dev)
        if q_pos is None and Lq > cos.shape[0]:
            raise ValueError(f"{Lq} query positions, tables of {cos.shape[0]}")
        if k is not None:
            k_pos = _lib.index32(k_pos, (B, k.shape[1]), "k_pos", dev)
            if k_pos is None and k.shape[1] > cos.shape[0]:
                raise ValueError(f"{k.shape[1]} key positions, tables of {cos.shape[0]}")
    else:
        q_pos = k_pos = None
    if k is None:
        k_pos = None
    if q_weight is not None:
        q_weight = q_weight.contiguous()
    if k_weight is not None:
        k_weight = k_weight.contiguous()
    return q, k, q_weight, k_weight, cos, sin, q_pos, k_pos, None if eps is None else float(eps), bool(interleaved)


def rope_fwd(q, k, q_weight, k_weight, cos, sin, q_pos, k_pos, eps, interleaved):
    """(q', k') without autograd."""
    return _forward(*_prepare(q, k, q_weight, k_weight, cos, sin, q_pos, k_pos, eps, interleaved))[2:]


def rope_bwd(q, k, q_weight, k_weight, cos, sin, q_pos, k_pos, eps, interleaved, gq, gk):
    """(dq, dk, dq_weight, dk_weight), None for weights that are not there."""
    args = list(_prepare(q, k, q_weight, k_weight, cos, sin, q_pos, k_pos, eps, interleaved))
    gq = _lib.like(gq, q.shape, q.dtype, "gq", q.device)
    if k is not None:
        gk = _lib.like(gk, k.shape, k.dtype, "gk", k.device)
    args[:2] = [None if t is None else _lib.rows16(t) for t in args[:2]]
    return _backward(*args, gq, gk, True, True)


def qk_norm_rope(q, k=None, q_weight=None, k_weight=None, cos=None, sin=None, *, q_pos=None, k_pos=None, eps=1e-6,
                 interleaved: bool = False):
    """(q', k') with every head normalised by its root mean square, weighted and
    rotated; k may be None (queries alone), and so may the weights and the tables.

    ``q_pos`` (B, Lq) and ``k_pos`` (B, Lk): rows of ``cos`` / ``sin``
    (positions, rotary_dim / 2), default 0, 1, 2, ...; a position outside the
    tables gives NaN in that token's rotated dims and sets the device error word.
    ``eps=None`` leaves the norm out.  Pairs are dims (i, i + rotary_dim / 2), or
    (2 i, 2 i + 1) with ``interleaved``; rotary_dim is a multiple of 16 (8
    interleaved).  Differentiable in q, k and the weights; rows of q and k may be
    strided (each head dense).
    """
    args = _prepare(q, k, q_weight, k_weight, cos, sin, q_pos, k_pos, eps, interleaved)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args[:4]):
        return _QkNormRope.apply(*args)
    return _forward(*args)[2:]
