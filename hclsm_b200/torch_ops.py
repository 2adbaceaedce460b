"""The library's entry points as PyTorch dispatcher operators (``torch.ops.hclsm_b200.*``).

Registered with ``torch.library.custom_op``: each op validates its inputs,
allocates outputs on the current device and stream, calls the C ABI, and turns
a status code into ``ValueError`` / ``NotImplementedError`` / ``RuntimeError``.
CUDA tensors only (no CPU kernel is registered).  Every op has a fake
(shape-only) implementation, so ``torch.compile`` can trace through them, and
``ssm_scan_fwd`` has a registered autograd formula:

* ``ssm_scan_fwd(x, dt, A_log, B, C, D, z, flags, keep_states) -> (y, states)``
  (hclsm/kernels/ssm_scan_kernel.py:394 ``ssm_scan_fn``); ``flags`` as the C
  ABI's (1 clamped arithmetic, 2 softplus of a raw dt); ``states`` holds the
  forward's snapshots for the backward when ``keep_states`` and the path
  applies, else it is empty;
* ``ssm_scan_bwd(x, dt, A_log, B, C, dy, D, z, flags, states)
  -> [dx, ddt, dA_log, dB, dC, dD, dz]`` (empty tensors for absent D / z);
* ``slot_attn_core(Q, K, V, scale, clamp, eps, return_attn) -> (out, attn)``
  (slot_attention_kernel.py:265-291, forward);
* ``event_compact(mask) -> (idx, pos, counts, meta)``,
  ``event_gather(states, idx, counts, meta, n_frames, pad_k)``,
  ``event_scatter(states, upd, pos, counts, pad_k)``,
  ``event_mha(qkv, key_pad, frames, T, H, HD, scale)``
  (sparse_event_attn.py:93-188, level1_event.py:33-54);
* ``qk_norm_rope_fwd`` / ``qk_norm_rope_bwd`` and ``cross_attention_fwd`` /
  ``cross_attention_bwd`` (both forwards with registered autograd formulas; of the
  cross attention's outputs o alone has gradients), and
  ``kv8_write`` / ``kv8_attention`` on the tensors of a ``Kv8Cache``
  (``kv8_write`` mutates them, and wants detached keys and values).

Scan inputs must already share one dtype (fp32 or bf16: x, dt, B, C, z) with
A_log and D in fp32, and be contiguous; ``hclsm_b200.kernels.ssm_scan`` does
that preparation for Python callers.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch
from torch import Tensor

from . import _lib
from .kernels import kv8_cache as _kv8
from .kernels import sparse_event_attn as _ev
from .kernels import ssm_scan_kernel as _scan
from .kernels.cross_attn import attention_bwd as _xattn_bwd
from .kernels.cross_attn import attention_fwd as _xattn_fwd
from .kernels.qk_rope import rope_bwd as _rope_bwd
from .kernels.qk_rope import rope_fwd as _rope_fwd
from .kernels.slot_attention_kernel import slot_attention_core as _slot_core

__all__ = ["ssm_scan_fwd", "ssm_scan_bwd", "slot_attn_core", "event_compact", "event_gather", "event_scatter",
           "event_mha", "qk_norm_rope_fwd", "qk_norm_rope_bwd", "cross_attention_fwd", "cross_attention_bwd",
           "kv8_write", "kv8_attention"]

_NS = "hclsm_b200"


def _check_scan(x, dt, A_log, B, C, D, z):
    _lib.require_cuda(x, dt, A_log, B, C, D, z)
    io = x.dtype
    if io not in (torch.float32, torch.bfloat16):
        raise ValueError("ssm_scan: x must be float32 or bfloat16")
    for name, t in (("dt", dt), ("B", B), ("C", C), ("z", z)):
        if t is not None and t.dtype != io:
            raise ValueError(f"ssm_scan: {name} must have x's dtype ({io})")
    if A_log.dtype != torch.float32 or (D is not None and D.dtype != torch.float32):
        raise ValueError("ssm_scan: A_log and D must be float32")
    for t in (x, dt, A_log, B, C, D, z):
        if t is not None and not t.is_contiguous():
            raise ValueError("ssm_scan: inputs must be contiguous")
    _scan._check_shapes(x, dt, A_log, B, C, D, z)


@torch.library.custom_op(f"{_NS}::ssm_scan_fwd", mutates_args=())
def ssm_scan_fwd(x: Tensor, dt: Tensor, A_log: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor],
                 z: Optional[Tensor], flags: int, keep_states: bool) -> Tuple[Tensor, Tensor]:
    _check_scan(x, dt, A_log, B, C, D, z)
    nseq, L, Dn = x.shape
    nb = _scan.states_bytes(nseq, L, Dn, B.shape[-1], x.dtype) if keep_states else 0
    states = torch.empty(nb, dtype=torch.uint8, device=x.device)
    y = _scan.scan_fwd_raw(x, dt, A_log, B, C, D, z, clamp=bool(flags & 1), dt_softplus=bool(flags & 2),
                           states=states if nb > 0 else None)
    return y, states


@ssm_scan_fwd.register_fake
def _(x, dt, A_log, B, C, D, z, flags, keep_states):
    nseq, L, Dn = x.shape
    nb = _scan.states_bytes(nseq, L, Dn, B.shape[-1], x.dtype) if keep_states else 0  # a host-side query
    return torch.empty_like(x), x.new_empty(nb, dtype=torch.uint8)


@torch.library.custom_op(f"{_NS}::ssm_scan_bwd", mutates_args=())
def ssm_scan_bwd(x: Tensor, dt: Tensor, A_log: Tensor, B: Tensor, C: Tensor, dy: Tensor, D: Optional[Tensor],
                 z: Optional[Tensor], flags: int, states: Tensor) -> List[Tensor]:
    _check_scan(x, dt, A_log, B, C, D, z)
    dy = dy.to(x.dtype).contiguous()
    g = _scan.scan_bwd_raw(x, dt, A_log, B, C, dy, D, z, clamp=bool(flags & 1), dt_softplus=bool(flags & 2),
                           states=states if states.numel() > 0 else None)
    # absent gradients as distinct empty tensors (outputs may not alias)
    return [g[0], g[1], g[2], g[3], g[4], g[5] if g[5] is not None else x.new_empty(0),
            g[6] if g[6] is not None else x.new_empty(0)]


@ssm_scan_bwd.register_fake
def _(x, dt, A_log, B, C, dy, D, z, flags, states):
    return [torch.empty_like(x), torch.empty_like(x), torch.empty_like(A_log), torch.empty_like(B),
            torch.empty_like(C), torch.empty_like(D) if D is not None else x.new_empty(0),
            torch.empty_like(z) if z is not None else x.new_empty(0)]


def _scan_setup(ctx, inputs, output):
    x, dt, A_log, B, C, D, z, flags, keep_states = inputs
    ctx.save_for_backward(x, dt, A_log, B, C, D, z, output[1])
    ctx.flags = flags


def _scan_backward(ctx, gy, gstates):
    x, dt, A_log, B, C, D, z, states = ctx.saved_tensors
    g = ssm_scan_bwd(x, dt, A_log, B, C, gy, D, z, ctx.flags, states)
    return (g[0], g[1], g[2], g[3], g[4], g[5] if D is not None else None, g[6] if z is not None else None,
            None, None)


torch.library.register_autograd(f"{_NS}::ssm_scan_fwd", _scan_backward, setup_context=_scan_setup)


@torch.library.custom_op(f"{_NS}::slot_attn_core", mutates_args=())
def slot_attn_core(Q: Tensor, K: Tensor, V: Tensor, scale: float, clamp: float, eps: float,
                   return_attn: bool) -> Tuple[Tensor, Tensor]:
    out, attn = _slot_core(Q, K, V, scale, clamp=clamp, eps=eps, return_attn=return_attn)
    return out, attn if attn is not None else out.new_empty(0)


@slot_attn_core.register_fake
def _(Q, K, V, scale, clamp, eps, return_attn):
    dt = torch.bfloat16 if {Q.dtype, K.dtype, V.dtype} == {torch.bfloat16} else torch.float32
    F, N, D = Q.shape
    out = Q.new_empty((F, N, D), dtype=dt)
    attn = Q.new_empty((F, N, K.shape[1]), dtype=torch.float32 if dt == torch.float32 else dt) if return_attn \
        else Q.new_empty(0, dtype=dt)
    return out, attn


@torch.library.custom_op(f"{_NS}::event_compact", mutates_args=())
def event_compact(mask: Tensor) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    _lib.require_cuda(mask)
    idx, pos, counts, meta = _ev.event_compact(mask)
    return idx, pos, counts, meta


@event_compact.register_fake
def _(mask):
    B, T = mask.shape
    i32 = torch.int32
    return (mask.new_empty(max(B * T, 1), dtype=i32), mask.new_empty(max(B * T, 1), dtype=i32),
            mask.new_empty(max(B, 1), dtype=i32), mask.new_empty(2, dtype=i32))


@torch.library.custom_op(f"{_NS}::event_gather", mutates_args=())
def event_gather(states: Tensor, idx: Tensor, counts: Tensor, meta: Tensor, n_frames: int, pad_k: int) -> Tensor:
    _lib.require_cuda(states, idx, counts, meta)
    return _ev.event_gather(states.contiguous(), idx, counts, meta, n_frames, pad_k=pad_k)


@event_gather.register_fake
def _(states, idx, counts, meta, n_frames, pad_k):
    B, T, N, D = states.shape
    return states.new_empty((n_frames, N, D))


@torch.library.custom_op(f"{_NS}::event_scatter", mutates_args=())
def event_scatter(states: Tensor, upd: Tensor, pos: Tensor, counts: Tensor, pad_k: int) -> Tensor:
    _lib.require_cuda(states, upd, pos, counts)
    return _ev.event_scatter(states.contiguous(), upd.to(states.dtype), pos, counts, pad_k=pad_k)


@event_scatter.register_fake
def _(states, upd, pos, counts, pad_k):
    return torch.empty_like(states)


@torch.library.custom_op(f"{_NS}::event_mha", mutates_args=())
def event_mha(qkv: Tensor, key_pad: Optional[Tensor], frames: int, T: int, H: int, HD: int, scale: float) -> Tensor:
    _lib.require_cuda(qkv, key_pad)
    if qkv.dtype not in (torch.float32, torch.bfloat16) or not qkv.is_contiguous():
        raise ValueError("event_mha: qkv must be contiguous float32 or bfloat16")
    kp = None if key_pad is None else key_pad.to(torch.uint8).contiguous()
    out = torch.empty(frames * T, H * HD, dtype=qkv.dtype, device=qkv.device)
    rc = _lib.load().hclsm_event_mha(_lib.ptr(qkv), _lib.ptr(kp), _lib.ptr(out), frames, T, H, HD, float(scale),
                                     _lib.dtype_code(qkv.dtype), _lib.stream_ptr(qkv.device))
    _lib.check(rc, "hclsm_event_mha")
    return out


@event_mha.register_fake
def _(qkv, key_pad, frames, T, H, HD, scale):
    return qkv.new_empty((frames * T, H * HD))


# ---- attention between sets of states ------------------------------------------------------------
@torch.library.custom_op(f"{_NS}::qk_norm_rope_fwd", mutates_args=())
def qk_norm_rope_fwd(q: Tensor, k: Tensor, q_weight: Optional[Tensor], k_weight: Optional[Tensor],
                     cos: Optional[Tensor], sin: Optional[Tensor], q_pos: Optional[Tensor], k_pos: Optional[Tensor],
                     eps: float, interleaved: bool) -> Tuple[Tensor, Tensor]:
    return _rope_fwd(q, k, q_weight, k_weight, cos, sin, q_pos, k_pos, eps, interleaved)


@qk_norm_rope_fwd.register_fake
def _(q, k, q_weight, k_weight, cos, sin, q_pos, k_pos, eps, interleaved):
    return q.new_empty(q.shape), k.new_empty(k.shape)


@torch.library.custom_op(f"{_NS}::qk_norm_rope_bwd", mutates_args=())
def qk_norm_rope_bwd(q: Tensor, k: Tensor, q_weight: Optional[Tensor], k_weight: Optional[Tensor],
                     cos: Optional[Tensor], sin: Optional[Tensor], q_pos: Optional[Tensor], k_pos: Optional[Tensor],
                     eps: float, interleaved: bool, gq: Tensor, gk: Tensor) -> List[Tensor]:
    g = _rope_bwd(q, k, q_weight, k_weight, cos, sin, q_pos, k_pos, eps, interleaved, gq, gk)
    return [q.new_empty(0, dtype=torch.float32) if t is None else t for t in g]


@qk_norm_rope_bwd.register_fake
def _(q, k, q_weight, k_weight, cos, sin, q_pos, k_pos, eps, interleaved, gq, gk):
    def w(t):
        return q.new_empty(0 if t is None else t.shape[0], dtype=torch.float32)

    return [q.new_empty(q.shape), k.new_empty(k.shape), w(q_weight), w(k_weight)]


def _rope_setup(ctx, inputs, output):
    if any(ctx.needs_input_grad[4:6]):
        raise NotImplementedError("qk_norm_rope_fwd has no gradients of cos and sin: detach them")
    ctx.save_for_backward(*inputs[:8])
    ctx.eps, ctx.interleaved = inputs[8:]


def _rope_backward(ctx, gq, gk):
    t = ctx.saved_tensors
    dq, dk, dqw, dkw = qk_norm_rope_bwd(*t, ctx.eps, ctx.interleaved, gq, gk)
    return (dq, dk, None if t[2] is None else dqw, None if t[3] is None else dkw) + (None,) * 6


torch.library.register_autograd(f"{_NS}::qk_norm_rope_fwd", _rope_backward, setup_context=_rope_setup)


@torch.library.custom_op(f"{_NS}::cross_attention_fwd", mutates_args=())
def cross_attention_fwd(q: Tensor, k: Tensor, v: Tensor, kv_lens: Optional[Tensor], key_mask: Optional[Tensor],
                        scale: float) -> Tuple[Tensor, Tensor, Tensor]:
    o, lse, lo = _xattn_fwd(q, k, v, kv_lens, key_mask, scale)
    return o, lse, q.new_empty(0) if lo is None else lo


@cross_attention_fwd.register_fake
def _(q, k, v, kv_lens, key_mask, scale):
    B, Lq, H, _ = q.shape
    return (q.new_empty(q.shape), q.new_empty((B, H, Lq), dtype=torch.float32),
            q.new_empty(q.shape if q.dtype == torch.bfloat16 else 0))


@torch.library.custom_op(f"{_NS}::cross_attention_bwd", mutates_args=())
def cross_attention_bwd(q: Tensor, k: Tensor, v: Tensor, o: Tensor, lse: Tensor, lo: Tensor, do: Tensor,
                        kv_lens: Optional[Tensor], key_mask: Optional[Tensor], scale: float) -> List[Tensor]:
    return list(_xattn_bwd(q, k, v, o, lse, lo if lo.numel() else None, do, kv_lens, key_mask, scale))


@cross_attention_bwd.register_fake
def _(q, k, v, o, lse, lo, do, kv_lens, key_mask, scale):
    return [t.new_empty(t.shape) for t in (q, k, v)]


def _xattn_setup(ctx, inputs, output):
    q, k, v, kv_lens, key_mask, scale = inputs
    ctx.save_for_backward(q, k, v, *output, kv_lens, key_mask)
    ctx.scale = scale
    ctx.set_materialize_grads(False)


def _xattn_backward(ctx, go, glse, glo):
    if glse is not None or glo is not None:
        raise NotImplementedError("cross_attention_fwd: only o has gradients; detach lse and lo")
    if go is None:
        return (None,) * 6
    q, k, v, o, lse, lo, kv_lens, key_mask = ctx.saved_tensors
    return (*cross_attention_bwd(q, k, v, o, lse, lo, go, kv_lens, key_mask, ctx.scale), None, None, None)


torch.library.register_autograd(f"{_NS}::cross_attention_fwd", _xattn_backward, setup_context=_xattn_setup)


@torch.library.custom_op(f"{_NS}::kv8_write",
                         mutates_args=("ck", "cv", "k_scale", "v_scale", "k_tail", "v_tail"))
def kv8_write(ck: Tensor, cv: Tensor, k_scale: Tensor, v_scale: Tensor, k_tail: Tensor, v_tail: Tensor, k: Tensor,
              v: Tensor, start: Tensor, count: Optional[Tensor]) -> None:
    if k.requires_grad or v.requires_grad:  # an operator that mutates has no autograd formula; grad mode is off here
        raise NotImplementedError("kv8_write has no gradients: detach k and v")
    _kv8.kv8_write(_kv8.Kv8Cache(ck, cv, k_scale, v_scale, k_tail, v_tail), k, v, start, count)


@kv8_write.register_fake
def _(ck, cv, k_scale, v_scale, k_tail, v_tail, k, v, start, count):
    return None


@torch.library.custom_op(f"{_NS}::kv8_attention", mutates_args=())
def kv8_attention(q: Tensor, ck: Tensor, cv: Tensor, k_scale: Tensor, v_scale: Tensor, k_tail: Tensor, v_tail: Tensor,
                  lens: Optional[Tensor], scale: float) -> Tensor:
    return _kv8.kv8_attention(q, _kv8.Kv8Cache(ck, cv, k_scale, v_scale, k_tail, v_tail), lens, scale=scale)


@kv8_attention.register_fake
def _(q, ck, cv, k_scale, v_scale, k_tail, v_tail, lens, scale):
    return q.new_empty(q.shape)
