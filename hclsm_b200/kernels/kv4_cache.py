"""A paged cache of keys and values in 4 bits, and the attention that reads it.

Every token is quantised by itself when it is written (groups of 32 dims share
a bf16 scale: 4.5 bits a value), so tokens come in any order and pages of
many sequences lie in one pool.  ``page_slots`` says where tokens go; tables
and lengths are arguments, so a step captures into a CUDA graph and can be replayed
with others.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch
from torch import Tensor

from .. import _lib

__all__ = ["Kv4Cache", "kv4_write", "kv4_read", "kv4_attention"]


@dataclass(init=False)
class Kv4Cache:
    """The cache's tensors, all contiguous: k, v (pages, Hkv, page, D / 2) uint8, k_scale, v_scale (pages, Hkv, page,
    D / 32) bfloat16; dtype (float32 or bfloat16) of the states that are written and read.  D is 32, 64, 96 or 128; page
    16, 32, 64 or 128."""

    k: Tensor
    v: Tensor
    k_scale: Tensor
    v_scale: Tensor
    dtype: torch.dtype = torch.bfloat16

    def __init__(self, k, v, k_scale, v_scale, dtype=torch.bfloat16):
        self.k, self.v, self.k_scale, self.v_scale, self.dtype = k, v, k_scale, v_scale, dtype
        self._args()

    def _args(self):
        """(hclsm_kv4_cache, Hkv, page, D, device, its index) for a call, from the tensors as they are now: nothing is kept,
        since a tensor that is changed in place (resize_, transpose_, its data) may stay at its address."""
        k, v, ks, vs = self.k, self.v, self.k_scale, self.v_scale
        dev, index = _lib.require_cuda(k), k.get_device()
        if v.get_device() != index or ks.get_device() != index or vs.get_device() != index:
            _lib.require_cuda(k, v, ks, vs)
        whole = k.shape
        if len(whole) != 4:
            raise ValueError("k must be (pages, Hkv, page, D / 2)")
        P, Hkv, page, half = whole
        D = 2 * half
        if page not in (16, 32, 64, 128) or D not in (32, 64, 96, 128) or Hkv < 1:
            raise ValueError(f"page must be 16, 32, 64 or 128 and head_dim 32, 64, 96 or 128, got {page} and {D}")
        if P * page >= 1 << 31:
            raise ValueError(f"{P} pages of {page} tokens pass 31 bits")
        shape = (P, Hkv, page, D // 32)
        if (v.shape != whole or k.dtype != torch.uint8 or v.dtype != torch.uint8 or not k.is_contiguous()
                or not v.is_contiguous()):
            raise ValueError(f"k and v must be contiguous {tuple(whole)} uint8")
        if (ks.shape != shape or vs.shape != shape or ks.dtype != torch.bfloat16 or vs.dtype != torch.bfloat16
                or not ks.is_contiguous() or not vs.is_contiguous()):
            raise ValueError(f"k_scale and v_scale must be contiguous {shape} bfloat16")
        return (_lib.KV4_CACHE.pack(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), P, Hkv, page, D,
                                    _lib.dtype_code(self.dtype)), Hkv, page, D, dev, index)

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int, *, page: int = 32, dtype=torch.bfloat16,
              device="cuda") -> "Kv4Cache":
        """A pool of ``pages`` pages of ``page`` tokens."""
        def zeros(width, dt):
            return torch.zeros(pages, kv_heads, page, width, dtype=dt, device=device)

        return cls(zeros(head_dim // 2, torch.uint8), zeros(head_dim // 2, torch.uint8),
                   zeros(head_dim // 32, torch.bfloat16), zeros(head_dim // 32, torch.bfloat16), dtype)

    @property
    def page(self) -> int:
        return self.k.shape[2]


def _no_derivatives(what, cache, *tensors):
    if torch.is_grad_enabled() and (cache.k_scale.requires_grad or cache.v_scale.requires_grad
                                    or any(t.requires_grad for t in tensors)):
        raise NotImplementedError(f"{what} has no gradients: call it under torch.no_grad()")
    if _lib.in_dual_level():
        _lib.no_tangents(cache.k_scale, cache.v_scale, *tensors)


def _table(table, dev):
    if table.dim() != 2:
        raise ValueError("table must be (B, pages of an entry)")
    return _lib.index32(table, tuple(table.shape), "table", dev)


def kv4_write(cache: Kv4Cache, k: Tensor, v: Tensor, slots: Tensor) -> None:
    """k, v (B, n, Hkv, D) into the cache, in place: token i of entry b goes to place slots[b, i] % page of page
    slots[b, i] // page (``page_slots`` makes them).  Negative slots are left out; one behind the cache is left out and
    sets the device error word.  The slots of one call must differ: of tokens that share one, what is kept is
    undefined.  No gradients: k and v that require them are refused."""
    _no_derivatives("kv4_write", cache, k, v)
    c, Hkv, _, D, dev, index = cache._args()
    if k.get_device() != index or v.get_device() != index:
        raise ValueError(f"k and v must be on {dev}, got {k.device} and {v.device}")
    if k.dim() != 4 or v.shape != k.shape or k.shape[2:] != (Hkv, D):
        raise ValueError(f"k and v must be (B, tokens, {Hkv}, {D}), got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype != cache.dtype or v.dtype != cache.dtype:
        raise TypeError(f"k and v must have the cache's dtype {cache.dtype}, got {k.dtype} and {v.dtype}")
    B, n = k.shape[:2]
    slots = _lib.index32(slots, (B, n), "slots", dev)
    if slots is None:
        raise ValueError("slots is required")
    k, v = _lib.rows16(k), _lib.rows16(v)
    _lib.check(_lib.load().hclsm_kv4_write(c, _lib.VIEW.pack(*_lib.view_args(k)), _lib.VIEW.pack(*_lib.view_args(v)),
                                           slots.data_ptr(), B, n, _lib.stream_ptr(dev)), "hclsm_kv4_write")
    _lib.changed(cache.k, cache.v, cache.k_scale, cache.v_scale)


def kv4_read(cache: Kv4Cache, table: Tensor, lens: Tensor | None = None):
    """(k, v), each (B, T, Hkv, D) in the cache's dtype with T = page * table.shape[1]: the first ``lens[b]`` tokens
    (default all; clamped to [0, T]) of the pages that table (B, T / page) names, as the values they stand for,
    zeros after them.  A page outside the cache below the length reads as zeros and sets the device error word."""
    _no_derivatives("kv4_read", cache)
    c, Hkv, page, D, dev, _ = cache._args()
    table = _table(table, dev)
    B, M = table.shape
    lens = _lib.index32(lens, (B,), "lens", dev)
    k, v = (torch.empty(B, M * page, Hkv, D, dtype=cache.dtype, device=dev) for _ in range(2))
    _lib.check(_lib.load().hclsm_kv4_read(c, table.data_ptr(), B, M, k.data_ptr(), v.data_ptr(), _lib.ptr(lens),
                                          _lib.stream_ptr(dev)), "hclsm_kv4_read")
    return k, v


def kv4_attention(q: Tensor, cache: Kv4Cache, table: Tensor, lens: Tensor | None = None, *,
                  scale: float | None = None) -> Tensor:
    """softmax(scale q k^T) v of q (B, Lq, H, D), in the cache's dtype, over the first ``lens[b]`` tokens (default all;
    clamped to the table's) of the pages that table (B, M) names; H is a multiple of Hkv.  An entry without tokens
    gives zeros; tokens of a page outside the cache do not count and set the device error word.
    Weights of up to 2^8 times values are summed in fp32 before they are divided by the weights' sum: values
    above some 2^119 over the number of tokens overflow.  No gradients."""
    _no_derivatives("kv4_attention", cache, q)
    c, Hkv, _, D, dev, index = cache._args()
    if q.get_device() != index:
        raise ValueError(f"q must be on {dev}, got {q.device}")
    table = _table(table, dev)
    B, M = table.shape
    if q.dim() != 4 or q.shape[0] != B or q.shape[3] != D:
        raise ValueError(f"q must be ({B}, tokens, heads, {D}), got {tuple(q.shape)}")
    Lq, H = q.shape[1], q.shape[2]
    if H < 1 or H % Hkv:
        raise ValueError(f"query heads ({H}) must be a multiple of key heads ({Hkv})")
    if q.dtype != cache.dtype:
        raise TypeError(f"q must have the cache's dtype {cache.dtype}, got {q.dtype}")
    scale = D ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    lens = _lib.index32(lens, (B,), "lens", dev)
    q = _lib.rows16(q)
    o = _lib.empty_like(q)
    lib, ws = _lib.load(), None
    n = lib.hclsm_kv4_attn_workspace_size(c, B, M, Lq, H)
    if n:
        ws = q.new_empty(n, dtype=torch.uint8)
    _lib.check(lib.hclsm_kv4_attn(c, table.data_ptr(), B, M, _lib.VIEW.pack(*_lib.view_args(q)), o.data_ptr(),
                                  _lib.ptr(lens), Lq, H, scale, _lib.ptr(ws), n, _lib.stream_ptr(dev)),
               "hclsm_kv4_attn")
    return o
