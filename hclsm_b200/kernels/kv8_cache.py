"""A cache of keys and values in 8 bits, and the attention that reads it.

Complete blocks of ``block`` tokens a head are int8 with one fp32 scale
(max|x| / 127); the last, incomplete block of each sequence stays in the inputs'
dtype (its scale is -1), so every value is rounded to 8 bits once, when its block
fills.  The
caller owns the positions: ``start`` (tokens already there) and ``lens`` (tokens
to attend to) are arguments, so a step captures into a CUDA graph and can be
replayed with other positions.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch
from torch import Tensor

from .. import _lib

__all__ = ["Kv8Cache", "kv8_write", "kv8_read", "kv8_attention"]


@dataclass(init=False)
class Kv8Cache:
    """The cache's tensors, all contiguous: k, v (B, Hkv, T, D) int8, k_scale,
    v_scale (B, Hkv, T / block) fp32, k_tail, v_tail (B, Hkv, block, D) in the
    inputs' dtype.  D is 32, 64, 96 or 128; block 16, 32, 64 or 128."""

    k: Tensor
    v: Tensor
    k_scale: Tensor
    v_scale: Tensor
    k_tail: Tensor
    v_tail: Tensor

    def __init__(self, k, v, k_scale, v_scale, k_tail, v_tail):
        self.k, self.v, self.k_scale, self.v_scale, self.k_tail, self.v_tail = k, v, k_scale, v_scale, k_tail, v_tail
        self._args()

    def _args(self):
        """(hclsm_kv8_cache, (B, Hkv, T, D), dtype, device, its index) for a call, from the tensors as they are now: nothing
        is kept, since a tensor that is changed in place (resize_, transpose_, its data) may stay at its address."""
        k, v, ks, vs, kt, vt = self.k, self.v, self.k_scale, self.v_scale, self.k_tail, self.v_tail
        dev, index = _lib.require_cuda(k), k.get_device()
        if (v.get_device() != index or ks.get_device() != index or vs.get_device() != index or kt.get_device() != index
                or vt.get_device() != index):
            _lib.require_cuda(k, v, ks, vs, kt, vt)
        whole, tail, dtype = k.shape, kt.shape, kt.dtype
        if len(whole) != 4 or len(tail) != 4:
            raise ValueError("k must be (B, Hkv, T, D), k_tail (B, Hkv, block, D)")
        B, Hkv, T, D = whole
        block = tail[2]
        if block not in (16, 32, 64, 128) or T % block:
            raise ValueError(f"block must be 16, 32, 64 or 128 and divide the capacity {T}, got {block}")
        if D not in (32, 64, 96, 128):
            raise ValueError(f"head_dim must be 32, 64, 96 or 128, got {D}")
        if (v.shape != whole or k.dtype != torch.int8 or v.dtype != torch.int8 or not k.is_contiguous()
                or not v.is_contiguous()):
            raise ValueError(f"k and v must be contiguous {tuple(whole)} int8")
        shape = (B, Hkv, T // block)
        if (ks.shape != shape or vs.shape != shape or ks.dtype != torch.float32 or vs.dtype != torch.float32
                or not ks.is_contiguous() or not vs.is_contiguous()):
            raise ValueError(f"k_scale and v_scale must be contiguous {shape} float32")
        shape = (B, Hkv, block, D)
        if (tail != shape or vt.shape != shape or vt.dtype != dtype or not kt.is_contiguous()
                or not vt.is_contiguous()):
            raise ValueError(f"k_tail and v_tail must be contiguous {shape} of one dtype")
        return (_lib.KV8_CACHE.pack(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), kt.data_ptr(), vt.data_ptr(), B,
                                    Hkv, T, D, block, _lib.dtype_code(dtype)), (B, Hkv, T, D), dtype, dev, index)

    @classmethod
    def empty(cls, batch: int, capacity: int, kv_heads: int, head_dim: int, *, block: int = 32, dtype=torch.bfloat16,
              device="cuda") -> "Kv8Cache":
        """A cache with room for ``capacity`` tokens (rounded up to whole blocks) a sequence."""
        T = (capacity + block - 1) // block * block

        def full(value, *shape, dt):
            return torch.full(shape, value, dtype=dt, device=device)

        return cls(*(full(0, batch, kv_heads, T, head_dim, dt=torch.int8) for _ in range(2)),
                   *(full(-1.0, batch, kv_heads, T // block, dt=torch.float32) for _ in range(2)),
                   *(full(0, batch, kv_heads, block, head_dim, dt=dtype) for _ in range(2)))

    @property
    def dtype(self) -> torch.dtype:
        return self.k_tail.dtype

    @property
    def block(self) -> int:
        return self.k_tail.shape[2]


def _no_derivatives(what, cache, k=None, v=None):
    if torch.is_grad_enabled() and ((k is not None and k.requires_grad) or (v is not None and v.requires_grad)
                                    or cache.k_scale.requires_grad or cache.v_scale.requires_grad
                                    or cache.k_tail.requires_grad or cache.v_tail.requires_grad):
        raise NotImplementedError(f"{what} has no gradients: call it under torch.no_grad()")
    if _lib.in_dual_level():
        _lib.no_tangents(k, v, cache.k_scale, cache.v_scale, cache.k_tail, cache.v_tail)


def kv8_write(cache: Kv8Cache, k: Tensor, v: Tensor, start: Tensor, count: Tensor | None = None) -> None:
    """Append k, v (B, n, Hkv, D), in place: token i of entry b becomes token
    ``start[b] + i`` of the cache, for the first ``count[b]`` tokens (default n).
    ``start[b]`` is the number of tokens already there (or, to write anew from there, a
    multiple of the block: what was behind it is gone).  A request that does not
    fit the capacity writes nothing and sets the device error word.  No gradients:
    k and v that require them are refused."""
    _no_derivatives("kv8_write", cache, k, v)
    c, (B, Hkv, _, D), dtype, dev, index = cache._args()
    if k.get_device() != index or v.get_device() != index:
        raise ValueError(f"k and v must be on {dev}, got {k.device} and {v.device}")
    if k.dim() != 4 or v.shape != k.shape or k.shape[0] != B or k.shape[2:] != (Hkv, D):
        raise ValueError(f"k and v must be ({B}, tokens, {Hkv}, {D}), got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype != dtype or v.dtype != dtype:
        raise TypeError(f"k and v must have the cache's dtype {dtype}, got {k.dtype} and {v.dtype}")
    start = _lib.index32(start, (B,), "start", dev)
    if start is None:
        raise ValueError("start is required")
    count = _lib.index32(count, (B,), "count", dev)
    k, v = _lib.rows16(k), _lib.rows16(v)
    _lib.check(_lib.load().hclsm_kv8_write(c, _lib.VIEW.pack(*_lib.view_args(k)),
                                           _lib.VIEW.pack(*_lib.view_args(v)), k.shape[1], start.data_ptr(),
                                           _lib.ptr(count), _lib.stream_ptr(dev)), "hclsm_kv8_write")
    _lib.changed(cache.k, cache.v, cache.k_scale, cache.v_scale, cache.k_tail, cache.v_tail)


def kv8_read(cache: Kv8Cache, lens: Tensor | None = None):
    """(k, v), each (B, T, Hkv, D) in the cache's dtype: the first ``lens[b]``
    tokens written (default all) as the values they stand for, zeros after them."""
    _no_derivatives("kv8_read", cache)
    c, (B, Hkv, T, D), dtype, dev, _ = cache._args()
    lens = _lib.index32(lens, (B,), "lens", dev)
    k, v = (torch.empty(B, T, Hkv, D, dtype=dtype, device=dev) for _ in range(2))
    _lib.check(_lib.load().hclsm_kv8_read(c, k.data_ptr(), v.data_ptr(), _lib.ptr(lens),
                                          _lib.stream_ptr(dev)), "hclsm_kv8_read")
    return k, v


def kv8_attention(q: Tensor, cache: Kv8Cache, lens: Tensor | None = None, *, scale: float | None = None) -> Tensor:
    """softmax(scale q k^T) v of q (B, Lq, H, D), in the cache's dtype, over the
    first ``lens[b]`` tokens written (default all of the capacity; clamped to [0, T]); H
    is a multiple of Hkv.  An entry without tokens gives zeros.  No gradients."""
    _no_derivatives("kv8_attention", cache, q)
    c, (B, Hkv, _, D), dtype, dev, index = cache._args()
    if q.get_device() != index:
        raise ValueError(f"q must be on {dev}, got {q.device}")
    if q.dim() != 4 or q.shape[0] != B or q.shape[3] != D:
        raise ValueError(f"q must be ({B}, tokens, heads, {D}), got {tuple(q.shape)}")
    Lq, H = q.shape[1], q.shape[2]
    if H < 1 or H % Hkv:
        raise ValueError(f"query heads ({H}) must be a multiple of key heads ({Hkv})")
    if q.dtype != dtype:
        raise TypeError(f"q must have the cache's dtype {dtype}, got {q.dtype}")
    scale = D ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    lens = _lib.index32(lens, (B,), "lens", dev)
    q = _lib.dense_last(q)
    o = q.new_empty(q.shape)
    lib, ws = _lib.load(), None
    n = lib.hclsm_kv8_attn_workspace_size(c, Lq, H)
    if n:
        ws = q.new_empty(n, dtype=torch.uint8)
    _lib.check(lib.hclsm_kv8_attn(c, _lib.VIEW.pack(*_lib.view_args(q)), o.data_ptr(), _lib.ptr(lens), Lq, H,
                                  scale, None if ws is None else ws.data_ptr(), n, _lib.stream_ptr(dev)),
               "hclsm_kv8_attn")
    return o
