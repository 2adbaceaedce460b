"""ctypes binding of ``libhclsm_b200.so`` (the C ABI declared in include/hclsm_b200.h).

The library is the only compute path: there is no CPU or PyTorch fallback.  A
missing library or a non-CUDA tensor raises.
"""
from __future__ import annotations

import ctypes
import os
import struct

import torch
from torch.autograd import forward_ad

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libhclsm_b200.so")

F32, BF16 = 0, 1
_STATUS = {
    1: (ValueError, "unsupported shape"),
    2: (TypeError, "unsupported dtype"),
    3: (ValueError, "misaligned pointer"),
    4: (ValueError, "workspace missing or too small"),
    5: (RuntimeError, "CUDA launch failed"),
    6: (RuntimeError, "device-side wait timed out"),
    7: (NotImplementedError, "input outside what this build supports"),
    8: (ValueError, "required pointer is NULL"),
}

_vp = ctypes.c_void_p
_i64 = ctypes.c_int64
_i32 = ctypes.c_int32
_sz = ctypes.c_size_t

# name -> (restype, argtypes)
SIGNATURES = {
    "hclsm_version": (ctypes.c_int, []),
    "hclsm_device_error": (ctypes.c_int, []),
    "hclsm_selftest_wait_timeout": (ctypes.c_int, [ctypes.c_uint32, _vp, _vp]),
    "hclsm_ssm_scan_fwd": (ctypes.c_int, [_vp] * 8 + [_i64, _i32, _i32, _i32, _i32, _i32, _vp]),
    "hclsm_ssm_scan_bwd_workspace_size": (_sz, [_i64, _i32, _i32, _i32]),
    "hclsm_ssm_scan_bwd": (ctypes.c_int, [_vp] * 15 + [_i64, _i32, _i32, _i32, _i32, _i32, _vp, _sz, _vp]),
    "hclsm_ssm_scan_states_size": (_sz, [_i64, _i32, _i32, _i32, _i32]),
    "hclsm_ssm_scan_fwd_states": (ctypes.c_int, [_vp] * 8 + [_i64, _i32, _i32, _i32, _i32, _i32, _vp, _sz, _vp]),
    "hclsm_ssm_scan_bwd_states": (ctypes.c_int, [_vp] * 15 + [_i64, _i32, _i32, _i32, _i32, _i32, _vp, _sz, _vp,
                                                              _sz, _vp]),
    "hclsm_l0_pool": (ctypes.c_int, [_vp, _i32, _vp, _vp, _i32, _i32, _i32, _i64, _vp]),
    "hclsm_l0_epilogue": (ctypes.c_int, [_vp, _i32, _vp, _vp, _i32, _i32, _i32, _i64, _vp]),
    "hclsm_l0_epilogue_bwd": (ctypes.c_int, [_vp, _i32, _vp, _vp, _i32, _vp, _i32, _i32, _i64, _vp]),
    "hclsm_slot_attn_core": (ctypes.c_int, [_vp] * 5 + [_i32] * 4 + [ctypes.c_float] * 3 + [_i32, _i32, _vp]),
    "hclsm_layernorm": (ctypes.c_int, [_vp] * 4 + [_i64, _i32, ctypes.c_float, _i32, _vp]),
    "hclsm_gru_cell": (ctypes.c_int, [_vp] * 6 + [_i64, _i32, _vp]),
    "hclsm_bias_act": (ctypes.c_int, [_vp] * 3 + [_i64, _i32, _i32, _i32, _vp]),
    "hclsm_residual_clamp": (ctypes.c_int, [_vp] * 5 + [_i64, _i32, ctypes.c_float, _vp]),
    "hclsm_event_detect": (ctypes.c_int, [_vp, _vp, _i32, _i32, _vp, _vp, _vp, _vp, _vp, _vp]),
    "hclsm_event_compact": (ctypes.c_int, [_vp, _i32, _i32, _i32] + [_vp] * 5),
    "hclsm_event_gather": (ctypes.c_int, [_vp] * 5 + [_i64, _i32, _i32, _i64, _i32, _vp]),
    "hclsm_event_scatter": (ctypes.c_int, [_vp] * 5 + [_i64, _i64, _i32, _i32, _i32, _vp]),
    "hclsm_event_mha": (ctypes.c_int, [_vp] * 3 + [_i32] * 4 + [ctypes.c_float, _i32, _vp]),
    "hclsm_swiglu": (ctypes.c_int, [_vp, _i32, _vp, _i64, _i32, _i32, _vp]),
    "hclsm_slot_attn_iter_workspace_size": (_sz, [_i32] * 3),
    "hclsm_slot_attn_iter": (ctypes.c_int, [_vp] * 6 + [_i32] * 4 + [_vp, _sz, _vp]),
    "hclsm_gru_cell_ln": (ctypes.c_int, [_vp, _vp, _i32] + [_vp] * 7 + [_i32, _i64, _i32, ctypes.c_float, _vp]),
    "hclsm_residual_clamp_ln": (ctypes.c_int, [_vp, _vp, _i32] + [_vp] * 6 + [_i32, _i64, _i32, ctypes.c_float,
                                                                           ctypes.c_float, _vp]),
    "hclsm_colsum_workspace_size": (_sz, [_i32]),
    "hclsm_colsum": (ctypes.c_int, [_vp, _vp, _i64, _i32, _vp, _sz, _vp]),
    "hclsm_layernorm_bwd_workspace_size": (_sz, [_i64, _i32]),
    "hclsm_layernorm_bwd": (ctypes.c_int, [_vp] * 6 + [_i64, _i32, ctypes.c_float, _i32, _vp, _sz, _vp]),
    "hclsm_gru_cell_bwd": (ctypes.c_int, [_vp] * 9 + [_i64, _i32, _vp]),
    "hclsm_slot_softmax_bwd": (ctypes.c_int, [_vp] * 4 + [_i32] * 3 + [ctypes.c_float] * 3 + [_i32, _vp]),
    "hclsm_residual_clamp_bwd": (ctypes.c_int, [_vp] * 5 + [_i64, _i32, ctypes.c_float, _vp]),
    "hclsm_relu_bwd": (ctypes.c_int, [_vp, _i32, _vp, _vp, _i32, _i64, _vp]),
    "hclsm_swiglu_bwd": (ctypes.c_int, [_vp, _vp, _vp, _i64, _i32, _i32, _vp]),
    "hclsm_event_mha_bwd": (ctypes.c_int, [_vp] * 4 + [_i32] * 4 + [ctypes.c_float, _i32, _vp]),
    "hclsm_qk_norm_rope": (ctypes.c_int, [_vp] * 4 + [_i32, _i32, _i64, _i32, ctypes.c_float, _i32, _i32, _vp]),
    "hclsm_qk_norm_rope_bwd_workspace_size": (_sz, [_i32]),
    "hclsm_qk_norm_rope_bwd": (ctypes.c_int, [_vp] * 4 + [_i32, _i32, _i64, _i32, ctypes.c_float, _i32, _i32, _vp,
                                                          _sz, _vp]),
    "hclsm_xattn_fwd_workspace_size": (_sz, [_vp]),
    "hclsm_xattn_fwd": (ctypes.c_int, [_vp, _vp, _sz, _vp]),
    "hclsm_xattn_bwd_workspace_size": (_sz, [_vp]),
    "hclsm_xattn_bwd": (ctypes.c_int, [_vp, _vp, _sz, _vp]),
    "hclsm_kv8_write": (ctypes.c_int, [_vp] * 3 + [_i32] + [_vp] * 3),
    "hclsm_kv8_read": (ctypes.c_int, [_vp] * 5),
    "hclsm_kv8_attn_workspace_size": (_sz, [_vp, _i32, _i32]),
    "hclsm_kv8_attn": (ctypes.c_int, [_vp] * 4 + [_i32, _i32, ctypes.c_float, _vp, _sz, _vp]),
    "hclsm_ssm_scan_bwd_noalloc_max_scratch": (_sz, []),
    "hclsm_ssm_scan_bwd_noalloc": (ctypes.c_int, [_vp] * 15 + [_i64, _i32, _i32, _i32, _i32, _i32, _vp]),
}


# The argument structs of include/hclsm_b200.h, packed with the C layout (a bytes object
# passes as a pointer; several times cheaper to make than a ctypes.Structure).
VIEW = struct.Struct("@Pqqq")                     # hclsm_view
ROPE_SIDE = struct.Struct("@6P3q2i")              # hclsm_rope_side
XATTN_ARGS = struct.Struct("@" + 4 * "Pqqq" + "8Pq7if")  # hclsm_xattn_args
KV8_CACHE = struct.Struct("@6P6i")                # hclsm_kv8_cache


class SlotIterWeights(ctypes.Structure):
    """hclsm_slot_iter_weights (include/hclsm_b200.h)."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("wq_t", "w_ih_t", "w_hh_t", "b_ih", "b_hh", "w1_t", "b1", "w2_t", "b2",
                                                "ln_attn_w", "ln_attn_b", "ln_mlp_w", "ln_mlp_b")]


_lib = None


def load() -> ctypes.CDLL:
    """Load the library (building nothing); raise if it is absent."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"hclsm_b200: native library {LIB_PATH} is missing; build it with "
                "`python -m hclsm_b200.build` (there is no fallback path)")
        lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


def check(rc: int, what: str) -> None:
    if rc != 0:
        exc, msg = _STATUS.get(rc, (RuntimeError, f"status {rc}"))
        raise exc(f"{what}: {msg} (hclsm status {rc})")


def ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


_get_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def stream_ptr(device) -> int:
    """The current stream of a CUDA device as an integer (a tensor's device has an index; the
    raw query skips the Stream object, about 3 us a call).  Kernels launch on the current
    device, so it has to be the tensors' one."""
    index = device.index
    if index is not None and index != _get_device():
        raise ValueError(f"hclsm_b200: tensors on {device}, current device cuda:{_get_device()}: call "
                         "torch.cuda.set_device or use torch.cuda.device")
    if _raw_stream is not None and index is not None:
        return _raw_stream(index)
    return torch.cuda.current_stream(device).cuda_stream


def dtype_code(dt: torch.dtype) -> int:
    if dt == torch.float32:
        return F32
    if dt == torch.bfloat16:
        return BF16
    raise TypeError(f"hclsm_b200: dtype {dt} not supported (float32 or bfloat16)")


def require_cuda(*tensors) -> torch.device:
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("hclsm_b200 ops run on CUDA tensors only (no CPU fallback)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError("hclsm_b200: all tensors must be on the same device")
    return dev


def dense_last(t):
    """t itself if its last dim is dense, else a contiguous copy."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def rows16(t):
    """The (B, L, H, D) tensor itself if its last dim is dense and every row starts on 16
    bytes, else an aligned contiguous copy.  The stride of a dim of one says nothing (the
    kernels do not use it): torch keeps any there, through contiguous() and clone() too."""
    sb, st, sh, sd = t.stride()
    if sd == 1 and t.data_ptr() % 16 == 0:
        e = t.element_size()
        if (sb | st | sh) * e % 16 == 0 or all(n == 1 or s * e % 16 == 0 for n, s in zip(t.shape[:3], (sb, st, sh))):
            return t
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def view_args(t):
    """The fields of hclsm_view for a (B, L, H, D) tensor."""
    sb, st, sh, _ = t.stride()
    return t.data_ptr(), sb, st, sh


def index32(t, shape, name, device):
    """An int32, contiguous index tensor of that shape on that device (int64 is converted), or None."""
    if t is None:
        return None
    if t.dtype != torch.int32:
        if t.dtype != torch.int64:
            raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")
        t = t.clamp(-(1 << 31), (1 << 31) - 1).to(torch.int32)  # out of range stays out of range
    if t.shape != shape:
        raise ValueError(f"{name} must be {shape}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")
    return t if t.is_contiguous() else t.contiguous()


def like(t, shape, dtype, name, device):
    """t, which a kernel takes to be a tensor of that shape, dtype and device; dense."""
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")
    return t if t.is_contiguous() else t.contiguous()


def in_dual_level() -> bool:
    """Whether a tensor can have a forward-mode tangent at all."""
    return getattr(forward_ad, "_current_level", 0) >= 0


def no_tangents(*tensors):
    """A forward-mode derivative (torch.autograd.forward_ad) is refused: the kernels would drop the tangents."""
    if not in_dual_level():
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("hclsm_b200: this operator has no forward-mode derivative")


def no_double_backward():
    """A backward made of this library's kernels has no graph of its own."""
    if torch.is_grad_enabled():
        raise RuntimeError("hclsm_b200: this operator has no second derivative (create_graph=True)")
