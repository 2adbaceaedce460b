"""Per-head norm with rotation, cross attention and the 8-bit state cache against
their definitions in 64 bits, at the sizes, masks and layouts where they can go
wrong, and their refusals.

Errors are 2-norms relative to the result's.  Tolerances: bf16 rounds to nearest
with unit roundoff u = 2^-8.  A norm's output is rounded once (u).  An attention
output sees the weights' rounding and its own (2 u); its gradients three at most:
the weights' (or their gradients'), their own, and the output's where it enters do . o.  fp32 results carry
sums of at most
a few thousand terms at 2^-24 each and hardware exp2 (2 ulp): 1e-5.
"""
import math
import os
import subprocess
import sys

import pytest
import torch

import hclsm_b200
from hclsm_b200.kernels import (Kv8Cache, cross_attention, kv8_attention, kv8_read, kv8_write, qk_norm_rope,
                                rope_tables)

pytestmark = pytest.mark.gpu
U = 2.0 ** -8
F32, BF16 = torch.float32, torch.bfloat16


def _tol(dtype, roundings):
    return roundings * U if dtype == BF16 else 1e-5


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _err(got, ref):
    got, ref = got.double(), ref.double()
    n = ref.norm()
    return float((got - ref).norm() / n) if n > 0 else float(got.norm())


@pytest.fixture(autouse=True)
def _clean():
    assert hclsm_b200.device_error() == 0
    yield
    assert hclsm_b200.device_error() == 0


# ---- norm and rotation --------------------------------------------------------------------------
def _rope_ref(x, w, cos, sin, pos, eps, inter):
    x = x.double()
    if eps is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        x = x * w.double()
    if cos is None:
        return x
    R = 2 * cos.shape[1]
    c, s = (t.double()[pos.long()][:, :, None] for t in (cos, sin))
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if inter else (x[..., :R // 2], x[..., R // 2:R])
    ya, yb = a * c - b * s, a * s + b * c
    y = torch.stack((ya, yb), -1).flatten(-2) if inter else torch.cat((ya, yb), -1)
    return torch.cat((y, x[..., R:]), -1)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D,R,inter,weight", [
    (1, 1, 1, 1, 1, 8, 8, True, True),
    (2, 1, 33, 6, 2, 64, 64, False, True),
    (3, 7, 5, 5, 5, 96, 48, False, False),
    (2, 65, 9, 3, 1, 128, 64, True, True),
    (1, 19, 300, 8, 4, 256, 256, False, True),
    (2, 11, 4, 40, 8, 32, 16, True, True),
    (2, 3, 8, 7, 7, 24, 0, False, True),
])
def test_rope(dtype, B, Lq, Lk, H, Hkv, D, R, inter, weight):
    g = _gen(D + Lq)
    q, k = _randn(g, B, Lq, H, D, dtype=dtype), _randn(g, B, Lk, Hkv, D, dtype=dtype)
    qw, kw = (1 + 0.2 * _randn(g, D) if weight else None for _ in range(2))
    cos, sin = rope_tables(512, R, 1000.0, scale=2.0) if R else (None, None)
    qp = torch.randint(0, 512, (B, Lq), generator=g, device="cuda", dtype=torch.int32)
    leaves = [t.requires_grad_() for t in (q, k, qw, kw) if t is not None]
    yq, yk = qk_norm_rope(q, k, qw, kw, cos, sin, q_pos=qp if R else None, interleaved=inter)
    gq, gk = _randn(g, B, Lq, H, D, dtype=dtype), _randn(g, B, Lk, Hkv, D, dtype=dtype)
    grads = torch.autograd.grad((yq, yk), leaves, (gq, gk))
    ref = [t.detach().double().requires_grad_() for t in leaves]
    rqw, rkw = (ref[2], ref[3]) if weight else (None, None)
    kp = torch.arange(Lk, device="cuda").expand(B, Lk)
    rq, rk = _rope_ref(ref[0], rqw, cos, sin, qp, 1e-6, inter), _rope_ref(ref[1], rkw, cos, sin, kp, 1e-6, inter)
    rg = torch.autograd.grad((rq, rk), ref, (gq.double(), gk.double()))
    assert yq.dtype == dtype and _err(yq, rq) < _tol(dtype, 1) and _err(yk, rk) < _tol(dtype, 1)
    for i, (a, b) in enumerate(zip(grads, rg)):
        assert a.dtype == leaves[i].dtype and _err(a, b) < (_tol(dtype, 1) if i < 2 else 1e-5), i


def test_rope_gradient_against_differences():
    g = _gen(5)
    q, w = _randn(g, 1, 4, 2, 16), 1 + 0.1 * _randn(g, 16)
    cos, sin = rope_tables(8, 16)
    pos = torch.arange(4, device="cuda")[None]
    q.requires_grad_(), w.requires_grad_()
    go = _randn(g, 1, 4, 2, 16)
    dq, dw = torch.autograd.grad(qk_norm_rope(q, None, w, None, cos, sin)[0], (q, w), go)
    uq, uw, h = _randn(g, *q.shape).double(), _randn(g, 16).double(), 1e-4

    def f(t):
        y = _rope_ref(q.detach().double() + t * uq, w.detach().double() + t * uw, cos, sin, pos, 1e-6, False)
        return float((y * go.double()).sum())

    num = (f(h) - f(-h)) / (2 * h)
    got = float((dq.double() * uq).sum() + (dw.double() * uw).sum())
    assert abs(got - num) < 1e-5 * (float(dq.norm() * uq.norm()) + float(dw.norm() * uw.norm()))


def test_rope_alone_strided_and_on_another_stream():
    g = _gen(6)
    qkv = _randn(g, 2, 10, 3, 4, 64, dtype=BF16)  # q, k of a fused projection
    cos, sin = rope_tables(10, 32)
    pos = torch.arange(10, device="cuda").expand(2, 10)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        yq, yk = qk_norm_rope(qkv[:, :, 0], qkv[:, :, 1], cos=cos, sin=sin, eps=None)
    torch.cuda.current_stream().wait_stream(st)
    assert _err(yq, _rope_ref(qkv[:, :, 0], None, cos, sin, pos, None, False)) < U
    assert _err(yk, _rope_ref(qkv[:, :, 1], None, cos, sin, pos, None, False)) < U
    # a head that does not start on 16 bytes, and a broadcast batch
    odd = _randn(g, 2, 10, 4 * 64 + 1, dtype=BF16)[:, :, 1:].unflatten(-1, (4, 64))
    assert _err(qk_norm_rope(odd)[0], _rope_ref(odd, None, None, None, None, 1e-6, False)) < U
    wide = odd[:1].expand(3, 10, 4, 64)
    assert _err(qk_norm_rope(wide)[0], _rope_ref(wide, None, None, None, None, 1e-6, False)) < U


def test_rope_weights_of_one_side_and_positions_in_64_bits():
    g = _gen(16)
    q, k = _randn(g, 2, 5, 4, 64).requires_grad_(), _randn(g, 2, 9, 2, 64).requires_grad_()
    w = (1 + 0.1 * _randn(g, 64)).requires_grad_()
    cos, sin = rope_tables(16, 64)
    pos = torch.randint(0, 16, (2, 9), generator=g, device="cuda")  # int64
    gq, gk = _randn(g, *q.shape), _randn(g, *k.shape)
    ref = [t.detach().double().requires_grad_() for t in (q, k, w)]
    at = torch.arange(5, device="cuda").expand(2, 5)
    for qw, kw in ((w, None), (None, w), (w, w)):
        y = qk_norm_rope(q, k, qw, kw, cos, sin, k_pos=pos)
        got = torch.autograd.grad(y, (q, k, w), (gq, gk))
        r = (_rope_ref(ref[0], None if qw is None else ref[2], cos, sin, at, 1e-6, False),
             _rope_ref(ref[1], None if kw is None else ref[2], cos, sin, pos, 1e-6, False))
        for a, b in zip((*y, *got), (*r, *torch.autograd.grad(r, ref, (gq.double(), gk.double())))):
            assert _err(a, b) < 1e-5
    # a position of 2^32 is outside, not position 0
    y, _ = qk_norm_rope(q[:, :1], None, cos=cos, sin=sin, q_pos=torch.full((2, 1), 1 << 32, device="cuda"))
    assert hclsm_b200.device_error() == 1 and torch.isnan(y).all()


def test_second_derivatives_are_refused():
    x = torch.randn(1, 4, 2, 64, device="cuda", requires_grad=True)
    for f in (lambda: cross_attention(x, x, x), lambda: qk_norm_rope(x)[0]):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(f().sum(), x, create_graph=True)


def test_rope_empty_and_outside_positions():
    q = torch.empty(2, 0, 4, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y, _ = qk_norm_rope(q, None, w)
    dq, dw = torch.autograd.grad(y, (q, w), torch.empty_like(y))
    assert y.shape == q.shape and dq.shape == q.shape and torch.equal(dw, torch.zeros(64, device="cuda"))
    cos, sin = rope_tables(4, 32)
    x = torch.ones(1, 3, 1, 64, device="cuda")
    y, _ = qk_norm_rope(x, cos=cos, sin=sin, q_pos=torch.tensor([[0, 4, -1]], device="cuda", dtype=torch.int32))
    assert hclsm_b200.device_error() == 1
    assert torch.isfinite(y[0, 0]).all() and torch.isnan(y[0, 1:, :, :32]).all() and torch.isfinite(y[..., 32:]).all()


def test_rope_refusals():
    q = torch.zeros(1, 4, 2, 64, device="cuda")
    cos, sin = rope_tables(4, 64)
    for bad, exc in ((lambda: qk_norm_rope(q.cpu()), ValueError),
                     (lambda: qk_norm_rope(q[0]), ValueError),
                     (lambda: qk_norm_rope(q.half()), TypeError),
                     (lambda: qk_norm_rope(q, q.bfloat16()), TypeError),
                     (lambda: qk_norm_rope(q[..., :20]), ValueError),
                     (lambda: qk_norm_rope(q, q[..., :32]), ValueError),
                     (lambda: qk_norm_rope(q, None, torch.ones(32, device="cuda")), ValueError),
                     (lambda: qk_norm_rope(q, None, torch.ones(64, device="cuda"), eps=None), ValueError),
                     (lambda: qk_norm_rope(q, cos=cos), ValueError),
                     (lambda: qk_norm_rope(q, cos=cos[:3], sin=sin[:3]), ValueError),
                     (lambda: qk_norm_rope(q, cos=cos[:, :12], sin=sin[:, :12]), ValueError),
                     (lambda: qk_norm_rope(q[..., :32], cos=cos, sin=sin), ValueError),
                     (lambda: qk_norm_rope(q, cos=cos, sin=sin, q_pos=torch.zeros(1, 3, device="cuda").int()),
                      ValueError),
                     (lambda: qk_norm_rope(q, cos=cos, sin=sin, q_pos=torch.zeros(1, 4, device="cuda")), TypeError),
                     (lambda: rope_tables(4, 7), ValueError)):
        with pytest.raises(exc):
            bad()


# ---- cross attention ------------------------------------------------------------------------------
def _allowed(B, Lk, lens, mask):
    ok = torch.ones(B, Lk, dtype=torch.bool, device="cuda")
    if lens is not None:
        ok &= torch.arange(Lk, device="cuda") < lens[:, None]
    return ok if mask is None else ok & mask


def _attn_ref(q, k, v, ok, scale=None):
    """64 bits, over what is allowed alone; ok (B, Lk)."""
    G = q.shape[2] // k.shape[2]
    q, k, v = (t.double() for t in (q, k, v))
    k, v = (torch.where(ok[:, :, None, None], t, 0.0).repeat_interleave(G, 2) for t in (k, v))
    s = torch.einsum("bihd,bjhd->bhij", q, k) * (q.shape[-1] ** -0.5 if scale is None else scale)
    s = s.masked_fill(~ok[:, None, None], -math.inf)
    p = torch.nan_to_num(torch.softmax(s, -1))  # a row without keys: zeros
    return torch.einsum("bhij,bjhd->bihd", p, v)


CASES = [  # B, Lq, Lk, H, Hkv, D
    (1, 1, 1, 1, 1, 64), (2, 1, 300, 4, 4, 64), (2, 1, 1000, 8, 2, 128), (3, 2, 77, 6, 2, 96), (2, 5, 130, 3, 3, 32),
    (2, 32, 196, 6, 6, 64), (1, 130, 257, 4, 1, 64), (1, 129, 128, 2, 2, 128), (2, 33, 65, 3, 3, 40),
    (1, 17, 50, 2, 1, 33), (1, 300, 520, 2, 1, 96), (1, 1, 4099, 16, 1, 128), (4, 70, 129, 1, 1, 8),
    (1, 64, 640, 5, 5, 32), (1, 257, 1, 2, 2, 64), (1, 140, 400, 8, 2, 120),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", CASES)
@pytest.mark.parametrize("masked", [False, True])
def test_cross_attention(dtype, shape, masked):
    B, Lq, Lk, H, Hkv, D = shape
    g = _gen(Lq * 1000 + Lk + D)
    q, k, v = (_randn(g, B, n, h, D, dtype=dtype) for n, h in ((Lq, H), (Lk, Hkv), (Lk, Hkv)))
    lens = mask = None
    if masked:
        lens = torch.randint(0, Lk + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        lens[0] = max(1, Lk - 3)
        mask = torch.rand(B, Lk, generator=g, device="cuda") > 0.3
        mask[0, 0] = True
    ok = _allowed(B, Lk, lens, mask)
    do = _randn(g, B, Lq, H, D, dtype=dtype)
    with torch.no_grad():
        o0 = cross_attention(q, k, v, kv_lens=lens, key_mask=mask)
    ref = [t.double().requires_grad_() for t in (q, k, v)]
    ro = _attn_ref(*ref, ok)
    assert o0.dtype == dtype and _err(o0, ro) < _tol(dtype, 2)
    for t in (q, k, v):
        t.requires_grad_()
    o = cross_attention(q, k, v, kv_lens=lens, key_mask=mask)
    assert _err(o, ro) < _tol(dtype, 2)
    grads = torch.autograd.grad(o, (q, k, v), do)
    for name, a, b in zip(("dq", "dk", "dv"), grads, torch.autograd.grad(ro, ref, do.double())):
        if b.norm() < 1e-12:  # one key: its weight is 1 whatever the scores; dq, dk are cancellation residues
            assert a.double().norm() < _tol(dtype, 3) * do.double().norm() * v.double().norm(), name
        else:
            assert _err(a, b) < _tol(dtype, 3), name


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Lq,Lk,D", [(1, 200, 64), (40, 200, 64), (150, 333, 128), (9, 70, 40)])
def test_what_is_not_allowed_may_be_nan(dtype, Lq, Lk, D):
    g = _gen(7)
    q, k, v = (_randn(g, 4, n, 2, D, dtype=dtype) for n in (Lq, Lk, Lk))
    lens = torch.tensor([0, 1, Lk // 2 + 1, Lk], device="cuda", dtype=torch.int32)
    mask = torch.rand(4, Lk, generator=g, device="cuda") > 0.2
    mask[1, 0], mask[3] = True, False
    ok = _allowed(4, Lk, lens, mask)
    ro = _attn_ref(q, k, v, ok)
    bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).min], device="cuda", dtype=dtype)
    fill = bad[torch.arange(Lk, device="cuda") % 4][None, :, None, None]
    kb, vb = (torch.where(ok[:, :, None, None], t, fill).requires_grad_() for t in (k, v))
    q.requires_grad_()
    o = cross_attention(q, kb, vb, kv_lens=lens, key_mask=mask)
    assert _err(o, ro) < _tol(dtype, 2)
    assert torch.equal(o[0], torch.zeros_like(o[0])) and torch.equal(o[3], torch.zeros_like(o[3]))
    do = _randn(g, 4, Lq, 2, D, dtype=dtype)
    dq, dk, dv = torch.autograd.grad(o, (q, kb, vb), do)
    ref = [t.detach().double().requires_grad_() for t in (q, k, v)]
    for name, a, b in zip(("dq", "dk", "dv"), (dq, dk, dv),
                          torch.autograd.grad(_attn_ref(*ref, ok), ref, do.double())):
        assert _err(a, b) < _tol(dtype, 3), name
    assert not dq[0].any() and not dq[3].any()
    assert not dk[~ok].any() and not dv[~ok].any()


def test_cross_attention_gradient_against_differences():
    g = _gen(8)
    q, k, v = (_randn(g, 2, n, h, 32).requires_grad_() for n, h in ((6, 4), (40, 2), (40, 2)))
    lens = torch.tensor([40, 23], device="cuda", dtype=torch.int32)
    do = _randn(g, 2, 6, 4, 32)
    grads = torch.autograd.grad(cross_attention(q, k, v, kv_lens=lens), (q, k, v), do)
    ok = _allowed(2, 40, lens, None)
    for i, name in enumerate(("dq", "dk", "dv")):
        u, h = _randn(g, *grads[i].shape).double(), 1e-4

        def f(t):
            x = [y.detach().double() for y in (q, k, v)]
            x[i] = x[i] + t * u
            return float((_attn_ref(*x, ok) * do.double()).sum())

        num, got = (f(h) - f(-h)) / (2 * h), float((grads[i].double() * u).sum())
        assert abs(got - num) < 1e-5 * float(grads[i].norm() * u.norm()), name


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Lq", [1, 200])
def test_cross_attention_strides_streams_and_repeats(dtype, Lq):
    g = _gen(9)
    kv = _randn(g, 2, 150, 2, 2, 64, dtype=dtype)  # keys and values of one projection
    q = _randn(g, 2, 4, Lq, 64, dtype=dtype).transpose(1, 2)  # head-major queries
    k, v = kv[:, :, 0], kv[:, :, 1]
    ok = _allowed(2, 150, None, None)
    ref = _attn_ref(q, k, v, ok, 0.3)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        o = cross_attention(q, k, v, scale=0.3)
    torch.cuda.current_stream().wait_stream(st)
    assert _err(o, ref) < _tol(dtype, 2)
    # rows that do not start on 16 bytes; a broadcast batch and a broadcast gradient
    odd = torch.empty(2, 150, 2 * 64 + 3, device="cuda", dtype=dtype)[:, :, 3:].unflatten(-1, (2, 64))
    odd.copy_(k)
    assert _err(cross_attention(q, odd, v, scale=0.3), ref) < _tol(dtype, 2)
    one = k[:1].expand(2, 150, 2, 64)
    leaves = [t.detach().requires_grad_() for t in (q, one, v)]
    do = torch.ones(1, device="cuda", dtype=dtype).expand(2, Lq, 4, 64)
    runs = [torch.autograd.grad(cross_attention(*leaves, scale=0.3), leaves, do) for _ in range(2)]
    ref = [t.detach().double().requires_grad_() for t in leaves]
    for a, b, c in zip(*runs, torch.autograd.grad(_attn_ref(*ref, ok, 0.3), ref, do.double())):
        assert torch.equal(a, b) and _err(a, c) < _tol(dtype, 3)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_cross_attention_large_scores_and_empty_sizes(dtype):
    g = _gen(10)
    q, k, v = (30 * _randn(g, 1, n, 2, 64, dtype=dtype) for n in (70, 300, 300))
    assert _err(cross_attention(q, k, v), _attn_ref(q, k, v, _allowed(1, 300, None, None))) < _tol(dtype, 2) * 10
    for Lq, Lk in ((0, 5), (3, 0), (0, 0)):
        q, k, v = (torch.zeros(2, n, 2, 64, device="cuda", dtype=dtype, requires_grad=True) for n in (Lq, Lk, Lk))
        o = cross_attention(q, k, v)
        assert o.shape == q.shape and not o.any()
        for a in torch.autograd.grad(o, (q, k, v), torch.ones_like(o)):
            assert not a.any()


def test_first_call_of_a_thread():
    """A thread without a current context: the forward and the backward (autograd's own thread) bind it themselves."""
    code = """
import threading, torch
from hclsm_b200.kernels import cross_attention
x = [torch.randn(2, 150, 2, 64, device="cuda").bfloat16().requires_grad_() for _ in range(3)]
out = []
t = threading.Thread(target=lambda: out.append(cross_attention(*x)))
t.start(), t.join()
g = torch.autograd.grad(out[0], x, torch.ones_like(out[0]))
assert all(torch.isfinite(v).all() for v in (out[0], *g))
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, "-c", code], check=True, cwd=root, timeout=300)


@pytest.mark.parametrize("Lq", [1, 150])
def test_offsets_past_32_bits(Lq):
    """Batch entries 2^31 elements apart, with nothing but stale memory between them."""
    g = _gen(15)
    far = torch.empty((1 << 31) + 300 * 64, device="cuda", dtype=BF16)
    k = far.as_strided((2, 300, 1, 64), (1 << 31, 64, 64, 1))
    k.copy_(_randn(g, 2, 300, 1, 64, dtype=BF16))
    q = _randn(g, 2, Lq, 1, 64, dtype=BF16).requires_grad_()
    ok, do = _allowed(2, 300, None, None), _randn(g, 2, Lq, 1, 64, dtype=BF16)
    kk = k.requires_grad_()
    o = cross_attention(q, kk, kk.detach())
    ref = [t.detach().double().requires_grad_() for t in (q, k)]
    ro = _attn_ref(ref[0], ref[1], ref[1].detach(), ok)
    assert _err(o, ro) < 2 * U
    for a, b in zip(torch.autograd.grad(o, (q, kk), do), torch.autograd.grad(ro, ref, do.double())):
        assert _err(a, b) < 3 * U


def test_cross_attention_refusals():
    q, k = torch.zeros(2, 3, 4, 64, device="cuda"), torch.zeros(2, 5, 2, 64, device="cuda")
    lens = torch.zeros(2, device="cuda", dtype=torch.int32)
    for bad, exc in ((lambda: cross_attention(q.cpu(), k, k), ValueError),
                     (lambda: cross_attention(q, k, k[:, :4]), ValueError),
                     (lambda: cross_attention(q[:1], k, k), ValueError),
                     (lambda: cross_attention(q[:, :, :3], k, k), ValueError),
                     (lambda: cross_attention(q, k[..., :32], k[..., :32]), ValueError),
                     (lambda: cross_attention(q.bfloat16(), k, k), TypeError),
                     (lambda: cross_attention(q.half(), k.half(), k.half()), TypeError),
                     (lambda: cross_attention(q, k, k, scale=0.0), ValueError),
                     (lambda: cross_attention(q, k, k, scale=math.inf), ValueError),
                     (lambda: cross_attention(q, k, k, kv_lens=lens[:1]), ValueError),
                     (lambda: cross_attention(q, k, k, kv_lens=lens.float()), TypeError),
                     (lambda: cross_attention(q, k, k, kv_lens=lens.cpu()), ValueError),
                     (lambda: cross_attention(q, k, k, key_mask=torch.ones(2, 5, device="cuda")), ValueError),
                     (lambda: cross_attention(q, k, k, key_mask=torch.ones(2, 4, device="cuda").bool()), ValueError),
                     (lambda: cross_attention(*(torch.zeros(1, 2, 1, 136, device="cuda") for _ in range(3))),
                      ValueError)):
        with pytest.raises(exc):
            bad()


# ---- the 8-bit cache --------------------------------------------------------------------------------
class _Plain:
    """The cache in 64 bits: every token's exact value until its block fills, then what 8 bits hold."""

    def __init__(self, B, T, Hkv, D, block):
        self.x, self.block = torch.zeros(2, B, T, Hkv, D, dtype=torch.float64, device="cuda"), block

    def write(self, kv, start, count):
        for b, (s, n) in enumerate(zip(start, count)):
            for i in range(2):
                self.x[i, b, s:s + n] = kv[i][b, :n].double()
                for blk in range(s // self.block, (s + n) // self.block):
                    t = self.x[i, b, blk * self.block:(blk + 1) * self.block]
                    # the scale and the quotient are fp32 numbers by definition
                    sc = (t.abs().amax((0, 2), keepdim=True).float()
                          / torch.tensor(127.0, device="cuda")).expand(t.shape)
                    r = torch.where(sc > 0, torch.round(t.float() / sc), 0.0)
                    t.copy_(r.double() * sc.double())


def _i32(*v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,block,Hkv,G", [(64, 32, 3, 1), (128, 16, 2, 4), (32, 128, 1, 2), (96, 64, 2, 17)])
def test_cache_write_read_attend(dtype, D, block, Hkv, G):
    g = _gen(D + block)
    B, T = 4, 5 * block
    cache, plain = Kv8Cache.empty(B, T - 1, Hkv, D, block=block, dtype=dtype), _Plain(B, T, Hkv, D, block)
    assert cache.k.shape[2] == T
    cache.k_tail.fill_(math.nan), cache.v_tail.fill_(math.nan)  # stale memory is never an operand
    start = [0, 0, 0, 0]
    # nothing; one token; up to a block's end; over several; one by one across an end; to the last token
    for counts in ((0, 1, block - 1, 2 * block + 3), (0, block - 1, 1, block - 4), (0, 1, 1, 1), (0, 2, block + 1, 1),
                   (1, 3 * block, 2, 2 * block - 1)):
        n = max(counts)
        kv = [_randn(g, B, n, Hkv, D, dtype=dtype) * 3 for _ in range(2)]
        kv8_write(cache, *kv, _i32(*start), _i32(*counts))
        plain.write(kv, start, counts)
        start = [a + c for a, c in zip(start, counts)]
        lens = _i32(*start)
        # and from the middle of what is there: inside a complete block, or inside the tail
        part = _i32(*(max(0, v - 1 - i) for i, v in enumerate(start)))
        q = _randn(g, B, 1, Hkv * G, D, dtype=dtype)
        ref = _attn_ref(q, plain.x[0], plain.x[1], _allowed(B, T, part, None))
        assert _err(kv8_attention(q, cache, part), ref) < _tol(dtype, 2)
        for got, want in zip(kv8_read(cache, lens), plain.x):
            assert got.dtype == dtype and _err(got, want) < (U if dtype == BF16 else 1e-6)
        ok = _allowed(B, T, lens, None)
        for Lq in (1, 3):
            q = _randn(g, B, Lq, Hkv * G, D, dtype=dtype)
            o = kv8_attention(q, cache, lens)
            assert _err(o, _attn_ref(q, plain.x[0], plain.x[1], ok)) < _tol(dtype, 2)
            assert torch.equal(o, kv8_attention(q, cache, lens))
    assert start[3] == T


def test_cache_long_and_shorter_views_of_it():
    g = _gen(12)
    B, T, Hkv, D = 2, 9000 // 32 * 32, 2, 64
    cache, plain = Kv8Cache.empty(B, T, Hkv, D), _Plain(B, T, Hkv, D, 32)
    kv = [_randn(g, B, T, Hkv, D, dtype=BF16) for _ in range(2)]
    kv8_write(cache, *kv, _i32(0, 0))
    plain.write(kv, [0, 0], [T, T])
    q = _randn(g, B, 2, 8, D, dtype=BF16)
    # lengths at a block's end, inside complete blocks, past the capacity, and all of it
    for lens in (_i32(T, 4096), _i32(4100, 17), _i32(T - 1, 1), _i32(T + 50, 0), None):
        if lens is not None:
            for got, want in zip(kv8_read(cache, lens), plain.x):
                keep = _allowed(B, T, lens.clamp(0, T), None)[:, :, None, None]
                assert _err(got, torch.where(keep, want, 0.0)) < U
        ok = _allowed(B, T, None if lens is None else lens.clamp(0, T), None)
        assert _err(kv8_attention(q, cache, lens, scale=0.2), _attn_ref(q, *plain.x, ok, 0.2)) < 2 * U


def test_cache_values_that_are_zero_or_not_finite_and_step_replay():
    cache = Kv8Cache.empty(1, 64, 1, 32, dtype=F32)
    x = torch.zeros(1, 64, 1, 32, device="cuda")
    x[0, 40, 0, 5] = math.inf
    kv8_write(cache, x, x, _i32(0))
    k, _ = kv8_read(cache)
    assert not k[0, :32].any() and torch.isnan(k[0, 32:]).all()
    q = torch.ones(1, 1, 1, 32, device="cuda")
    assert not kv8_attention(q, cache, _i32(32)).any() and torch.isnan(kv8_attention(q, cache, _i32(64))).all()
    # a step captured once and replayed with other positions
    g = _gen(13)
    cache, plain = Kv8Cache.empty(2, 96, 2, 64), _Plain(2, 96, 2, 64, 32)
    k, v, q = (_randn(g, 2, 1, h, 64, dtype=BF16) for h in (2, 2, 4))
    start, lens = _i32(0, 0), _i32(1, 1)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        kv8_write(cache, k, v, start)
        kv8_attention(q, cache, lens)
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv8_write(cache, k, v, start)
        o = kv8_attention(q, cache, lens)
    for t in range(70):
        for x in (k, v, q):
            x.copy_(_randn(g, *x.shape, dtype=BF16))
        start.fill_(t), lens.fill_(t + 1)
        graph.replay()
        plain.write((k, v), [t, t], [1, 1])
        assert _err(o, _attn_ref(q, *plain.x, _allowed(2, 96, lens, None))) < 2 * U, t


def test_cache_offsets_past_32_bits():
    """The second sequence's states start 2^31 bytes into the cache."""
    g = _gen(14)
    cache, plain = Kv8Cache.empty(2, 1 << 24, 1, 128), _Plain(2, 96, 1, 128, 32)
    kv = [_randn(g, 2, 90, 1, 128, dtype=BF16) for _ in range(2)]
    kv8_write(cache, *kv, _i32(0, 0))
    plain.write(kv, [0, 0], [90, 90])
    q = _randn(g, 2, 1, 2, 128, dtype=BF16)
    lens = _i32(17, 90)
    assert _err(kv8_attention(q, cache, lens), _attn_ref(q, *plain.x, _allowed(2, 96, lens, None))) < 2 * U
    assert cache.k[1, 0, :64].any() and not cache.k[0, 0, 64:].any()


def test_cache_requests_that_do_not_fit_write_nothing():
    cache = Kv8Cache.empty(1, 32, 1, 32, dtype=F32)
    x = torch.ones(1, 8, 1, 32, device="cuda")
    for start, count in ((25, 8), (-1, 8), (0, 9), (0, -1), (2 ** 31 - 4, 8)):
        kv8_write(cache, x, x, _i32(start), _i32(count))
        assert hclsm_b200.device_error() == 1
        assert not cache.k.any() and not cache.k_tail.any() and (cache.k_scale == -1).all()


def test_cache_refusals():
    c = Kv8Cache.empty(2, 64, 2, 64)
    x, q, at = (torch.zeros(2, 3, h, 64, device="cuda", dtype=BF16) for h in (2, 4, 4))
    at = _i32(0, 0)
    parts = [c.k, c.v, c.k_scale, c.v_scale, c.k_tail, c.v_tail]

    def swap(i, t):
        return Kv8Cache(*parts[:i], t, *parts[i + 1:])

    for bad, exc in ((lambda: Kv8Cache.empty(2, 64, 2, 48), ValueError),
                     (lambda: Kv8Cache.empty(2, 64, 2, 64, block=24), ValueError),
                     (lambda: Kv8Cache.empty(2, 64, 2, 64, dtype=torch.float16), TypeError),
                     (lambda: swap(1, c.v[:, :, :32]), ValueError),
                     (lambda: swap(2, c.k_scale.double()), ValueError),
                     (lambda: swap(5, c.v_tail.float()), ValueError),
                     (lambda: swap(0, c.k.transpose(0, 1)), ValueError),
                     (lambda: kv8_write(c, x, x[:, :2], at), ValueError),
                     (lambda: kv8_write(c, x.float(), x.float(), at), TypeError),
                     (lambda: kv8_write(c, x, x, at[:1]), ValueError),
                     (lambda: kv8_write(c, x, x, None), ValueError),
                     (lambda: kv8_write(c, x, x, at.float()), TypeError),
                     (lambda: kv8_read(c, at.cpu()), ValueError),
                     (lambda: kv8_attention(q[:1], c, at), ValueError),
                     (lambda: kv8_attention(q[:, :, :3], c, at), ValueError),
                     (lambda: kv8_attention(q.float(), c, at), TypeError),
                     (lambda: kv8_attention(q, c, at, scale=-1.0), ValueError),
                     (lambda: kv8_attention(q.clone().requires_grad_(), c, at), NotImplementedError)):
        with pytest.raises(exc):
            bad()
