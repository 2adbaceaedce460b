"""Further edges of the attention operators: long sweeps with part-filled query tiles, layouts with free strides,
accuracy that only the right intermediate types give, and derivatives that are refused instead of dropped.

Errors are 2-norms relative to the result's, u = 2^-8 is bf16's unit roundoff.
"""
import pytest
import torch

import hclsm_b200
from hclsm_b200.kernels import Kv8Cache, cross_attention, kv8_attention, kv8_read, kv8_write, qk_norm_rope
from hclsm_b200.kernels.cross_attn import attention_bwd, attention_fwd
from test_attention_ops_gpu import BF16, F32, U, _allowed, _attn_ref, _err, _gen, _i32, _Plain, _randn, _rope_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean():
    assert hclsm_b200.device_error() == 0
    yield
    assert hclsm_b200.device_error() == 0


@pytest.mark.parametrize("D", [32, 40, 64])
@pytest.mark.parametrize("Lq", [129, 160, 200, 300, 333])
@pytest.mark.parametrize("Lk", [700, 2049, 4100])
@pytest.mark.parametrize("masked", [False, True])
def test_long_sweeps_with_part_filled_query_tiles(D, Lq, Lk, masked):
    """bf16 forward, heads up to 64, more than 128 queries: many tiles of keys go round the ring of staged tiles, the
    last query tile has warps without a row, and scores that grow along the keys raise the maximum again and again.
    Weights and output are rounded once each: 2 u."""
    g = _gen(Lq + Lk + D)
    B, H, Hkv = 2, 2, 1
    q, k, v = (_randn(g, B, n, h, D) for n, h in ((Lq, H), (Lk, Hkv), (Lk, Hkv)))
    lens = mask = None
    if masked:
        lens = torch.tensor([Lk - 3, Lk // 2 + 5], device="cuda", dtype=torch.int32)
        mask = torch.rand(B, Lk, generator=g, device="cuda") > 0.3
    ok = _allowed(B, Lk, lens, mask)
    rise = torch.linspace(0, 8, Lk, device="cuda")[None, :, None, None]  # times sqrt(D) log2 e in log2
    for up in (0.0, 1.0):
        qq, kk, vv = (q + up).to(BF16), (k + up * rise).to(BF16), v.to(BF16)
        runs = [cross_attention(qq, kk, vv, kv_lens=lens, key_mask=mask) for _ in range(3)]
        assert _err(runs[0], _attn_ref(qq, kk, vv, ok)) < 2 * U
        assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


def _single(g, dtype, L, odd):
    """(1, L, 4, 64) whose strides of size-1 dims are no multiple of 16 bytes: one entry of a padded buffer (odd batch
    stride), or for L = 1 the first token of a padded projection (odd batch and token strides)."""
    if L == 1:
        return _randn(g, 1, 8, 4 * 64 + odd, dtype=dtype)[..., :256].unflatten(-1, (4, 64))[:, :1]
    flat = _randn(g, 3 * (L * 256 + odd), dtype=dtype)
    return flat.as_strided((1, L, 4, 64), (L * 256 + odd, 256, 64, 1), 0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("L", [1, 70])
@pytest.mark.parametrize("odd", [1, 4])
def test_strides_of_dims_of_one_do_not_count(dtype, L, odd):
    """A dim of one is never stepped over, so its stride is no reason to refuse, copy or take a slower form: results are
    those of dense tensors to the bit."""
    g = _gen(L + odd)
    x, y = _single(g, dtype, L, odd), _single(g, dtype, L, odd)
    dense = [t.new_empty(t.shape).copy_(t) for t in (x, y)]
    runs = []
    for q, k in ((x, y), dense):
        q, k = (t.detach().requires_grad_() for t in (q, k))
        out = qk_norm_rope(q, k)
        runs.append([*out, *torch.autograd.grad(out, (q, k), dense)])
    for a, b in zip(*runs):
        assert torch.equal(a, b)
    assert _err(runs[0][0], _rope_ref(x, None, None, None, None, 1e-6, False)) < (U if dtype == BF16 else 1e-5)
    caches = [Kv8Cache.empty(1, 96, 4, 64, dtype=dtype) for _ in range(2)]
    for c, (k, v) in zip(caches, ((x, y), dense)):
        kv8_write(c, k, v, _i32(0))
    for a, b in zip(*(kv8_read(c, _i32(L)) for c in caches)):
        assert torch.equal(a, b)
    # one query over 2000 keys of one batch entry: the form that splits the keys
    k, v = _single(g, dtype, 2000, odd), _single(g, dtype, 2000, odd)
    for Lq in (1, 150):
        q = _randn(g, 1, Lq, 4, 64, dtype=dtype)
        kd, vd = (t.new_empty(t.shape).copy_(t) for t in (k, v))
        assert torch.equal(cross_attention(q, k, v), cross_attention(q, kd, vd))


@pytest.mark.parametrize("far", [0, 5, 15])
@pytest.mark.parametrize("D,G,block", [(64, 4, 32), (128, 12, 16), (32, 1, 64)])
def test_cache_blocks_of_large_values_and_no_weight(far, D, G, block):
    """A block whose values are 1e6 to 1e30 times the others' but whose keys weigh e^-60 and less, or one of zeros whose
    keys weigh e^25 and more, takes nothing from the precision of the others: 2 u as ever."""
    g = _gen(D + far)
    T = 16 * block
    for size, unit, key in ((1e6, 1.0, -10.0), (1e10, 1.0, -10.0), (1e14, 1.0, -10.0), (1e30, 1.0, -10.0),
                            (1e30, 1e-35, -10.0), (0.0, 1.0, 4.0), (0.0, 1e-20, 4.0)):
        k, v = 0.5 * _randn(g, 2, T, 2, D), unit * _randn(g, 2, T, 2, D)
        k[:, far * block:(far + 1) * block] = key
        v[:, far * block:(far + 1) * block] *= size
        q = (1 + 0.3 * _randn(g, 2, 1, 2 * G, D)).to(BF16)
        k, v = k.to(BF16), v.to(BF16)
        scale = 7.5 / D  # q . k scale = -75 or 30, +- 15 %, there
        cache, plain = Kv8Cache.empty(2, T, 2, D, block=block), _Plain(2, T, 2, D, block)
        kv8_write(cache, k, v, _i32(0, 0))
        plain.write((k, v), [0, 0], [T, T])
        for lens in (_i32(T, T), _i32(T, T - block // 2)):
            got = kv8_attention(q, cache, lens, scale=scale)
            assert _err(got, _attn_ref(q, *plain.x, _allowed(2, T, lens, None), scale)) < 2 * U, (size, unit)


def _one_rounding(ref):
    """The error of the 64-bit result rounded to bf16 once: what an output cannot be better than."""
    return _err(ref.to(BF16), ref)


@pytest.mark.parametrize("Lq,Lk,D", [(200, 2000, 64), (200, 2000, 128), (40, 2000, 64), (1, 9000, 128)])
def test_forward_error_is_that_of_two_roundings(Lq, Lk, D):
    """Weights are rounded to bf16 once, independently of each other, and so is the output: with random values both errors
    are of one size, sqrt(2) of one; 10 % for what else there is (exponentials 1e-4, sums in fp32)."""
    g = _gen(Lq + D)
    q, k, v = (_randn(g, 2, n, 4, D, dtype=BF16) for n in (Lq, Lk, Lk))
    ref = _attn_ref(q, k, v, _allowed(2, Lk, None, None))
    assert _err(cross_attention(q, k, v), ref) < 1.1 * 2 ** 0.5 * _one_rounding(ref)


@pytest.mark.parametrize("D,G", [(64, 1), (128, 4), (64, 12)])
def test_cache_error_is_that_of_one_rounding(D, G):
    """Weights against the cache are fp16 (3 bits more than the output): the output's rounding is nearly all of the error.
    bf16 weights would give sqrt(2) of it."""
    g = _gen(D + G)
    T = 8192
    cache, plain = Kv8Cache.empty(2, T, 2, D), _Plain(2, T, 2, D, 32)
    kv = [_randn(g, 2, T, 2, D, dtype=BF16) for _ in range(2)]
    kv8_write(cache, *kv, _i32(0, 0))
    plain.write(kv, [0, 0], [T, T])
    q = _randn(g, 2, 1, 2 * G, D, dtype=BF16)
    ref = _attn_ref(q, *plain.x, _allowed(2, T, None, None))
    assert _err(kv8_attention(q, cache, _i32(T, T)), ref) < 1.15 * _one_rounding(ref)


@pytest.mark.parametrize("Lq,D", [(1, 64), (40, 64), (200, 64), (200, 128), (40, 33)])
def test_what_rounding_took_from_the_output_reaches_the_backward(Lq, D):
    """With queries of zero the weights of 4 keys are 1/4 exactly, and values of 64 + N(0, 1) make the output's rounding
    (steps of 0.5) as large as what do . (v - o) is made of: gradients are right only through lo.  o + lo: 16 bits, 2^-16.
    dq: the weights' gradients and the result rounded once each, and sums of 64 D terms, 2 u and an eighth more."""
    g = _gen(Lq + D)
    q = torch.zeros(2, Lq, 2, D, device="cuda", dtype=BF16)
    k, v, do = (_randn(g, 2, n, 2, D) for n in (4, 4, Lq))
    k, v, do = k.to(BF16), (64 + v).to(BF16), do.to(BF16)
    ok = _allowed(2, 4, None, None)
    o, lse, lo = attention_fwd(q, k, v, None, None, D ** -0.5)
    ref = [t.double().requires_grad_() for t in (q, k, v)]
    ro = _attn_ref(*ref, ok)
    assert _err(o.double() + lo.double(), ro) < 2.0 ** -16 and _err(o, ro) > 2.0 ** -11
    got = attention_bwd(q, k, v, o, lse, lo, do, None, None, D ** -0.5)
    want = torch.autograd.grad(ro, ref, do.double())
    assert _err(got[0], want[0]) < 2.25 * U and _err(got[2], want[2]) < 2.25 * U
    # the halves are summed: which of the two holds what is nothing to the backward
    swapped = attention_bwd(q, k, v, lo, lse, o, do, None, None, D ** -0.5)
    for a, b in zip(got, swapped):
        assert torch.equal(a, b)
