"""The operators that remember a history on the GPU: every kernel that a call can choose, and bounds that a lost piece of an
operand or a wrong correction does not meet, against plain definitions in 64 bits."""
import pytest
import torch

import hclsm_b200
from hclsm_b200 import _lib
from hclsm_b200.kernels import Kv4Cache, decay_attention, kv4_attention
from memory_ref import decay_grads, decay_ref, kv4_unpack
from test_memory_ops_gpu import _check_decay, _decays, _inputs, _near

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def no_device_error():
    hclsm_b200.device_error()
    yield
    assert hclsm_b200.device_error() == 0


# ---- decaying linear attention: two blocks a multiprocessor, segments of unequal head dims -------------
def _segments(B, L, H, D, Dv, backward):
    """Bytes of the workspace, which a bf16 call has where its histories are cut into segments."""
    lib, some = _lib.load(), 1 << 20
    views = [x for d in (D, D, Dv, Dv) for x in (some, L * H * d, H * d, d)]
    a = _lib.DECAY_ARGS.pack(*views, *(some,) * 5, *(some,) * 4, 0, B, L, H, D, Dv, _lib.BF16, 1.0)
    return (lib.hclsm_decay_attn_bwd_workspace_size if backward else lib.hclsm_decay_attn_fwd_workspace_size)(a)


@pytest.mark.parametrize("L", [1, 128, 300])
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("D,Dv", [(64, 64), (32, 64), (64, 40)])
def test_decay_attention_of_more_heads_than_multiprocessors(L, state, D, Dv):
    """240 heads forward, 480 or 720 passes backward, in both directions of time; with and without a state that is returned."""
    B, H = 40, 6
    assert B * H > torch.cuda.get_device_properties(0).multi_processor_count
    x, g = _inputs(B, L, H, D, Dv, BF, state), _decays(H)
    lens = torch.randint(0, L + 1, (B,), device="cuda", dtype=torch.int32)
    lens[0] = L
    _check_decay(x, g, lens, BF, D ** -0.5)
    o = decay_attention(x["q"], x["k"], x["v"], g, state=x["S0"], lens=lens)  # the state is not returned
    gr = g.clamp(min=-1e30)
    ro, _ = decay_ref(x["q"], x["k"], x["v"], gr, x["S0"], lens, D ** -0.5)
    ao, _ = decay_ref(*(x[n].abs() for n in ("q", "k", "v")), gr, None if x["S0"] is None else x["S0"].abs(), lens, D ** -0.5)
    _near(o, ro, 2.0 ** -8 * ro.abs() + (2.0 ** -8 + (L + D + Dv + 256) * 2.0 ** -24) * ao, "o")


@pytest.mark.parametrize("B,L,H,D,Dv", [(1, 2500, 2, 64, 128), (1, 2500, 2, 128, 64), (2, 1700, 3, 128, 32), (2, 1700, 2, 40, 96)])
@pytest.mark.parametrize("state,ragged", [(False, False), (True, True)])
def test_decay_attention_segments_of_unequal_head_dims(B, L, H, D, Dv, state, ragged):
    assert _segments(B, L, H, D, Dv, False) and _segments(B, L, H, D, Dv, True)
    x, g = _inputs(B, L, H, D, Dv, BF, state), _decays(H)
    lens = torch.tensor([L - 131, 0][:B], device="cuda", dtype=torch.int32) if ragged else None
    _check_decay(x, g, lens, BF, D ** -0.5)


def test_decay_attention_segments_of_more_blocks_than_multiprocessors():
    """A long history in more segments than multiprocessors.  Heads that forget e^-30 over 600 tokens: a window of the history is
    what the definition gives on the window and 600 tokens around it."""
    B, L, H, D, margin = 1, 40000, 6, 64, 600
    for backward in (False, True):
        assert _segments(B, L, H, D, D, backward) // (H * D * D * 4) * H > torch.cuda.get_device_properties(0).multi_processor_count
    x = _inputs(B, L, H, D, D, BF, False)
    g = -torch.linspace(0.05, 1.0, H, device="cuda")
    leaves = [x[n].requires_grad_() for n in ("q", "k", "v")]
    o, S = decay_attention(*leaves, g, return_state=True)
    alone = decay_attention(*(t.detach() for t in leaves), g)
    grads = torch.autograd.grad(o, leaves, x["do"])
    x = {n: None if t is None else t.detach() for n, t in x.items()}
    fp32, e = (margin * 3 + 2 * D + 256) * 2.0 ** -24, 2.0 ** -8
    for at in (0, 5000, 19937, L - 800):
        lo, hi = max(at - margin, 0), min(at + 800 + margin, L)
        keep = slice(at - lo, at - lo + 800)
        part = [x[n][:, lo:hi] for n in ("q", "k", "v")]
        do = x["do"][:, lo:hi]
        ro, rS = decay_ref(*part, g, scale=D ** -0.5)
        ao, aS = decay_ref(*(t.abs() for t in part), g, scale=D ** -0.5)
        for got in (o.detach(), alone):
            _near(got[:, at:at + 800], ro[:, keep], (e * ro.abs() + (e + fp32) * ao)[:, keep], "o")
        if hi == L:
            _near(S.detach(), rS, fp32 * aS, "state")
        want = decay_grads(*part, g, None, None, D ** -0.5, do, None)
        most = decay_grads(*(t.abs() for t in part), g, None, None, D ** -0.5, do.abs(), None)
        for n, got, w, m in zip(("dq", "dk", "dv"), grads, want, most):
            _near(got[:, at:at + 800], w[:, keep], (e * w.abs() + (e + fp32) * m)[:, keep], n)


# ---- attention over the 4-bit cache ---------------------------------------------------------------------
def _pieces(x, n):
    """x (64 bits, fp32 numbers) as the sum of its n first bf16 pieces."""
    out = torch.zeros_like(x)
    for _ in range(n):
        out = out + (x - out).float().bfloat16().double()
    return out


def _attend(q, k, vc, vs, scale, whole_queries=True, whole_weights=True):
    """Attention of q (B, Lq, H, D) over keys k (B, T, Hkv, D), codes vc of values and their scales vs (B, T, Hkv, D / 32), all
    in 64 bits; a kernel that lost the third piece of a query, or of a weight times a value's scale, would give the
    result with that flag false."""
    G = q.shape[2] // k.shape[2]
    k, vc, vs = (t.repeat_interleave(G, 2) for t in (k, vc, vs))
    q = q if whole_queries else _pieces(q, 2)
    s = torch.einsum("bihd,bjhd->bhij", q, k) * scale
    p = torch.exp(s - s.amax(-1, keepdim=True))
    w = p[..., None] * vs.transpose(1, 2)[:, :, None]  # (B, H, Lq, T, D / 32)
    if not whole_weights:
        w = _pieces(w.float().double(), 2)
    o = torch.einsum("bhijg,bjhgd->bihgd", w, vc.unflatten(-1, (-1, 32))).flatten(-2)
    return o / p.sum(-1).transpose(1, 2)[..., None]


def _random_cache(B, T, Hkv, D, page, dtype, gen):
    M = T // page
    cache = Kv4Cache.empty(B * M, Hkv, D, page=page, dtype=dtype)
    for t in (cache.k, cache.v):
        t.random_(0, 256, generator=gen)
    for t in (cache.k_scale, cache.v_scale):
        t.copy_((torch.rand(t.shape, generator=gen, device="cuda") * 0.3 + 0.1)
                * torch.where(torch.rand(t.shape, generator=gen, device="cuda") < 0.5, -1.0, 1.0))
    table = torch.randperm(B * M, generator=gen, device="cuda").int().view(B, M).contiguous()

    def dense(t):
        return t[table.long()].transpose(2, 3).flatten(1, 2)  # (B, T, Hkv, .)

    codes = [dense(kv4_unpack(t)).double() - 8 for t in (cache.k, cache.v)]
    scales = [dense(t).double() for t in (cache.k_scale, cache.v_scale)]
    return cache, table, codes, scales


@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("B,T,Lq,H,Hkv,page", [(2, 512, 1, 8, 2, 16), (1, 512, 1, 8, 1, 32), (2, 448, 7, 6, 2, 64),
                                               (1, 256, 16, 4, 4, 128)])
def test_kv4_attention_of_fp32_states_uses_three_pieces(B, T, Lq, H, Hkv, page, D):
    """The norm of the error, in units of 2^-24 of the result's.  Scores: a group's 6 products are cut off by a half to one unit
    each, so a score is some 4 units off, 3 of its fma into the exponent and the exponential's 2; a weight's error is that times the
    score's size (1.2 times `peak`), the exponential's own 4 units and one of its last piece.  The output's sum is cut off 6
    times for 32 tokens, once or twice a warp here, and rounded some 4 times after that.  With peak 0.5 the root of their squares
    is about 8, and 12 with peak 2: 16 and 24 units are the bounds.  Without the third piece of a weight, or of a query at
    peak 2, the definition itself is beyond them, as is checked."""
    gen = torch.Generator(device="cuda").manual_seed(D + T)
    cache, table, (kc, vc), (ks, vs) = _random_cache(B, T, Hkv, D, page, F32, gen)
    k = (kc.unflatten(-1, (-1, 32)) * ks[..., None]).flatten(-2)
    q = torch.randn(B, Lq, H, D, generator=gen, device="cuda")
    for peak, bound, lost in ((0.5, 16 * 2.0 ** -24, "whole_weights"), (2.0, 24 * 2.0 ** -24, "whole_queries")):
        scale = peak * D ** -0.5
        want = _attend(q.double(), k, vc, vs, scale)
        two = _attend(q.double(), k, vc, vs, scale, **{lost: False})
        assert (two - want).norm() > bound * want.norm(), "inputs that do not tell"
        got = kv4_attention(q, cache, table, scale=scale)
        err = float((got.double() - want).norm() / want.norm())
        assert err <= bound, f"peak {peak}: {err * 2 ** 24} units"


@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("B,T,Lq,H,Hkv,page", [(2, 512, 1, 8, 2, 16), (1, 512, 1, 8, 1, 32), (2, 448, 7, 6, 2, 64)])
def test_kv4_attention_of_bf16_states_rounds_weights_and_result_alone(B, T, Lq, H, Hkv, page, D):
    """The norm of the error.  A bf16 rounding is off by up to 2^-8 of a number's power of two, evenly spread: 2^-8 / sqrt(3) of
    that in the mean of squares, 2^-9.3 of numbers that lie anywhere between two powers.  The result's and its weights' (times
    a scale) together are 2^-8.8, the scores' fp32 sums far below: 2^-8 is the bound.  Scores wrong by 0.01 would be beyond."""
    gen = torch.Generator(device="cuda").manual_seed(D + T)
    cache, table, (kc, vc), (ks, vs) = _random_cache(B, T, Hkv, D, page, BF, gen)
    k = (kc.unflatten(-1, (-1, 32)) * ks[..., None]).flatten(-2)
    q = torch.randn(B, Lq, H, D, generator=gen, device="cuda").to(BF)
    want = _attend(q.double(), k, vc, vs, D ** -0.5)
    got = kv4_attention(q, cache, table)
    assert (got.double() - want).norm() <= 2.0 ** -8 * want.norm()


def _packed(codes):
    """Bytes (..., D / 2) of codes (..., D), 0 to 15: what kv4_unpack undoes."""
    D = codes.shape[-1]
    out = torch.zeros(*codes.shape[:-1], D // 2, dtype=torch.uint8, device=codes.device)
    for d in range(D):
        block, r = divmod(d, 64)
        at = block * 64 + (r % 32 // 4 * 8 + r // 32 * 4 + r % 4 if block * 64 + 64 <= D else r)
        out[..., at // 2] |= codes[..., d] << 4 * (at % 2)
    assert torch.equal(kv4_unpack(out), codes)
    return out


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("Lq", [1, 5])
def test_kv4_attention_scores_are_exact_where_the_numbers_are_whole(D, Lq, dtype):
    """Tokens in pairs whose keys are equal, held as codes c with scale 2 and 2 c with scale 1, and whose values are opposite.
    Whole queries: every term of a score, and what is taken off it for codes that are held with 128 or 8 added, is a whole number
    that fp32 holds, so the weights of a pair are the same bits and the output is zero but for the sums' cut offs (one a
    token at most, 2^-23 of the sum).  Anything wrong in what is taken off differs by 2 between the two."""
    gen = torch.Generator(device="cuda").manual_seed(D)
    T, page, H = 256, 32, 3
    c = torch.randint(-4, 4, (T // 2, D), generator=gen, device="cuda")
    v = torch.randint(-7, 8, (T // 2, D), generator=gen, device="cuda")
    kc, vc = torch.stack((c, 2 * c), 1).flatten(0, 1), torch.stack((v, v), 1).flatten(0, 1)
    ks = torch.tensor([2.0, 1.0], device="cuda").repeat(T // 2)[:, None].expand(T, D // 32)
    vs = torch.tensor([1.0, -1.0], device="cuda").repeat(T // 2)[:, None].expand(T, D // 32)
    cache = Kv4Cache(*(_packed((t + 8).to(torch.uint8)).view(T // page, 1, page, D // 2) for t in (kc, vc)),
                     *(t.contiguous().to(BF).view(T // page, 1, page, D // 32) for t in (ks, vs)), dtype)
    table = torch.arange(T // page, device="cuda", dtype=torch.int32)[None]
    q = torch.randint(-3, 4, (1, Lq, H, D), generator=gen, device="cuda").to(dtype)
    s = torch.einsum("bihd,td->bhit", q.double(), (kc * ks.repeat_interleave(32, -1)).double()) * D ** -0.5 / 4
    most = torch.einsum("bhit,td->bihd", torch.softmax(s, -1), vc.abs().double())
    o = kv4_attention(q, cache, table, scale=D ** -0.5 / 4)
    assert float(s.std()) > 1  # weights that differ
    assert ((o.double()).abs() <= T * 2.0 ** -23 * most).all()
