"""The operators that remember a history on the GPU: calls at the edges of what they are documented to take, against plain
definitions in 64 bits.  Tolerances count roundings as test_memory_ops_gpu.py does."""
import pytest
import torch

import hclsm_b200
from hclsm_b200.kernels import (Kv4Cache, PageTable, decay_attention, decay_attention_step, kv4_attention, kv4_write,
                                pages_resize)
from hclsm_b200.kernels.decay_attn import decay_bwd
from memory_ref import decay_grads, decay_ref

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
HALF_STEP = {BF: 2.0 ** -8, F32: 2.0 ** -24}  # eps / 2


@pytest.fixture(autouse=True)
def no_device_error():
    hclsm_b200.device_error()
    yield
    assert hclsm_b200.device_error() == 0


def _near(got, want, tol, name):
    assert got.shape == want.shape, name
    over = ((got.double() - want).abs() - tol).max()
    assert over <= 0, f"{name}: {float(over)} over its tolerance"
    assert torch.isfinite(got).all(), name


# ---- scales -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,L,H,D,Dv", [(2, 150, 6, 64, 64), (1, 2500, 6, 64, 64), (40, 200, 6, 64, 64), (1, 1700, 6, 128, 128),
                                        (2, 150, 6, 20, 8)])
@pytest.mark.parametrize("scale,up,dstate", [(1e-39, 1.0, 1.0), (1e-20, 1.0, 1e30), (64.0, 1.0, 1.0), (1e20, 1e-20, 1.0)])
def test_decay_attention_gradients_of_any_scale(B, L, H, D, Dv, scale, up, dstate, dtype):
    """The final state's gradient reaches k, v and the first state without the scale, however small that is; the other
    terms have it.  Decays on both sides of where the powers on the diagonal are formed in two ways."""
    gen = torch.Generator(device="cuda").manual_seed(5)

    def r(*s, f=1.0):
        return torch.randn(*s, generator=gen, device="cuda") * f

    q, k, v = r(B, L, H, D).to(dtype), r(B, L, H, D, f=D ** -0.5).to(dtype), r(B, L, H, Dv).to(dtype)
    do, S0, dS = r(B, L, H, Dv, f=up).to(dtype), r(B, H, D, Dv), r(B, H, D, Dv, f=dstate)
    g = torch.tensor([-0.01, -2.6, -2.65, -2.75, -2.78, -20.0], device="cuda")
    leaves = [t.requires_grad_() for t in (q, k, v, S0)]
    o, S = decay_attention(q, k, v, g, state=S0, scale=scale, return_state=True)
    grads = torch.autograd.grad((o, S), leaves, (do, dS))
    q, k, v, S0 = (t.detach() for t in leaves)
    fp32, e = (L + D + Dv + 256) * 2.0 ** -24, HALF_STEP[dtype]
    want = decay_grads(q, k, v, g, S0, None, scale, do, dS)
    most = decay_grads(q.abs(), k.abs(), v.abs(), g, S0.abs(), None, scale, do.abs(), dS.abs())
    # a power of a decay below 2^-126 is zero, times the product of a row (entries below 8) and the gradient of the state; and
    # each bf16 weight below 2^-126 (of 128 in a chunk, or of the state) is off by 2^-134, times a row's entry, which is less
    low = 2.0 ** -126 * 128 * 8 * max(8.0, float(dS.abs().max()))
    for n, got, w, m in zip(("dq", "dk", "dv", "dS0"), grads, want, most):
        half = e if n != "dS0" else 0.0
        _near(got, w, half * w.abs() + (half + fp32) * m + low, n)


# ---- one token after another ----------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
def test_decay_attention_step_forgets_at_the_rate_it_is_given(dtype):
    """Slow heads over 4096 tokens against the recurrence in 64 bits.  A token rounds each value of the state once, by at most
    2^-24 of it and on either side alike: over n tokens the roundings' sum is some sqrt(n / 3) 2^-24 and, over a few
    thousand values, hardly ever above six times that.  A decay of one fp32 number is up to n 2^-25 off, always the same way."""
    n, H, D = 4096, 6, 16
    g = torch.tensor([-1e-3, -2.0 ** -12, -1e-5, -1e-6, -3e-7, 0.0], device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(7)
    q, k, v = (torch.randn(n, 1, H, D, generator=gen, device="cuda").to(dtype) for _ in range(3))
    k *= 1e-3  # the first state is most of what is there
    state = torch.rand(1, H, D, D, generator=gen, device="cuda") + 1
    want, decay, most = state.double(), g.double().exp().view(1, H, 1, 1), state.double()
    for t in range(n):
        want = decay * want + k[t].double()[..., None] * v[t].double()[..., None, :]
        most = torch.maximum(most, want.abs())
        o = decay_attention_step(q[t], k[t], v[t], g, state, scale=1.0)
    tol = 6 * (n / 3) ** 0.5 * 2.0 ** -24
    assert tol < 1.4e-5
    # bf16: a product's last bit may be 2^-24, half the state's.  Of a head that loses less than a bit of what it loses a token
    # over the whole run (1e-6: 8 to 16 bits a token, 4096 1e-6 of that over the run) the rest is then the same at every
    # token and so is its rounding: such heads are compared in fp32 alone.
    heads = [0, 1, 2, 5] if dtype == BF else list(range(H))
    _near(state[:, heads], want[:, heads], tol * most[:, heads], "state")
    o, want, most, q = o[:, heads], want[:, heads], most[:, heads], q[:, :, heads]
    terms = torch.einsum("bhi,bhij->bhj", q[-1].double().abs(), most)
    _near(o, torch.einsum("bhi,bhij->bhj", q[-1].double(), want), (tol + (D + 16) * 2.0 ** -24 + HALF_STEP[dtype]) * terms, "o")
    # with next to nothing added a whole history of tokens is one factor
    state = torch.rand(1, H, D, D, generator=gen, device="cuda") + 1
    first, none = state.double(), torch.zeros_like(k[0])
    for t in range(n):
        decay_attention_step(none, none, none, g, state)
    want = (g.double() * n).exp().view(1, H, 1, 1) * first
    _near(state[:, [0, 1, 5]], want[:, [0, 1, 5]], tol * want[:, [0, 1, 5]], "state")


# ---- lengths next to 2^31 -------------------------------------------------------------------------
def test_decay_attention_of_31_bits_of_tokens():
    """One number a token, fp32: what the last tokens see is the sum over all before, and what is behind the length is zero.
    Heads that forget: a token sees no more than some 60 others, in chunks of 64 by n = 400 terms' rounding."""
    L, n, g = (1 << 31) - 1, 1000, torch.tensor([-0.7], device="cuda")
    q, k, v = (torch.full((1, 1, 1, 1), x, device="cuda").expand(1, L, 1, 1) for x in (2.0, 0.5, 3.0))
    tail = [t[:, :n] for t in (q, k, v)]
    ro, rS = decay_ref(*tail, g, scale=0.25)
    tol = 400 * 2.0 ** -24
    lens = torch.tensor([L - 5], device="cuda")
    o, S = decay_attention(q, k, v, g, scale=0.25, lens=lens, return_state=True)
    _near(o[:, L - 305:L - 5], ro[:, -300:], tol * ro[:, -300:], "o")
    assert (o[:, L - 5:] == 0).all()
    _near(S, rS, tol * rS, "state")
    del o
    want = decay_grads(*tail, g, None, None, 0.25, tail[2], None)
    got = decay_bwd(q, k, v, g, None, None, 0.25, v, None)
    for a, w, name in zip(got, want, ("dq", "dk", "dv")):
        _near(a[:, L - 300:], w[:, -300:], tol * w[:, -300:], name)
        first = w[:, :300] if name == "dq" else w[:, 300:600]  # dq looks back, the others ahead
        _near(a[:, :300], first, tol * first, name)


def test_decay_attention_of_31_bits_of_tokens_on_the_tensor_cores():
    """Rows of 16 bytes, bf16, all but the last zeros: the last chunks and the state behind them."""
    L, n, g = (1 << 31) - 1, 5000, torch.tensor([-0.01], device="cuda")
    x = torch.zeros(1, L, 1, 8, device="cuda", dtype=BF)
    x[:, L - n:].normal_()
    tail = x[:, L - n:].clone()
    o, S = decay_attention(x, x, x, g, return_state=True)
    ro, rS = decay_ref(tail, tail, tail, g, scale=8 ** -0.5)
    ao, aS = decay_ref(*(tail.abs(),) * 3, g, scale=8 ** -0.5)
    fp32 = (n + 2 * 8 + 256) * 2.0 ** -24
    _near(o[:, L - n:], ro, 2.0 ** -8 * (ro.abs() + ao) + fp32 * ao, "o")
    _near(S, rS, fp32 * aS, "state")
    assert (o[:, :L - n] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_kv4_attention_of_31_bits_of_tokens(dtype):
    """Pages of 16 that repeat, 2^31 - 16 tokens: all scores are zero but those of the last page, whose tokens weigh as much as
    all others.  The sums of these weights and values are exact in fp32; e^18.75 is off by 2^-20 of it."""
    M = (1 << 27) - 1
    cache = Kv4Cache.empty(2, 1, 32, page=16, dtype=dtype)
    k, v = (torch.zeros(1, 32, 1, 32, device="cuda", dtype=dtype) for _ in range(2))
    k[:, 16:, :, 0], v[:, :16], v[:, 16:] = 8.0, 1.0, 3.0  # held exactly
    kv4_write(cache, k, v, torch.arange(32, device="cuda", dtype=torch.int32)[None])
    table = torch.zeros(1, M, device="cuda", dtype=torch.int32)
    table[0, -1] = 1
    q = torch.zeros(1, 1, 1, 32, device="cuda", dtype=dtype)
    q[..., 0] = 18.75 / 8
    for lens in (None, torch.tensor([16 * M - 1], device="cuda")):
        last = 16 if lens is None else 15
        e = last * torch.tensor(18.75, dtype=torch.float64).exp()
        want = ((M - 1) * 16 + 3 * e) / ((M - 1) * 16 + e)
        got = kv4_attention(q, cache, table, lens, scale=1.0)
        assert (got.double() - want.cuda()).abs().max() <= (2 * HALF_STEP[dtype] + 2.0 ** -18) * want


# ---- page tables ------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,columns", [(1, 256), (4, 256), (300, 64), (2000, 64), (4, 8192 * 32), (1024, 1024)])
def test_pages_are_not_lost_where_the_old_lengths_fall_short(B, columns):
    """A growth that is asked for again with the lengths from before it, or with lengths that understate one entry, changes
    nothing and sets the error word, in each of the kernels (one block, a cluster, several rounds of entries, all SMs)."""
    pages = PageTable.empty(B, columns, 5 * B + 7, page=32)
    gen = torch.Generator(device="cuda").manual_seed(B)
    old = torch.randint(0, 33, (B,), generator=gen, device="cuda", dtype=torch.int32)
    pages_resize(pages, torch.zeros_like(old), old)
    new = old + 33 if columns > 64 else torch.full_like(old, 64)
    pages_resize(pages, old, new)
    assert hclsm_b200.device_error() == 0
    parts = pages.table, pages.free, pages.n_free
    was = [t.clone() for t in parts]

    def refused(a, b):
        pages_resize(pages, a, b)
        assert hclsm_b200.device_error() == 1
        assert all(torch.equal(x, y) for x, y in zip(was, parts))

    refused(old, new)  # the same call again
    last = new.clone()
    last[B - 1] = 0  # one entry that has pages is said to have none, the others give theirs up
    refused(last, torch.where(torch.arange(B, device="cuda") == B - 1, 40, 0))
    pages_resize(pages, new, old)  # the lengths as they are
    pages_resize(pages, old, new)
    assert hclsm_b200.device_error() == 0
    assert all(torch.equal(x, y) for x, y in zip(was, parts))
    held = torch.cat((pages.table[pages.table >= 0], pages.free[:int(pages.n_free)]))
    assert torch.equal(held.sort().values, torch.arange(5 * B + 7, device="cuda", dtype=torch.int32))
