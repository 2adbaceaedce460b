"""The operators that remember a history on the GPU: decaying linear attention, the paged 4-bit cache, its page tables,
against plain definitions in 64 bits.

Tolerances count roundings.  ``abs`` below is the same formula on absolute values, so it bounds every sum of
products by its terms.  bf16: the result is rounded once, and so is each weight (of tokens of a chunk) or entry of
the state that it is a sum over: 2^-8 of the result and 2^-8 of abs.  fp32 sums of n terms: n 2^-24 of abs, n the
length of the longest chain (tokens and head dim) and 256 for the decays' exponentials.
"""
import random

import pytest
import torch

import hclsm_b200
from hclsm_b200.kernels import (Kv4Cache, PageTable, decay_attention, decay_attention_step, kv4_attention, kv4_read,
                                kv4_write, page_slots, pages_resize)
from memory_ref import PagesRef, decay_grads, decay_ref, kv4_ref, kv4_unpack, kv4_values

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


# ---- decaying linear attention -----------------------------------------------------------------
def _decays(H):
    """From forgetting within a token or two to hardly at all, one without any decay, one of nothing kept."""
    g = torch.log1p(-(2.0 ** -torch.linspace(0.5, 13, H, dtype=torch.float64))).float()
    if H > 2:
        g[H // 2], g[1] = 0.0, -float("inf")
    return g.cuda()


def _inputs(B, L, H, D, Dv, dtype, state, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=gen, device="cuda")

    x = {"q": r(B, L, H, D).to(dtype), "k": (r(B, L, H, D) * D ** -0.5).to(dtype), "v": r(B, L, H, Dv).to(dtype),
         "do": r(B, L, H, Dv).to(dtype)}
    x["S0"], x["dS"] = (r(B, H, D, Dv), r(B, H, D, Dv)) if state else (None, None)
    return x


def _abs(x):
    return None if x is None else x.abs()


def _check_decay(x, g, lens, dtype, scale, run_backward=True):
    B, L, H, D = x["q"].shape
    gr = g.clamp(min=-1e30)
    leaves = {n: x[n].clone().requires_grad_() for n in ("q", "k", "v", "S0") if x[n] is not None}
    o, S = decay_attention(leaves["q"], leaves["k"], leaves["v"], g, state=leaves.get("S0"), lens=lens, scale=scale,
                           return_state=True)
    ro, rS = decay_ref(x["q"], x["k"], x["v"], gr, x["S0"], lens, scale)
    ao, aS = decay_ref(_abs(x["q"]), _abs(x["k"]), _abs(x["v"]), gr, _abs(x["S0"]), lens, scale)
    fp32 = (L + D + x["v"].shape[3] + 256) * 2.0 ** -24
    e = HALF_STEP[dtype]
    _near(o.detach(), ro, e * ro.abs() + (e + fp32) * ao, "o")
    _near(S.detach(), rS, fp32 * aS, "state")
    if not run_backward:
        return
    out, up = ((o,), (x["do"],)) if x["dS"] is None else ((o, S), (x["do"], x["dS"]))
    grads = torch.autograd.grad(out, list(leaves.values()), up)
    want = decay_grads(x["q"], x["k"], x["v"], gr, x["S0"], lens, scale, x["do"], x["dS"])
    most = decay_grads(*(_abs(x[n]) for n in ("q", "k", "v")), gr, _abs(x["S0"]), lens, scale, _abs(x["do"]), _abs(x["dS"]))
    for n, got, w, a in zip(("dq", "dk", "dv", "dS0"), grads, want, most):
        r = e if n != "dS0" else 0.0
        _near(got, w, r * w.abs() + (r + fp32) * a, n)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,L,H,D,Dv,state,ragged", [
    (1, 1, 1, 64, 64, False, False),
    (2, 1, 3, 32, 64, True, False),
    (2, 63, 4, 64, 64, True, True),
    (2, 128, 4, 64, 64, False, False),
    (3, 129, 4, 128, 128, True, True),
    (2, 333, 5, 96, 32, True, True),
    (1, 257, 3, 64, 128, True, False),
    (2, 200, 3, 128, 64, False, True),
    (1, 2500, 2, 64, 64, True, False),   # cut into segments
    (2, 1700, 3, 128, 128, True, True),
    (1, 700, 4, 8, 24, True, True),
    (2, 150, 3, 20, 7, True, True),      # rows that are not whole 16 bytes
])
def test_decay_attention(B, L, H, D, Dv, state, ragged, dtype):
    x, g = _inputs(B, L, H, D, Dv, dtype, state), _decays(H)
    lens = None
    if ragged:
        lens = torch.randint(0, L + 1, (B,), device="cuda", dtype=torch.int32)
        lens[0] = L - L // 3
    _check_decay(x, g, lens, dtype, D ** -0.5)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_decay_attention_lengths_at_chunk_borders(dtype):
    """Lengths of nothing, one, whole chunks and one token around them; what is behind them may be NaN."""
    n = [0, 1, 2, 63, 64, 65, 127, 128, 129, 191, 192, 255, 256, 257, 300, 1000]
    x, g = _inputs(len(n), 300, 3, 64, 64, dtype, True), _decays(3)
    lens = torch.tensor(n, device="cuda", dtype=torch.int32)
    for b, m in enumerate(n):
        for name in ("q", "k", "v", "do"):
            x[name][b, m:] = float("nan")
    leaves = [x[i].requires_grad_() for i in ("q", "k", "v", "S0")]
    o, S = decay_attention(*leaves[:3], g, state=leaves[3], lens=lens, return_state=True)
    grads = torch.autograd.grad((o, S), leaves, (x["do"], x["dS"]))
    for b, m in enumerate(n):
        assert (o[b, m:] == 0).all() and all((t[b, m:] == 0).all() for t in grads[:3])
        if m == 0:
            assert torch.equal(S[b], x["S0"][b])
    clean = {i: (t if t is None else torch.nan_to_num(t.detach())) for i, t in x.items()}
    _check_decay(clean, g, lens, dtype, 0.125)
    again = decay_attention(clean["q"], clean["k"], clean["v"], g, state=clean["S0"], lens=lens, return_state=True)
    assert torch.equal(again[0], o) and torch.equal(again[1], S)  # what does not count changes no bit


@pytest.mark.parametrize("dtype", [BF, F32])
def test_decay_attention_strides_and_streams(dtype):
    B, L, H, D = 2, 190, 3, 64
    x, g = _inputs(B, L, H, D, D, dtype, False), _decays(H)
    want = decay_attention(x["q"], x["k"], x["v"], g)
    packed = torch.cat((x["q"], x["k"], x["v"]), -1)  # views of one projection, heads 192 apart
    q, k, v = packed.split(D, -1)
    assert torch.equal(decay_attention(q, k, v, g), want)
    heads_first = [x[n].transpose(1, 2).contiguous().transpose(1, 2) for n in ("q", "k", "v")]
    assert torch.equal(decay_attention(*heads_first, g), want)
    odd = [torch.empty(B, L, H, D + 1, device="cuda", dtype=dtype)[..., 1:].copy_(x[n]) for n in ("q", "k", "v")]
    got = decay_attention(*odd, g)
    _near(got, want.double(), 2.0 ** -6 * want.double().abs() + 2.0 ** -6, "rows off 16 bytes")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = decay_attention(x["q"], x["k"], x["v"], g)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("L", [1, 70, 300])
def test_decay_attention_fast_decays_and_large_scores(L, dtype):
    """A token's weight is no larger than its score, whatever powers of the decay it is formed from."""
    x = _inputs(2, L, 6, 128, 128, dtype, True)
    for n in ("q", "k", "v", "do"):
        x[n] *= 64
    g = torch.tensor([-2.6, -2.7, -2.75, -2.77, -2.78, -20.0], device="cuda")
    _check_decay(x, g, None, dtype, 128 ** -0.5)
    x["S0"] = x["dS"] = None
    _check_decay(x, g, torch.tensor([L, L // 2], device="cuda", dtype=torch.int32), dtype, 128 ** -0.5)


def test_decay_attention_is_linear_in_each_argument():
    """Differences: o and the state are linear in v, so <do, o(v = u)> + <dS, S(v = u)> is the gradient in v times u, exactly but
    for rounding; likewise k and the state, and o in q."""
    B, L, H, D = 2, 300, 3, 64
    x, g = _inputs(B, L, H, D, D, F32, True), _decays(3)
    g = g.clamp(min=-50.0)
    leaves = [x[n].clone().requires_grad_() for n in ("q", "k", "v", "S0")]
    o, S = decay_attention(*leaves[:3], g, state=leaves[3], return_state=True)
    grads = torch.autograd.grad((o, S), leaves, (x["do"], x["dS"]))
    for i in range(4):
        u = torch.randn_like(x["S0"] if i == 3 else x["q"])
        at = [x["q"], x["k"], x["v"], x["S0"]]
        lo, hi = list(at), list(at)
        lo[i], hi[i] = at[i] - u, at[i] + u
        f = [decay_attention(*a[:3], g, state=a[3], return_state=True) for a in (lo, hi)]
        diff = ((f[1][0].double() - f[0][0].double()) * x["do"]).sum() + ((f[1][1].double() - f[0][1].double()) * x["dS"]).sum()
        terms = sum(((a[0].double() * x["do"]).abs().sum() + (a[1].double() * x["dS"]).abs().sum()) for a in f)
        want = 2 * (grads[i].double() * u).sum()
        assert abs(diff - want) <= 700 * 2.0 ** -24 * terms


def test_decay_attention_goes_on_from_its_state():
    """A history in two halves gives what the whole gives, and so do single tokens."""
    B, L, H, D = 2, 200, 3, 64
    x, g = _inputs(B, L, H, D, D, F32, True), _decays(H)
    whole, S = decay_attention(x["q"], x["k"], x["v"], g, state=x["S0"], return_state=True)
    a, Sa = decay_attention(*(x[n][:, :77] for n in ("q", "k", "v")), g, state=x["S0"], return_state=True)
    b, Sb = decay_attention(*(x[n][:, 77:] for n in ("q", "k", "v")), g, state=Sa, return_state=True)
    ao, aS = decay_ref(*(x[n].abs() for n in ("q", "k", "v")), g.clamp(min=-1e30), x["S0"].abs(), None, D ** -0.5)
    fp32 = 2 * (L + 2 * D + 256) * 2.0 ** -24
    _near(torch.cat((a, b), 1), whole.double(), fp32 * ao, "halves")
    _near(Sb, S.double(), fp32 * aS, "state of halves")
    state = x["S0"].clone()
    steps = torch.stack([decay_attention_step(*(x[n][:, t] for n in ("q", "k", "v")), g, state) for t in range(L)], 1)
    _near(steps, whole.double(), fp32 * ao, "steps")
    _near(state, S.double(), fp32 * aS, "state of steps")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,H,D,Dv", [(1, 1, 64, 64), (3, 5, 128, 128), (2, 3, 96, 32), (2, 4, 20, 7), (300, 6, 64, 64),
                                      (2, 2, 1, 1)])
def test_decay_attention_step(B, H, D, Dv, dtype):
    x, g = _inputs(B, 1, H, D, Dv, dtype, True), _decays(H)
    q, k, v = (x[n][:, 0] for n in ("q", "k", "v"))
    active = torch.rand(B, device="cuda") > 0.3
    active[0] = True
    ro, rS = decay_ref(x["q"], x["k"], x["v"], g.clamp(min=-1e30), x["S0"], None, 0.25)
    ao, aS = decay_ref(*(x[n].abs() for n in ("q", "k", "v")), g.clamp(min=-1e30), x["S0"].abs(), None, 0.25)
    on = active[:, None, None]
    ro, rS = torch.where(on, ro[:, 0], 0.0), torch.where(on[..., None], rS, x["S0"].double())
    state, out = x["S0"].clone(), torch.full_like(x["S0"], float("nan"))
    e, fp32 = HALF_STEP[dtype], (D + 16) * 2.0 ** -24
    o = decay_attention_step(q, k, v, g, state, out=out, active=active, scale=0.25)
    assert torch.equal(state, x["S0"])
    _near(o, ro, e * ro.abs() + fp32 * ao[:, 0], "o")
    _near(out, rS, fp32 * aS, "state")
    o2 = decay_attention_step(q, k, v, g, state, active=active, scale=0.25)
    assert torch.equal(o2, o) and torch.equal(state, out)
    assert torch.equal(state[~active], x["S0"][~active])


def test_decay_attention_backward_of_a_state_that_has_moved_on():
    """The step changes its state in place: a backward that needs the state as it was says so."""
    x, g = _inputs(2, 3, 2, 64, 32, BF, True), _decays(2)
    o = decay_attention(x["q"].requires_grad_(), x["k"], x["v"], g, state=x["S0"])
    decay_attention_step(x["k"][:, 0], x["k"][:, 0], x["v"][:, 0], g, x["S0"], out=torch.empty_like(x["S0"]))
    torch.autograd.grad(o, x["q"], x["do"], retain_graph=True)
    decay_attention_step(x["k"][:, 0], x["k"][:, 0], x["v"][:, 0], g, x["S0"])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(o, x["q"], x["do"])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_decay_attention_broadcast_inputs(dtype):
    """Dims that are expanded (strides of zero), and their gradients' sums."""
    B, L, H, D = 2, 140, 3, 64
    x, g = _inputs(B, L, H, D, D, dtype, False), _decays(H)
    k1, v1 = x["k"][:, :, :1].clone().requires_grad_(), x["v"][:1].clone().requires_grad_()
    k, v = k1.expand(B, L, H, D), v1.expand(B, L, H, D)
    o = decay_attention(x["q"], k, v, g)
    full = [t.detach().contiguous().requires_grad_() for t in (k, v)]
    want = decay_attention(x["q"], *full, g)
    fp32 = (L + 2 * D + 256) * 2.0 ** -24
    ao = decay_ref(x["q"].abs(), full[0].detach().abs(), full[1].detach().abs(), g.clamp(min=-1e30), scale=D ** -0.5)[0]
    # expanded bf16 rows go by the fp32 path: each is off the definition by its roundings
    _near(o.detach(), want.detach().double(), 4 * HALF_STEP[dtype] * (want.detach().double().abs() + ao) + 2 * fp32 * ao, "o")
    dk, dv = torch.autograd.grad(o, (k1, v1), x["do"])
    wk, wv = torch.autograd.grad(want, full, x["do"])
    assert dk.shape == k1.shape and dv.shape == v1.shape
    for got, ref in ((dk, wk.double().sum(2, keepdim=True)), (dv, wv.double().sum(0, keepdim=True))):
        assert (got.double() - ref).norm() <= (2.0 ** -6 if dtype == BF else 1e-5) * ref.norm()


def test_decay_attention_value_that_is_not_finite():
    """It reaches its own chunk and what comes behind it, in its entry and head alone."""
    x, g = _inputs(2, 500, 3, 64, 64, BF, False), torch.full((3,), -0.01, device="cuda")
    clean = decay_attention(x["q"], x["k"], x["v"], g)
    x["v"][1, 300, 1, 5] = float("nan")
    o = decay_attention(x["q"], x["k"], x["v"], g)
    assert torch.equal(o[0], clean[0]) and torch.equal(o[1, :, 0], clean[1, :, 0]) and torch.equal(o[1, :, 2], clean[1, :, 2])
    assert torch.equal(o[1, :256, 1], clean[1, :256, 1]) and o[1, 300:, 1, 5].isnan().all()


def test_decay_attention_far_offsets():
    """More than 2^31 elements: the last tokens, whose heads forget within a few, against a call on them alone."""
    L, H, D, n = 300000, 64, 128, 512
    g = torch.full((H,), -0.7, device="cuda")
    q, k, v = (torch.empty(1, L, H, D, device="cuda", dtype=BF).normal_() for _ in range(3))
    o, S = decay_attention(q, k, v, g, return_state=True)
    tail = [t[:, L - n:].contiguous() for t in (q, k, v)]
    ro, rS = decay_ref(*tail, g, scale=D ** -0.5)
    ao, aS = decay_ref(*(t.abs() for t in tail), g, scale=D ** -0.5)
    fp32 = (n + 2 * D + 256) * 2.0 ** -24
    _near(o[:, L - 200:], ro[:, -200:], 2.0 ** -8 * (ro.abs() + ao)[:, -200:] + fp32 * ao[:, -200:], "o")
    _near(S, rS, fp32 * aS, "state")
    del o, S
    v = v.requires_grad_()
    o = decay_attention(q, k, v, g)
    dv, = torch.autograd.grad(o, v, q)
    rv = decay_grads(*tail, g, None, None, D ** -0.5, tail[0], None)[2]
    av = decay_grads(*(t.abs() for t in tail), g, None, None, D ** -0.5, tail[0].abs(), None)[2]
    _near(dv[:, L - 200:], rv[:, -200:], 2.0 ** -8 * (rv.abs() + av)[:, -200:] + fp32 * av[:, -200:], "dv")


def test_two_streams_at_once():
    """Calls that run side by side on two streams, each with workspaces of its own, give what they give alone."""
    x, g = _inputs(1, 6000, 2, 64, 64, BF, False), _decays(2)  # cut into segments
    cache, table = _pool(2, 40960, 1, 64, 32, BF)
    cache.k_scale.fill_(0.25), cache.v_scale.fill_(0.5)
    q = torch.randn(2, 1, 2, 64, device="cuda", dtype=BF)  # more splits than a cluster joins
    want = decay_attention(x["q"], x["k"], x["v"], g, return_state=True), kv4_attention(q, cache, table)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((decay_attention(x["q"], x["k"], x["v"], g, return_state=True), kv4_attention(q, cache, table)))
    torch.cuda.synchronize()
    for (o, S), a in got:
        assert torch.equal(o, want[0][0]) and torch.equal(S, want[0][1]) and torch.equal(a, want[1])


def test_two_graphs_of_the_same_calls():
    """Two captured graphs, their memory in one pool, replayed in turn."""
    x, g = _inputs(1, 6000, 2, 64, 64, BF, False), _decays(2)
    cache, table = _pool(2, 40960, 1, 64, 32, BF)
    cache.k_scale.fill_(0.25), cache.v_scale.fill_(0.5)
    q = torch.randn(2, 1, 2, 64, device="cuda", dtype=BF)

    def calls():
        return decay_attention(x["q"], x["k"], x["v"], g), kv4_attention(q, cache, table)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        calls()
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(calls())
        graphs.append(graph)
    for _ in range(3):
        for t in (x["q"], x["v"], q):
            t.normal_()
        want = calls()
        for graph, out in zip(graphs, outs):
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("B,H,D", [(8, 6, 64), (1, 16, 128)])
def test_decay_attention_segments_on_busy_multiprocessors(B, H, D):
    """Segments of many chunks, blocks of several calls side by side: whichever warp is held up, no wait misses its turn."""
    x, g = _inputs(B, 4096, H, D, D, BF, False), _decays(H)

    def call():
        leaves = [x[n].detach().requires_grad_() for n in ("q", "k", "v")]
        o = decay_attention(*leaves, g)
        return (o, *torch.autograd.grad(o, leaves, x["do"]))

    want = call()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    wrong = []
    for _ in range(40):
        for s in streams:
            with torch.cuda.stream(s):
                wrong += [(a != b).any() for a, b in zip(call(), want)]
    torch.cuda.synchronize()
    assert not torch.stack(wrong).any()


def test_decay_attention_empty():
    x, g = _inputs(2, 0, 3, 64, 32, BF, True), _decays(3)
    leaves = [x[n].requires_grad_() for n in ("q", "k", "v", "S0")]
    o, S = decay_attention(*leaves[:3], g, state=leaves[3], return_state=True)
    assert o.shape == (2, 0, 3, 32) and torch.equal(S, x["S0"])
    grads = torch.autograd.grad((o, S), leaves, (x["do"], x["dS"]))
    assert torch.equal(grads[3], x["dS"])
    o, S = decay_attention(*(t.detach() for t in leaves[:3]), g, return_state=True)
    assert (S == 0).all()


def test_decay_attention_same_bits_again():
    x, g = _inputs(2, 1500, 3, 64, 64, BF, True), _decays(3)
    first = None
    for _ in range(3):
        leaves = [x[n].detach().requires_grad_() for n in ("q", "k", "v", "S0")]
        o, S = decay_attention(*leaves[:3], g, state=leaves[3], return_state=True)
        got = (o, S, *torch.autograd.grad((o, S), leaves, (x["do"], x["dS"])))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


# ---- the 4-bit cache -----------------------------------------------------------------------------
def _pool(B, T, Hkv, D, page, dtype, seed=0):
    """A cache whose pages lie scattered, with scales of NaN in the pages that no entry has, and its table."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    M = T // page
    P = B * M + 5
    cache = Kv4Cache.empty(P, Hkv, D, page=page, dtype=dtype)
    for t in (cache.k, cache.v):
        t.random_(0, 256, generator=gen)
    for t in (cache.k_scale, cache.v_scale):
        t.fill_(float("nan"))
    order = torch.randperm(P, generator=gen, device="cuda").int()
    return cache, order[:B * M].view(B, M).contiguous()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_kv4_write_and_read(D, page, dtype):
    """Codes and scales bit for bit, ties and extremes among them; what is read is what they stand for."""
    B, Hkv, n = 3, 2, 2 * page + 5
    cache, table = _pool(B, 4 * page, Hkv, D, page, dtype)
    x = [torch.randn(B, n, Hkv, D, device="cuda").to(dtype) for _ in range(2)]
    x[0][0, 0] = 0.0
    x[0][0, 1] = 1e-38
    x[0][0, 2] = 3e38
    x[0][0, 3, :, 0::2] = -3e38
    x[0][0, 4] = torch.randint(-16, 17, (Hkv, D), device="cuda") / 2.0  # ties: the scale is 1 or -1
    x[0][0, 4, :, ::32] = 8.0
    x[0][0, 5] = -x[0][0, 4]
    x[1][1, 7] *= 1e-30
    x[1][1, 8] = torch.randint(-33, 34, (Hkv, D), device="cuda") * 1.2345678
    x[1][1, 9] = 2.0 ** -130
    start = torch.tensor([0, 3, page - 1], device="cuda", dtype=torch.int32)
    count = torch.tensor([n, n - 9, 1], device="cuda", dtype=torch.int32)
    before = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    slots = page_slots(table, start, n, count=count, page=page)
    kv4_write(cache, *x, slots)
    want = [kv4_ref(t) for t in x]
    at = (slots >= 0).nonzero(as_tuple=True)
    s = slots[at].long()
    touched = torch.zeros(cache.k.shape[0], page, dtype=torch.bool, device="cuda")
    touched[s // page, s % page] = True
    for i, (q, sc) in enumerate(((cache.k, cache.k_scale), (cache.v, cache.v_scale))):
        assert torch.equal(kv4_unpack(q[s // page, :, s % page]), want[i][0][at])
        assert torch.equal(sc[s // page, :, s % page], want[i][1][at])
        keep = ~touched[:, None, :, None]
        assert torch.equal(torch.where(keep, q, 0), torch.where(keep, before[i], 0))
        assert torch.equal(torch.where(keep, sc, 0).nan_to_num(), torch.where(keep, before[2 + i], 0).nan_to_num())
    lens = torch.where(start == 0, count, 0)  # entry 0 is written from its first token
    k, v = kv4_read(cache, table, lens)
    for got, (codes, sc) in zip((k, v), want):
        assert torch.equal(got[0, :n], kv4_values(codes, sc)[0].to(dtype)) and (got[0, n:] == 0).all() and (got[1:] == 0).all()


def test_kv4_group_that_is_not_finite():
    cache, table = _pool(1, 32, 1, 64, 32, BF)
    x = torch.randn(1, 4, 1, 64, device="cuda", dtype=BF)
    x[0, 1, 0, 3], x[0, 2, 0, 40] = float("inf"), float("nan")
    kv4_write(cache, x, x, page_slots(table, torch.zeros(1, device="cuda", dtype=torch.int32), 4))
    k, v = kv4_read(cache, table, torch.tensor([4], device="cuda"))
    assert k[0, 1, 0, :32].isnan().all() and k[0, 1, 0, 32:].isfinite().all()
    assert k[0, 2, 0, 32:].isnan().all() and k[0, 2, 0, :32].isfinite().all() and k[0, 3].isfinite().all()
    assert torch.equal(k.nan_to_num(), v.nan_to_num())


def _attention_ref(q, k, v, lens, scale):
    """(o, sum of weights times |v|) over dense states (B, T, Hkv, D) in 64 bits."""
    B, Lq, H, D = q.shape
    G = H // k.shape[2]
    q, k, v = q.double(), k.double().repeat_interleave(G, 2), v.double().repeat_interleave(G, 2)
    s = torch.einsum("bihd,bjhd->bhij", q, k) * scale
    there = torch.arange(k.shape[1], device="cuda") < lens[:, None]
    s = s.masked_fill(~there[:, None, None], -torch.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    return torch.einsum("bhij,bjhd->bihd", p, v), torch.einsum("bhij,bjhd->bihd", p, v.abs())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,Lq,H,Hkv,D,page", [
    (1, 32, 1, 1, 1, 64, 32), (3, 256, 1, 6, 6, 64, 32), (2, 160, 1, 8, 2, 128, 16), (2, 192, 3, 5, 1, 96, 64),
    (2, 4096, 1, 4, 1, 64, 16), (2, 2560, 32, 6, 3, 32, 128), (1, 8192, 7, 8, 2, 128, 32), (5, 384, 1, 10, 2, 32, 32),
    (2, 1024, 17, 12, 12, 96, 16),
    (128, 96, 1, 16, 8, 32, 32), (129, 64, 1, 8, 8, 64, 16),  # several waves of blocks, equal lengths among them
    *((2, 128, Lq, 9, 3, D, 32) for D in (32, 64, 96, 128) for Lq in (1, 3))])  # each kernel: up to 8 rows, and more
def test_kv4_attention(B, T, Lq, H, Hkv, D, page, dtype):
    cache, table = _pool(B, T, Hkv, D, page, dtype)
    lens = torch.randint(0, T + 1, (B,), device="cuda", dtype=torch.int32)
    lens[0] = T - 5
    for sc in (cache.k_scale, cache.v_scale):  # only tokens that count have scales that are numbers
        dense = torch.rand(B, T, Hkv, D // 32, device="cuda") * 0.3 + 0.1
        dense *= torch.where(torch.rand_like(dense) < 0.5, -1.0, 1.0)
        for b in range(B):
            n = int(lens[b])
            ids = table[b].long()
            full = torch.where(torch.arange(T, device="cuda")[:, None, None] < n, dense[b], float("nan"))
            sc[ids] = full.view(T // page, page, Hkv, D // 32).transpose(1, 2).bfloat16()
    q = torch.randn(B, Lq, H, D, device="cuda").to(dtype)
    k, v = kv4_read(cache, table, lens)
    as32 = Kv4Cache(cache.k, cache.v, cache.k_scale, cache.v_scale, F32)
    k, v = kv4_read(as32, table, lens)  # a code times a bf16 scale is an fp32 number
    scale = D ** -0.5
    want, most = _attention_ref(q, k, v, lens, scale)
    o = kv4_attention(q, cache, table, lens)
    # scores: fp32 sums of terms as large as |q| times 144 scales (bf16: 128 + code) or |q| times the value (fp32)
    size = (144 * 0.4 if dtype == BF else 8 * 0.4) * q.double().abs().sum(-1).max() * scale
    off = 2 * (D + 8) * 2.0 ** -23 * size  # of a weight, relative, in numerator and denominator
    e = HALF_STEP[dtype]
    sums = (T / 32 + 64) * 2.0 ** -24
    _near(o, want, e * want.abs() + (e + off + sums) * most, "o")
    assert (o[lens == 0] == 0).all()
    assert torch.equal(o, kv4_attention(q, cache, table, lens))
    wide = torch.zeros(B, Lq, H + 1, 2 * D, device="cuda", dtype=dtype)
    wide[:, :, 1:, D:] = q
    assert torch.equal(o, kv4_attention(wide[:, :, 1:, D:], cache, table, lens))


def test_kv4_attention_far_pages():
    """Offsets of codes past 31 bits of bytes."""
    P, Hkv, page, D = 20000, 8, 128, 128  # 1.3 GB of codes each
    cache = Kv4Cache.empty(P * 2, Hkv, D, page=page)
    table = torch.tensor([[2 * P - 1, 0, 2 * P - 2, P]], device="cuda", dtype=torch.int32)
    k, v = (torch.randn(1, 500, Hkv, D, device="cuda", dtype=BF) for _ in range(2))
    kv4_write(cache, k, v, page_slots(table, torch.zeros(1, device="cuda", dtype=torch.int32), 500, page=page))
    lens = torch.tensor([500], device="cuda", dtype=torch.int32)
    gk, gv = kv4_read(cache, table, lens)
    for x, got in ((k, gk), (v, gv)):
        assert torch.equal(got[:, :500], kv4_values(*kv4_ref(x)).to(BF))
    small = Kv4Cache.empty(4, Hkv, D, page=page)
    first = torch.arange(4, device="cuda", dtype=torch.int32)[None]
    kv4_write(small, k, v, page_slots(first, torch.zeros(1, device="cuda", dtype=torch.int32), 500, page=page))
    q = torch.randn(1, 1, Hkv, D, device="cuda", dtype=BF)
    assert torch.equal(kv4_attention(q, cache, table, lens), kv4_attention(q, small, first, lens))


@pytest.mark.parametrize("page", [16, 32, 128])
def test_kv4_pages_outside_the_cache(page):
    """They do not count, what is there does, and the device error word says so."""
    cache, table = _pool(2, 4 * page, 1, 64, page, BF)
    cache.k_scale.fill_(0.25), cache.v_scale.fill_(0.5)
    q = torch.randn(2, 1, 2, 64, device="cuda", dtype=BF)
    lens = torch.tensor([4 * page, 3 * page - 1], device="cuda", dtype=torch.int32)
    bad = table.clone()
    bad[0, 1], bad[1, 3] = cache.k.shape[0], -1  # the second is behind its entry's length
    rest = table[0][[0, 2, 3]][None].contiguous()
    want = kv4_attention(q[:1], cache, rest, torch.tensor([3 * page], device="cuda"))
    other = kv4_attention(q, cache, table, lens)
    assert hclsm_b200.device_error() == 0
    o = kv4_attention(q, cache, bad, lens)
    assert hclsm_b200.device_error() == 1
    assert torch.equal(o[1], other[1])
    # the same weights in another order of sums
    assert (o[:1].double() - want.double()).abs().max() <= 2.0 ** -7 * want.abs().max()
    k, _ = kv4_read(cache, bad, lens)
    assert hclsm_b200.device_error() == 1
    assert (k[0, page:2 * page] == 0).all() and (k[0, 2 * page:] != 0).any()
    slots = torch.full((2, 1), cache.k.shape[0] * page, device="cuda", dtype=torch.int32)
    x = torch.ones(2, 1, 1, 64, device="cuda", dtype=BF)
    before = cache.k.clone()
    kv4_write(cache, x, x, slots)
    assert hclsm_b200.device_error() == 1
    assert torch.equal(before, cache.k)


# ---- page tables ---------------------------------------------------------------------------------
def _same(pages, ref):
    assert pages.table.tolist() == ref.table and pages.free.tolist() == ref.free and int(pages.n_free) == ref.n


@pytest.mark.parametrize("B,T,page,P", [(1, 100, 16, 7), (5, 300, 32, 40), (64, 2048, 32, 64 * 64), (1500, 200, 16, 9000),
                                        (300, 1, 128, 300), (50, 9000, 16, 20000), (1024, 700, 32, 17000)])
def test_pages_resize(B, T, page, P):
    """Random growth and shrinking against lists, requests that cannot be met among them."""
    rng = random.Random(B)
    pages = PageTable.empty(B, T, P, page=page)
    ref = PagesRef(pages.table.cpu(), pages.free.cpu(), pages.n_free, page)
    lens, met = [0] * B, 0
    room = pages.table.shape[1] * page
    for _ in range(12):
        new = [rng.choice([x, min(room, x + rng.randint(0, T)), rng.randint(0, T), 0]) for x in lens]
        ok = ref.resize(lens, new)
        pages_resize(pages, torch.tensor(lens, device="cuda"), torch.tensor(new, device="cuda"))
        assert hclsm_b200.device_error() == (0 if ok else 1)
        _same(pages, ref)
        if ok:
            lens, met = new, met + 1
    assert met
    held = [p for row in ref.table for p in row if p >= 0]
    assert len(set(held)) == len(held) and sorted(held + ref.free[:ref.n]) == list(range(P))


@pytest.mark.parametrize("columns", [256, 8192 * 32])  # a small table, and one whose pages all SMs move
def test_pages_resize_undone_and_refused(columns):
    pages = PageTable.empty(4, columns, 20, page=32)
    t = lambda *x: torch.tensor(x, device="cuda", dtype=torch.int32)  # noqa: E731
    pages_resize(pages, t(0, 0, 0, 0), t(100, 0, 33, 64))
    was = [x.clone() for x in (pages.table, pages.free, pages.n_free)]
    pages_resize(pages, t(100, 0, 33, 64), t(256, 32, 33, 65))
    pages_resize(pages, t(256, 32, 33, 65), t(100, 0, 33, 64))
    same = lambda: all(torch.equal(a, b) for a, b in zip(was, (pages.table, pages.free, pages.n_free)))  # noqa: E731
    assert same()
    for old, new in (((100, 0, 33, 64), (256, 256, 256, 64)), ((100, 0, 33, 64), (columns + 1, 0, 0, 0)),
                     ((100, 0, -1, 64), (0, 0, 0, 0)), ((100, 0, 64, 256), (100, 0, 33, 64))):
        assert hclsm_b200.device_error() == 0
        pages_resize(pages, t(*old), t(*new))  # too many, too long, negative, pages that are not held
        assert hclsm_b200.device_error() == 1
        assert same()


@pytest.mark.parametrize("n", [1, 5, 70])
def test_page_slots(n):
    table = torch.tensor([[3, 7, -1], [0, 1, 2]], device="cuda", dtype=torch.int32)
    for start, count in (((0, 31), None), ((30, 90), (n, 3)), ((-2, 2 ** 31 - 3), (n, 0)), ((95, 96), (n, n))):
        s, c = (None if x is None else torch.tensor(x, device="cuda", dtype=torch.int32) for x in (start, count))
        got = page_slots(table, s, n, count=c, page=32).tolist()
        for b in range(2):
            for i in range(n):
                at = start[b] + i
                page = table[b][at // 32].item() if 0 <= at < 96 else -1
                ok = page >= 0 and (count is None or i < count[b])
                assert got[b][i] == (page * 32 + at % 32 if ok else -1)
    assert page_slots(table, torch.zeros(2, device="cuda", dtype=torch.int64), 0).shape == (2, 0)


# ---- together ------------------------------------------------------------------------------------
def test_page_slots_of_a_page_number_that_no_slot_holds():
    """Shifted it would be some other page's slot; so it names none, and the write that is given it sets the error word."""
    table = torch.tensor([[1, (1 << 26) + 1, (1 << 26) - 1, -1]], dtype=torch.int32, device="cuda")
    slots = page_slots(table, torch.tensor([31], device="cuda"), 66, page=32)
    want = [63] + [2 ** 31 - 1] * 32 + list(range(2 ** 31 - 32, 2 ** 31)) + [-1]
    assert slots.tolist() == [want]
    assert page_slots(table, torch.tensor([0], device="cuda"), 4, page=1).tolist() == [[1, (1 << 26) + 1, (1 << 26) - 1, -1]]
    cache = Kv4Cache.empty(4, 1, 32, page=32)
    before = cache.k.clone()
    kv = torch.randn(1, 32, 1, 32, device="cuda", dtype=BF)
    kv4_write(cache, kv, kv, slots[:, 1:33])
    assert hclsm_b200.device_error() != 0 and torch.equal(cache.k, before)


def test_rollout_with_pages_cache_and_state_as_a_graph():
    """A rollout step (pages, slots, write, attention, decaying state) captured once and replayed as histories grow gives what
    eager calls give, and the values of a plain attention over what was written."""
    B, H, Hkv, D, page, steps = 3, 4, 2, 64, 16, 40
    g = _decays(H)
    gen = torch.Generator(device="cuda").manual_seed(3)
    tokens = [torch.randn(steps, B, 1, h, D, generator=gen, device="cuda", dtype=BF) for h in (H, Hkv, Hkv)]
    kh = [torch.randn(steps, B, H, D, generator=gen, device="cuda", dtype=BF) * 0.1 for _ in range(2)]

    class Rollout:
        def __init__(self):
            self.pages = PageTable.empty(B, 64, 12, page=page)
            self.cache = Kv4Cache.empty(12, Hkv, D, page=page)
            self.lens = torch.tensor([0, 5, 17], device="cuda", dtype=torch.int32)
            pages_resize(self.pages, torch.zeros_like(self.lens), self.lens)
            self.state = torch.zeros(B, H, D, D, device="cuda")
            self.x = [t[0].clone() for t in (*tokens, *kh)]

        def step(self):
            q, k, v, kd, vd = self.x
            pages_resize(self.pages, self.lens, self.lens + 1)
            kv4_write(self.cache, k, v, page_slots(self.pages.table, self.lens, 1, page=page))
            self.lens += 1
            return kv4_attention(q, self.cache, self.pages.table, self.lens), decay_attention_step(
                q[:, 0], kd, vd, g, self.state)

        def feed(self, t):
            for a, b in zip(self.x, (*tokens, *kh)):
                a.copy_(b[t])

    eager, graphed = Rollout(), Rollout()
    warm = Rollout()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        warm.step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = graphed.step()
    for t in range(steps):
        eager.feed(t), graphed.feed(t)
        want = eager.step()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), t
    assert torch.equal(graphed.pages.table, eager.pages.table) and torch.equal(graphed.lens, eager.lens)
    # entry 0 started empty: what its query sees is what was written, as the codes stand for it
    seen = [kv4_values(*kv4_ref(tokens[i][:, 0, 0]))[None] for i in (1, 2)]
    want, most = _attention_ref(tokens[0][-1][:1], *seen, torch.tensor([steps], device="cuda"), D ** -0.5)
    _near(out[0][:1], want, 2.0 ** -8 * want.abs() + 2.0 ** -7 * most, "o")
    ro, rS = decay_ref(tokens[0][:, :1, 0].transpose(0, 1), kh[0][:, :1].transpose(0, 1), kh[1][:, :1].transpose(0, 1),
                       g.clamp(min=-1e30), None, None, D ** -0.5)
    _, aS = decay_ref(*(t.abs() for t in (tokens[0][:, :1, 0].transpose(0, 1), kh[0][:, :1].transpose(0, 1), kh[1][:, :1].transpose(0, 1))), g.clamp(min=-1e30))
    _near(eager.state[:1], rS, 500 * 2.0 ** -24 * aS, "state")


def test_decay_training_step_as_a_graph():
    from hclsm_b200 import GraphedStep

    x, g = _inputs(2, 300, 3, 64, 64, BF, False), _decays(3)
    w = torch.nn.Linear(64, 64, bias=False, device="cuda", dtype=BF)

    def train():
        (decay_attention(x["q"], x["k"], w(x["v"]), g).float() * x["do"].float()).sum().backward()

    train()
    want = w.weight.grad.clone()
    step = GraphedStep(train, [w.weight])
    w.weight.grad.zero_()
    step()
    assert torch.equal(w.weight.grad, want)


def test_dispatcher_operators_give_the_functions_results():
    import hclsm_b200.torch_ops  # noqa: F401

    ops = torch.ops.hclsm_b200
    x, g = _inputs(2, 150, 3, 64, 32, BF, True), _decays(3)
    want = [x[n].detach().requires_grad_() for n in ("q", "k", "v", "S0")]
    o, S = decay_attention(*want[:3], g, state=want[3], return_state=True)
    grads = torch.autograd.grad((o, S), want, (x["do"], x["dS"]))
    got = [x[n].detach().requires_grad_() for n in ("q", "k", "v", "S0")]
    o2, S2 = ops.decay_attention_fwd(*got[:3], g, got[3], None, 0.125)
    grads2 = torch.autograd.grad((o2, S2), got, (x["do"], x["dS"]))
    assert torch.equal(o, o2) and torch.equal(S, S2) and all(torch.equal(a, b) for a, b in zip(grads, grads2))
    only = torch.autograd.grad(ops.decay_attention_fwd(*got[:3], g, got[3], None, 0.125)[1], got, x["dS"])
    ref = decay_grads(x["q"], x["k"], x["v"], g.clamp(min=-1e30), x["S0"], None, 0.125, torch.zeros_like(x["do"]), x["dS"])
    assert (only[0] == 0).all() and torch.allclose(only[3].double(), ref[3], rtol=1e-5, atol=1e-5)
    state, other = x["S0"].clone(), x["S0"].clone()
    a = ops.decay_attention_step(*(x[n][:, 0] for n in ("q", "k", "v")), g, state, None, 0.125)
    assert torch.equal(a, decay_attention_step(*(x[n][:, 0] for n in ("q", "k", "v")), g, other)) and torch.equal(state, other)
    pages = PageTable.empty(2, 64, 8)
    lens = torch.tensor([20, 40], device="cuda", dtype=torch.int32)
    none = torch.zeros_like(lens)
    ops.pages_resize(pages.table, pages.free, pages.n_free, 32, none, lens)
    assert int(pages.n_free) == 5
    cache = Kv4Cache.empty(8, 3, 64)
    k = torch.randn(2, 40, 3, 64, device="cuda", dtype=BF)
    slots = ops.page_slots(pages.table, none, 40, lens, 32)
    ops.kv4_write(cache.k, cache.v, cache.k_scale, cache.v_scale, k, k, slots)
    parts = (cache.k, cache.v, cache.k_scale, cache.v_scale, pages.table, lens)
    assert all(torch.equal(a, b) for a, b in zip(ops.kv4_read(*parts, BF), kv4_read(cache, pages.table, lens)))
    assert torch.equal(ops.kv4_attention(k[:, :1], *parts, 0.125), kv4_attention(k[:, :1], cache, pages.table, lens))
