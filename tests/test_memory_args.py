"""The operators that remember a history on the CPU: what they hand to the library and what they refuse (the device check
stubbed, the library replaced by one that records its arguments), and the tests' own reference against differences."""
import pytest
import torch
from torch.autograd import forward_ad

import hclsm_b200.torch_ops  # noqa: F401  (registers the ops)
from hclsm_b200 import _lib
from hclsm_b200.kernels import (Kv4Cache, PageTable, decay_attention, decay_attention_step, kv4_attention, kv4_read,
                                kv4_write, page_slots, pages_resize)
from hclsm_b200.kernels.decay_attn import decay_bwd
from memory_ref import decay_grads, decay_ref, kv4_ref, kv4_unpack, kv4_values

BF, I32 = torch.bfloat16, torch.int32


class _Library:
    """Records each call's arguments; workspace queries give 0."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0

        return call


@pytest.fixture
def lib(monkeypatch):
    rec = _Library()
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(_lib, "load", lambda: rec)
    monkeypatch.setattr(_lib, "stream_ptr", lambda dev: 0)
    return rec


def _refused(lib, exc, call, *args, **kw):
    with pytest.raises(exc):
        call(*args, **kw)
    assert not lib.calls


def test_reference_gradients_by_differences():
    """The written-out gradients of the tests' reference are the derivatives of its values."""
    torch.manual_seed(0)
    B, L, H, D, Dv = 2, 9, 2, 3, 4
    q, k, v = (torch.randn(B, L, H, n, dtype=torch.float64) for n in (D, D, Dv))
    S0, dS = (torch.randn(B, H, D, Dv, dtype=torch.float64) for _ in range(2))
    do, g, lens = torch.randn_like(v), torch.tensor([-0.3, 0.0]), torch.tensor([5, 9])

    def f(q, k, v, S0):
        o, S = decay_ref(q, k, v, g, S0, lens, 0.7)
        return (o * do).sum() + (S * dS).sum()

    args, h = [q, k, v, S0], 1e-6
    for i, grad in enumerate(decay_grads(q, k, v, g, S0, lens, 0.7, do, dS)):
        flat = args[i].view(-1)
        for j in range(0, flat.numel(), 5):
            at = flat[j].item()
            flat[j] = at + h
            up = f(*args)
            flat[j] = at - h
            down = f(*args)
            flat[j] = at
            assert abs((up - down) / (2 * h) - grad.reshape(-1)[j]) < 1e-6


def test_reference_is_the_recurrence():
    torch.manual_seed(1)
    q, k, v = (torch.randn(1, 6, 2, 3, dtype=torch.float64) for _ in range(3))
    g, S = torch.tensor([-0.5, -2.0]).double(), torch.randn(1, 2, 3, 3, dtype=torch.float64)
    o, last = decay_ref(q, k, v, g, S, None, 0.5)
    for t in range(6):
        S = S * g.exp().view(1, 2, 1, 1) + k[:, t, :, :, None] * v[:, t, :, None]
        assert torch.allclose(o[:, t], 0.5 * (q[:, t, :, None] @ S)[:, :, 0])
    assert torch.allclose(S, last)


def test_packing_of_codes():
    """Dims 0 to 3 and 32 to 35 share the first word; 32 dims behind the last 64 are in order."""
    b = torch.zeros(48, dtype=torch.uint8)
    b[0], b[1], b[2], b[3] = 0x10, 0x32, 0x54, 0x76
    b[32], b[47] = 0x21, 0xfe
    c = kv4_unpack(b)
    assert c[:4].tolist() == [0, 1, 2, 3] and c[32:36].tolist() == [4, 5, 6, 7]
    assert c[64:66].tolist() == [1, 2] and c[94:].tolist() == [14, 15]


def test_codes_of_ties_and_zeros():
    x = torch.zeros(3, 32)
    x[0, :6] = torch.tensor([8.0, 0.5, 1.5, -8.0, -7.5, -0.5])
    x[1, :5] = torch.tensor([-8.0, 0.5, 1.5, 7.5, 7.4])
    codes, scale = kv4_ref(x)
    assert scale.flatten().tolist() == [-1.0, 1.0, 0.0]
    assert kv4_values(codes, scale)[0, :6].tolist() == [8.0, 0.0, 2.0, -7.0, -7.0, 0.0]
    assert kv4_values(codes, scale)[1, :5].tolist() == [-8.0, 0.0, 2.0, 7.0, 7.0]
    assert (kv4_values(codes, scale)[2] == 0).all()


def _qkv(**kw):
    x = {"q": torch.zeros(2, 5, 3, 64, dtype=BF), "k": torch.zeros(2, 5, 3, 64, dtype=BF),
         "v": torch.zeros(2, 5, 3, 32, dtype=BF), "log_decay": torch.zeros(3), "state": torch.zeros(2, 3, 64, 32)}
    return {**x, **kw}


def _decay(x, **kw):
    return decay_attention(x["q"], x["k"], x["v"], x["log_decay"], state=x["state"], **kw)


def test_decay_attention_arguments(lib):
    x = _qkv()
    o, s = _decay(x, return_state=True)
    assert o.shape == (2, 5, 3, 32) and s.shape == (2, 3, 64, 32) and s.dtype == torch.float32
    name, args = lib.calls[-1]
    a = _lib.DECAY_ARGS.unpack(args[0])
    assert name == "hclsm_decay_attn_fwd" and len(args[0]) == 4 * 32 + 10 * 8 + 7 * 4
    assert a[0] == x["q"].data_ptr() and a[1:4] == (960, 192, 64) and a[12] == 0
    assert a[16] == o.data_ptr() and a[20] == x["log_decay"].data_ptr() and a[22] == s.data_ptr()
    assert a[26:32] == (2, 5, 3, 64, 32, _lib.BF16) and a[32] == 0.125
    assert torch.is_tensor(_decay(x))
    # a state that may not be written as it is: a copy
    _decay(_qkv(state=torch.zeros(2, 3, 32, 64).transpose(2, 3)))


def test_decay_attention_refusals(lib):
    z = torch.zeros
    for bad in (dict(k=z(2, 5, 3, 32, dtype=BF)), dict(v=z(2, 4, 3, 32, dtype=BF)), dict(v=z(2, 5, 2, 32, dtype=BF)),
                dict(q=z(2, 5, 3, 160, dtype=BF), k=z(2, 5, 3, 160, dtype=BF)), dict(v=z(2, 5, 3, 129, dtype=BF)),
                dict(log_decay=z(2)), dict(log_decay=z(3, dtype=BF)), dict(log_decay=z(3, dtype=torch.float64)),
                dict(state=z(2, 3, 32, 64)), dict(state=z(2, 3, 64, 32, dtype=BF)), dict(q=z(2, 3, 64, dtype=BF))):
        _refused(lib, ValueError, _decay, _qkv(**bad))
    for bad in (dict(k=z(2, 5, 3, 64)), dict(v=z(2, 5, 3, 32)),
                {n: z(2, 5, 3, 64, dtype=torch.float16) for n in ("q", "k")} | dict(v=z(2, 5, 3, 32, dtype=torch.float16))):
        _refused(lib, TypeError, _decay, _qkv(**bad))
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        _refused(lib, ValueError, _decay, _qkv(), scale=scale)
    _refused(lib, ValueError, _decay, _qkv(), lens=z(3, dtype=I32))
    _refused(lib, TypeError, _decay, _qkv(), lens=z(2))
    _refused(lib, NotImplementedError, _decay, _qkv(log_decay=z(3, requires_grad=True)))
    with torch.no_grad():
        _decay(_qkv(log_decay=z(3, requires_grad=True)))
    with forward_ad.dual_level():
        lib.calls.clear()
        q = forward_ad.make_dual(_qkv()["q"], torch.ones(2, 5, 3, 64, dtype=BF))
        _refused(lib, NotImplementedError, _decay, _qkv(q=q))


def test_decay_attention_has_no_second_derivative(lib):
    x = _qkv(v=torch.zeros(2, 5, 3, 32, dtype=BF, requires_grad=True))
    o = _decay(x)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(o.sum(), x["v"], create_graph=True)


def test_decay_attention_gradients_that_are_asked_for(lib):
    """The state's gradient only where it is wanted; an output that is not used has none."""
    x = _qkv(state=torch.zeros(2, 3, 64, 32, requires_grad=True), v=torch.zeros(2, 5, 3, 32, dtype=BF, requires_grad=True))
    o, s = _decay(x, return_state=True)
    torch.autograd.grad(s.sum(), (x["v"], x["state"]))
    a = _lib.DECAY_ARGS.unpack(lib.calls[-1][1][0])
    assert lib.calls[-1][0] == "hclsm_decay_attn_bwd" and a[23] and a[24]
    o, s = _decay(_qkv(v=x["v"]), return_state=True)
    torch.autograd.grad(o.sum(), x["v"])
    a = _lib.DECAY_ARGS.unpack(lib.calls[-1][1][0])
    assert not a[23] and not a[24]
    for name, bad, exc in (("do", torch.zeros(2, 5, 3, 64, dtype=BF), ValueError), ("do", torch.zeros(2, 5, 3, 32), TypeError),
                           ("dstate", torch.zeros(2, 3, 32, 64), ValueError),
                           ("dstate", torch.zeros(2, 3, 64, 32, dtype=BF), TypeError)):
        lib.calls.clear()
        t = {"do": torch.zeros(2, 5, 3, 32, dtype=BF), "dstate": None, name: bad}
        y = _qkv()
        _refused(lib, exc, decay_bwd, y["q"], y["k"], y["v"], y["log_decay"], y["state"], None, None, t["do"], t["dstate"])


def _step(**kw):
    z = torch.zeros
    x = dict(q=z(2, 3, 64), k=z(2, 3, 64), v=z(2, 3, 32), g=z(3), state=z(2, 3, 64, 32))
    x.update({n: kw.pop(n) for n in tuple(kw) if n in x})
    return decay_attention_step(x["q"], x["k"], x["v"], x["g"], x["state"], **kw)


def test_decay_step_arguments_and_refusals(lib):
    z = torch.zeros
    state, out = z(2, 3, 64, 32), z(2, 3, 64, 32)
    assert _step(state=state).shape == (2, 3, 32)
    a = _lib.DECAY_ARGS.unpack(lib.calls[-1][1][0])
    assert a[21] == a[22] == state.data_ptr() and a[26:32] == (2, 1, 3, 64, 32, _lib.F32)
    _step(state=state, out=out)
    a = _lib.DECAY_ARGS.unpack(lib.calls[-1][1][0])
    assert a[21] == state.data_ptr() and a[22] == out.data_ptr()
    lib.calls.clear()
    two = z(3, 3, 64, 32)
    for kw in (dict(state=two[:2], out=two[1:]), dict(out=z(2, 3, 32, 64)), dict(out=z(2, 3, 64, 32, dtype=BF)),
               dict(state=z(2, 3, 32, 64).transpose(2, 3)), dict(out=z(2, 3, 32, 64).transpose(2, 3)),
               dict(active=z(2)), dict(active=z(3, dtype=torch.bool)), dict(k=z(2, 3, 32)), dict(v=z(2, 2, 32)), dict(g=z(2)),
               dict(q=z(2, 3, 200), k=z(2, 3, 200)), dict(scale=0.0), dict(state=z(2, 3, 64, 64))):
        _refused(lib, ValueError, _step, **kw)
    _refused(lib, TypeError, _step, v=z(2, 3, 32, dtype=BF))
    for n, shape in (("q", (2, 3, 64)), ("v", (2, 3, 32)), ("state", (2, 3, 64, 32)), ("out", (2, 3, 64, 32)), ("g", (3,))):
        _refused(lib, NotImplementedError, _step, **{n: z(*shape, requires_grad=True)})


def _cache(**kw):
    return Kv4Cache.empty(7, 2, 64, page=16, device="cpu", **kw)


def test_kv4_arguments(lib):
    c, x = _cache(), torch.zeros(3, 4, 2, 64, dtype=BF)
    table, slots = torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 4, dtype=I32)
    kv4_write(c, x, x, slots)
    k, v = kv4_read(c, table)
    assert k.shape == v.shape == (3, 32, 2, 64) and k.dtype == BF
    assert kv4_attention(x.repeat(1, 1, 3, 1), c, table, torch.zeros(3)[:].to(I32)).shape == (3, 4, 6, 64)
    seen = {n: a for n, a in lib.calls}
    for n in ("hclsm_kv4_write", "hclsm_kv4_read", "hclsm_kv4_attn"):
        a = _lib.KV4_CACHE.unpack(seen[n][0])
        assert a == (c.k.data_ptr(), c.v.data_ptr(), c.k_scale.data_ptr(), c.v_scale.data_ptr(), 7, 2, 16, 64, _lib.BF16)
    # tensors that were assigned since: the present ones
    c.k = c.k.clone()
    kv4_write(c, x, x, slots)
    assert _lib.KV4_CACHE.unpack(lib.calls[-1][1][0])[0] == c.k.data_ptr()


def test_kv4_refusals(lib):
    z = torch.zeros
    x, slots, table = z(3, 4, 2, 64, dtype=BF), z(3, 4, dtype=I32), z(3, 2, dtype=I32)
    for name, bad in (("v", lambda t: t[:6]), ("k", lambda t: t.int()), ("k_scale", lambda t: t.float()),
                      ("v_scale", lambda t: t[:, :1]), ("k", lambda t: t.transpose(1, 2)), ("k", lambda t: t[..., :24])):
        c = _cache()
        setattr(c, name, bad(getattr(c, name)))
        for call in (lambda: kv4_write(c, x, x, slots), lambda: kv4_read(c, table), lambda: kv4_attention(x, c, table)):
            _refused(lib, ValueError, call)
    c = _cache()
    _refused(lib, TypeError, _cache, dtype=torch.float16)
    for kw in (dict(page=24), dict(head_dim=48), dict(kv_heads=0)):
        _refused(lib, ValueError, Kv4Cache.empty, **{**dict(pages=3, kv_heads=1, head_dim=64, device="cpu"), **kw})
    for kw in (dict(page=24), dict(page=0), dict(pages=-1), dict(max_tokens=-1)):
        _refused(lib, ValueError, PageTable.empty, **{**dict(batch=2, max_tokens=64, pages=4, device="cpu"), **kw})
    for k, s in ((x[:, :, :1], slots), (x[..., :32], slots), (x, slots[:, :3]), (x, None)):
        _refused(lib, ValueError, kv4_write, c, k, k, s)
    _refused(lib, ValueError, kv4_write, c, x, x[:, :3], slots)
    _refused(lib, TypeError, kv4_write, c, x.float(), x.float(), slots)
    _refused(lib, TypeError, kv4_write, c, x, x, slots.float())
    for q, t in ((x[:2], table), (x[:, :, :1], table), (x[..., :32], table), (x, table[0])):
        _refused(lib, ValueError, kv4_attention, q, c, t)
    _refused(lib, ValueError, kv4_attention, x, c, table, z(2, dtype=I32))
    _refused(lib, ValueError, kv4_attention, x, c, table, scale=-1.0)
    _refused(lib, TypeError, kv4_attention, x.float(), c, table)
    _refused(lib, TypeError, kv4_read, c, table.float())
    r = x.clone().requires_grad_()
    _refused(lib, NotImplementedError, kv4_write, c, r, x, slots)
    _refused(lib, NotImplementedError, kv4_attention, r, c, table)
    with torch.no_grad():
        kv4_attention(r, c, table)
    with forward_ad.dual_level():
        lib.calls.clear()
        _refused(lib, NotImplementedError, kv4_attention, forward_ad.make_dual(x, x), c, table)


def test_pages_arguments_and_refusals(lib):
    z = torch.zeros
    p = PageTable.empty(3, 100, 9, page=32, device="cpu")
    assert p.table.shape == (3, 4) and p.free.tolist() == list(range(8, -1, -1)) and p.n_free.tolist() == [9]
    lens = z(3, dtype=torch.int64)
    pages_resize(p, lens, lens)
    name, a = lib.calls[-1]
    assert name == "hclsm_pages_resize" and a[:7] == (p.table.data_ptr(), 3, 4, p.free.data_ptr(), p.n_free.data_ptr(), 9, 32)
    assert page_slots(p.table, lens, 5).shape == (3, 5)
    lib.calls.clear()
    for bad in (dict(table=p.table.long()), dict(table=p.table.t()), dict(table=p.table[0]), dict(free=p.free.long()),
                dict(free=p.free[::2]), dict(n_free=z(2, dtype=I32)), dict(n_free=z(1)), dict(page=24), dict(page=0)):
        q = PageTable(**{**dict(table=p.table, free=p.free, n_free=p.n_free, page=32), **bad})
        _refused(lib, ValueError, pages_resize, q, lens, lens)
    _refused(lib, ValueError, pages_resize, p, lens[:2], lens)
    _refused(lib, ValueError, pages_resize, p, lens, None)
    _refused(lib, TypeError, pages_resize, p, lens.float(), lens)
    for kw in (dict(page=48), dict(n=-1), dict(start=lens[:1]), dict(start=None), dict(count=lens[:1]), dict(table=p.table[0])):
        a = {**dict(table=p.table, start=lens, n=2), **kw}
        _refused(lib, ValueError, page_slots, a.pop("table"), a.pop("start"), a.pop("n"), **a)


def test_c_entries_refuse_on_the_host():
    """Status codes of the library itself, before anything reaches a GPU."""
    lib = _lib.load()
    none = (0, 0, 0, 0)

    def decay(B=1, L=4, H=1, D=64, Dv=64, dtype=_lib.BF16, scale=1.0):
        return _lib.DECAY_ARGS.pack(*none * 4, *(0,) * 10, B, L, H, D, Dv, dtype, scale)

    for kw, rc in ((dict(D=129), 1), (dict(Dv=0), 1), (dict(H=0), 1), (dict(B=-1), 1), (dict(scale=0.0), 1),
                   (dict(scale=float("nan")), 1), (dict(dtype=2), 2), (dict(), 8), (dict(B=0), 0)):
        for f in (lib.hclsm_decay_attn_fwd, lib.hclsm_decay_attn_bwd):
            assert f(decay(**kw), None, 0, None) == rc, kw
        assert lib.hclsm_decay_attn_step(decay(**kw), None, None) == rc, kw
    assert lib.hclsm_decay_attn_fwd(None, None, 0, None) == 8

    def cache(pages=4, Hkv=1, page=32, D=64, dtype=_lib.BF16, p=0):
        return _lib.KV4_CACHE.pack(p, p, p, p, pages, Hkv, page, D, dtype)

    for kw, rc in ((dict(page=24), 1), (dict(D=48), 1), (dict(D=256), 1), (dict(Hkv=0), 1), (dict(dtype=7), 2), (dict(), 8),
                   (dict(p=8), 3), (dict(pages=1 << 27), 1)):
        assert lib.hclsm_kv4_read(cache(**kw), None, 1, 1, None, None, None, None) == rc, kw
        assert lib.hclsm_kv4_write(cache(**kw), None, None, None, 1, 1, None) == rc, kw
        assert lib.hclsm_kv4_attn(cache(**kw), None, 1, 1, None, None, None, 1, 1, 1.0, None, 0, None) == rc, kw
    assert lib.hclsm_pages_resize(None, 1, 1, None, None, 1, 24, None, None, None, 0, None) == 1
    assert lib.hclsm_pages_resize(None, 1, 1, None, None, 1, 32, None, None, None, 0, None) == 8
    assert lib.hclsm_pages_resize(None, 1, 1, None, None, 1 << 27, 32, None, None, None, 0, None) == 1
    assert lib.hclsm_pages_resize_workspace_size(64, 64) == 0 and lib.hclsm_pages_resize_workspace_size(64, 2048) > 0
    assert lib.hclsm_pages_resize(16, 64, 2048, 16, 16, 9, 32, 16, 16, None, 0, None) == 4
    assert lib.hclsm_page_slots(None, 1, 1, 32, None, None, 4, None, None) == 8
    assert lib.hclsm_page_slots(None, 1, 1, 31, None, None, 4, None, None) == 1
    assert lib.hclsm_page_slots(None, 1, 1, 32, None, None, 0, None, None) == 0


def test_dispatcher_operators_trace_and_refuse(lib):
    """Shapes under fake tensors; what mutates takes detached tensors; no gradient of log_decay."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops, z = torch.ops.hclsm_b200, torch.zeros
    with FakeTensorMode():
        q, v = z(2, 5, 3, 64, dtype=BF), z(2, 5, 3, 32, dtype=BF)
        o, s = ops.decay_attention_fwd(q, q, v, z(3), None, None, 0.125)
        assert o.shape == v.shape and o.dtype == BF and s.shape == (2, 3, 64, 32) and s.dtype == torch.float32
        g = ops.decay_attention_bwd(q, q, v, z(3), s, None, 0.125, v, None)
        assert [t.shape for t in g] == [q.shape, q.shape, v.shape, s.shape]
        codes, scale = z(7, 3, 16, 32, dtype=torch.uint8), z(7, 3, 16, 2, dtype=BF)
        table = z(2, 4, dtype=I32)
        k, _ = ops.kv4_read(codes, codes, scale, scale, table, None, torch.float32)
        assert k.shape == (2, 64, 3, 64) and k.dtype == torch.float32
        assert ops.kv4_attention(q, codes, codes, scale, scale, table, None, 0.125).shape == q.shape
        assert ops.page_slots(table, z(2, dtype=I32), 6, None, 16).shape == (2, 6)
        assert ops.decay_attention_step(q[:, 0], q[:, 0], v[:, 0], z(3), s, None, 0.125).shape == (2, 3, 32)
    x = _qkv(q=z(2, 5, 3, 64, dtype=BF, requires_grad=True))
    with pytest.raises(NotImplementedError):
        ops.decay_attention_fwd(x["q"], x["k"], x["v"], z(3, requires_grad=True), None, None, 0.125)
    c = _cache()
    k = z(3, 4, 2, 64, dtype=BF, requires_grad=True)
    with pytest.raises(NotImplementedError):
        ops.kv4_write(c.k, c.v, c.k_scale, c.v_scale, k, k, z(3, 4, dtype=I32))
    with pytest.raises(NotImplementedError):
        ops.decay_attention_step(z(2, 3, 64, requires_grad=True), z(2, 3, 64), z(2, 3, 32), z(3), z(2, 3, 64, 32), None, 1.0)
