"""What the attention operators hand to the library, and what they refuse, seen on the CPU: the device check is stubbed
and the library replaced by one that records its arguments."""
import copy
import io
import pickle

import pytest
import torch
from torch.autograd import forward_ad

import hclsm_b200.torch_ops  # noqa: F401  (registers the ops)
from hclsm_b200 import _lib
from hclsm_b200.kernels import Kv8Cache, cross_attention, kv8_attention, kv8_read, kv8_write, qk_norm_rope
from hclsm_b200.kernels.cross_attn import attention_bwd


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


NAMES = ("k", "v", "k_scale", "v_scale", "k_tail", "v_tail")


def _cache(**kw):
    return Kv8Cache.empty(2, 64, 1, 32, device="cpu", **kw)


def _addresses(cache):
    return [getattr(cache, n).data_ptr() for n in NAMES]


def _uses_its_own(lib, cache):
    """Every call on the cache gets the addresses of the tensors that it has now."""
    B, Hkv, T, D = cache.k.shape
    x = torch.zeros(B, 3, Hkv, D, dtype=cache.dtype)
    at = torch.zeros(B, dtype=torch.int32)
    lib.calls.clear()
    kv8_write(cache, x, x, at)
    kv8_read(cache, at)
    o = kv8_attention(x, cache, at)
    assert o.shape[0] == B
    seen = {n: _lib.KV8_CACHE.unpack(a[0]) for n, a in lib.calls}
    assert {"hclsm_kv8_write", "hclsm_kv8_read", "hclsm_kv8_attn"} <= set(seen)
    for n, c in seen.items():
        assert list(c[:6]) == _addresses(cache), n
        assert c[6:] == (B, Hkv, T, D, cache.block, _lib.BF16), n


def test_cache_copies_use_their_own_memory(lib):
    cache = _cache()
    _uses_its_own(lib, cache)
    file = io.BytesIO()
    torch.save(cache, file)
    file.seek(0)
    copies = [copy.deepcopy(cache), pickle.loads(pickle.dumps(cache)), torch.load(file, weights_only=False)]
    for c in copies:
        assert not set(_addresses(c)) & set(_addresses(cache))
        _uses_its_own(lib, c)
    shallow = copy.copy(cache)  # the same tensors
    assert _addresses(shallow) == _addresses(cache)
    _uses_its_own(lib, shallow)
    shallow.k = shallow.k.clone()
    _uses_its_own(lib, shallow)
    _uses_its_own(lib, cache)


@pytest.mark.parametrize("name", NAMES)
def test_cache_tensors_that_are_assigned_or_moved(lib, name):
    cache = _cache()
    setattr(cache, name, getattr(cache, name).clone())
    _uses_its_own(lib, cache)
    t = getattr(cache, name)
    t.data = t.data.clone()  # the same tensor object over other memory
    _uses_its_own(lib, cache)
    t.set_(t.clone())
    _uses_its_own(lib, cache)


def test_cache_tensors_that_no_longer_fit_are_refused(lib):
    x, at = torch.zeros(2, 3, 1, 32, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    for name, bad in (("v", lambda t: t[:, :, :32]), ("k", lambda t: t[:1]), ("k_scale", lambda t: t.double()),
                      ("v_tail", lambda t: t.float()), ("k_tail", lambda t: t.transpose(0, 1))):
        cache = _cache()
        setattr(cache, name, bad(getattr(cache, name)))
        lib.calls.clear()
        for call in (lambda: kv8_write(cache, x, x, at), lambda: kv8_read(cache, at),
                     lambda: kv8_attention(x, cache, at)):
            with pytest.raises(ValueError):
                call()
        assert not lib.calls


def test_rows_of_16_bytes_ignore_dims_of_one():
    """Only a dim that is stepped over needs a stride of whole 16 bytes; what is returned always satisfies that."""
    big = torch.zeros(3, 8, 4 * 64 + 4, dtype=torch.bfloat16)
    token = big[:1, :1, :256].unflatten(-1, (4, 64))        # strides (2080, 260, 64, 1)
    head = torch.zeros(2, 5, 1, 68, dtype=torch.bfloat16)[..., :64]
    for t, same in ((token, True), (big[:, :, :256].unflatten(-1, (4, 64)), False), (token[..., 1:33], False),
                    (head, False), (head[:1, :1], True),
                    (big.as_strided((1, 3, 4, 64), (2083, 264, 64, 1)), True), (torch.zeros(2, 3, 4, 64), True),
                    (torch.zeros(64 * 12 + 1)[1:].view(1, 3, 4, 64), False),
                    (torch.zeros(2, 3, 64, 4).transpose(2, 3), False)):
        r = _lib.rows16(t)
        assert torch.equal(r, t) and (r is t) == same
        assert r.stride(3) == 1 and r.data_ptr() % 16 == 0
        assert all(n == 1 or s * r.element_size() % 16 == 0 for n, s in zip(r.shape[:3], r.stride()))


def test_backward_operators_refuse_tensors_that_do_not_belong(lib):
    """The kernels read o, lse, lo and the gradients at the sizes of q and k: another size, type or device is refused."""
    ops = torch.ops.hclsm_b200
    bf, f32 = torch.bfloat16, torch.float32
    q, k = torch.zeros(2, 5, 4, 64, dtype=bf), torch.zeros(2, 9, 2, 64, dtype=bf)
    good = dict(o=torch.zeros_like(q), lse=torch.zeros(2, 4, 5), lo=torch.zeros_like(q), do=torch.zeros_like(q))

    def xattn(q=q, k=k, **kw):
        a = {**good, **kw}
        return ops.cross_attention_bwd(q, k, k, a["o"], a["lse"], a["lo"], a["do"], None, None, 0.125)

    for name, bad, exc in (("o", q[:, :4], ValueError), ("o", q.float(), TypeError), ("do", q[:1], ValueError),
                           ("do", q.float(), TypeError), ("do", q[..., :32], ValueError),
                           ("lse", torch.zeros(2, 5, 4), ValueError), ("lse", torch.zeros(2, 4, 5, dtype=bf), TypeError),
                           ("lo", q[:, :1], ValueError), ("lo", torch.zeros(2, 5, 4, 64), TypeError)):
        with pytest.raises(exc):
            xattn(**{name: bad})
    with pytest.raises(ValueError):
        attention_bwd(q, k, k, good["o"].to("meta"), good["lse"], good["lo"], good["do"], None, None, 0.125)
    f = {n: t.float() for n, t in good.items()}
    with pytest.raises(TypeError):
        xattn(q.float(), k.float(), **{**f, "lo": good["lo"]})

    def rope(gq=q, gk=k):
        return ops.qk_norm_rope_bwd(q, k, None, None, None, None, None, None, 1e-6, False, gq, gk)

    for kw, exc in ((dict(gq=q[:, :4]), ValueError), (dict(gq=q.float()), TypeError), (dict(gk=q), ValueError),
                    (dict(gk=k.to(torch.float16)), TypeError)):
        with pytest.raises(exc):
            rope(**kw)
    assert not lib.calls
    # what belongs goes through, an o that is not dense as a dense copy
    xattn(), rope()
    xattn(o=torch.zeros(2, 4, 5, 64, dtype=bf).transpose(1, 2))
    assert [n for n, _ in lib.calls if n.endswith("bwd")] == ["hclsm_xattn_bwd", "hclsm_qk_norm_rope_bwd",
                                                              "hclsm_xattn_bwd"]
    xattn(q.float(), k.float(), **{**f, "lo": torch.empty(0)})


def test_rotation_by_an_empty_table_is_refused():
    """Before anything is launched, positions given or not: there is no row to read."""
    native = _lib.load()
    for pos in (0, 16):
        side = _lib.ROPE_SIDE.pack(16, 0, 16, 0, pos, 0, 64, 64, 64, 1, 1)
        assert native.hclsm_qk_norm_rope(side, None, 16, 16, 0, 32, 1, 64, 1e-6, _lib.F32, 0, None) == 1
        side = _lib.ROPE_SIDE.pack(16, 16, 16, 0, pos, 0, 64, 64, 64, 1, 1)
        assert native.hclsm_qk_norm_rope_bwd(side, None, 16, 16, 0, 32, 1, 64, 1e-6, _lib.F32, 0, None, 0, None) == 1


def test_forward_mode_derivatives_are_refused_not_dropped(lib):
    ops, at = torch.ops.hclsm_b200, torch.zeros(2, dtype=torch.int32)
    x, w = torch.zeros(2, 3, 1, 32, dtype=torch.bfloat16), torch.ones(32)
    cos, sin = torch.ones(8, 16), torch.zeros(8, 16)
    cache, other = _cache(), _cache()
    with forward_ad.dual_level():
        d, dw, dc = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, w, cos))
        other.k_tail = forward_ad.make_dual(other.k_tail, torch.ones_like(other.k_tail))
        for call in (lambda: cross_attention(d, x, x), lambda: cross_attention(x, x, d), lambda: qk_norm_rope(d),
                     lambda: qk_norm_rope(x, d), lambda: qk_norm_rope(x, None, dw),
                     lambda: qk_norm_rope(x, cos=dc, sin=sin), lambda: kv8_write(cache, d, x, at),
                     lambda: kv8_write(cache, x, d, at), lambda: kv8_attention(d, cache, at),
                     lambda: kv8_attention(x, other, at), lambda: kv8_read(other, at),
                     lambda: ops.cross_attention_fwd(x, d, x, None, None, 0.1),
                     lambda: ops.qk_norm_rope_fwd(d, x, None, None, None, None, None, None, 1e-6, False)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        assert not lib.calls
        cross_attention(x, x, x), qk_norm_rope(x), kv8_attention(x, cache, at)  # no tangents
        assert forward_ad.unpack_dual(d).tangent is not None


def test_cache_calls_refuse_to_cut_a_graph(lib):
    x, at = torch.zeros(2, 3, 1, 32, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    g = x.clone().requires_grad_()
    cache, other = _cache(), _cache()
    other.v_tail.requires_grad_()
    c = (cache.k, cache.v, cache.k_scale, cache.v_scale, cache.k_tail, cache.v_tail)
    calls = (lambda: kv8_write(cache, g, x, at), lambda: kv8_write(cache, x, g, at), lambda: kv8_attention(g, cache, at),
             lambda: kv8_write(cache, (g * 2), x, at), lambda: kv8_write(other, x, x, at), lambda: kv8_read(other, at),
             lambda: kv8_attention(x, other, at))
    for call in calls:
        with pytest.raises(NotImplementedError, match="no gradients"):
            call()
    for k, v in ((g, x), (x, g)):
        with pytest.raises(NotImplementedError, match="no gradients"):
            torch.ops.hclsm_b200.kv8_write(*c, k, v, at, None)
    assert not lib.calls
    with torch.no_grad():
        for call in calls:
            call()
    assert lib.calls


def test_gradients_of_lse_and_lo_are_refused_not_dropped(lib):
    q, k = torch.zeros(2, 5, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 9, 2, 64, dtype=torch.bfloat16)
    leaves = [t.requires_grad_() for t in (q, k, k.clone())]
    for use in (lambda o, lse, lo: o.float().sum() + lse.sum(), lambda o, lse, lo: lse.sum(),
                lambda o, lse, lo: o.float().sum() + lo.float().sum()):
        out = torch.ops.hclsm_b200.cross_attention_fwd(*leaves, None, None, 0.125)
        with pytest.raises(NotImplementedError, match="only o has gradients"):
            use(*out).backward()
    o, lse, lo = torch.ops.hclsm_b200.cross_attention_fwd(*leaves, None, None, 0.125)
    lib.calls.clear()
    (o.float().sum() + lse.detach().sum()).backward()
    assert [n for n, _ in lib.calls][-1] == "hclsm_xattn_bwd" and all(t.grad.shape == t.shape for t in leaves)


def test_gradients_of_the_rotation_tables_are_refused_not_dropped(lib):
    x = torch.zeros(2, 3, 1, 32, dtype=torch.bfloat16)
    xg, cos, sin = x.clone().requires_grad_(), torch.ones(8, 16), torch.zeros(8, 16)
    cg, op = cos.clone().requires_grad_(), torch.ops.hclsm_b200.qk_norm_rope_fwd
    for q in (x, xg):
        for c, s in ((cg, sin), (cos, cg), (cg * 2, sin)):
            with pytest.raises(NotImplementedError, match="cos and sin"):
                qk_norm_rope(q, cos=c, sin=s)
            with pytest.raises(NotImplementedError, match="cos and sin"):
                op(q, q, None, None, c, s, None, None, 1e-6, False)
    lib.calls.clear()
    with torch.no_grad():
        qk_norm_rope(x, cos=cg, sin=sin)
        op(x, x, None, None, cg, sin, None, None, 1e-6, False)
    y, _ = op(xg, x, None, None, cos, sin, None, None, 1e-6, False)
    y.sum().backward()
    assert len(lib.calls) == 4


def test_tensors_of_another_device_than_the_current_one_are_refused(monkeypatch):
    """A launch goes to the current device, where the other's addresses mean nothing."""
    monkeypatch.setattr(_lib, "_get_device", lambda: 0, raising=False)
    monkeypatch.setattr(_lib, "_raw_stream", lambda index: 1000 + index)
    assert _lib.stream_ptr(torch.device("cuda", 0)) == 1000
    with pytest.raises(ValueError, match="current device"):
        _lib.stream_ptr(torch.device("cuda", 1))
