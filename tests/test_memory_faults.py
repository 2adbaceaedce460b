"""The operators that remember a history, on the CPU: calls and tables at the edges of what they are documented to take."""
import pytest
import torch

from hclsm_b200 import _lib
from hclsm_b200.kernels import (Kv4Cache, Kv8Cache, PageTable, decay_attention_step, kv4_attention, kv4_read, kv4_write,
                                kv8_attention, kv8_read, kv8_write, pages_resize)

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


def test_kv4_tensors_that_were_changed_where_they_are(lib):
    """A tensor changed in place may keep its address: the call takes its present shape, or refuses it."""
    c = Kv4Cache.empty(4, 1, 32, page=32, device="cpu")
    at = c.k.data_ptr()
    for t in (c.k, c.v):
        t.resize_(8, 1, 16, 16)
    table, x, slots = torch.zeros(1, 3, dtype=I32), torch.zeros(1, 2, 1, 32, dtype=BF), torch.zeros(1, 2, dtype=I32)
    calls = (lambda: kv4_read(c, table), lambda: kv4_write(c, x, x, slots), lambda: kv4_attention(x, c, table))
    for call in calls:  # the scales are those of pages of 32
        with pytest.raises(ValueError):
            call()
    for t in (c.k_scale, c.v_scale):
        t.resize_(8, 1, 16, 1)
    assert c.k.data_ptr() == at
    for call in calls:
        lib.calls.clear()
        call()
        assert _lib.KV4_CACHE.unpack(lib.calls[-1][1][0])[4:8] == (8, 1, 16, 32)
    assert calls[0]()[0].shape == (1, 48, 1, 32)
    c.k.transpose_(0, 2), c.v.transpose_(0, 2)  # 16 pages of 8 tokens
    d = Kv4Cache.empty(32, 1, 32, page=32, device="cpu")
    d.k.transpose_(0, 2)  # the same shape, in another order
    e = Kv4Cache.empty(4, 1, 32, page=32, device="cpu")
    e.k_scale.data = e.k_scale.data.view(torch.float16)
    lib.calls.clear()
    for cache in (c, d, e):
        for call in (lambda: kv4_read(cache, table), lambda: kv4_write(cache, x, x, slots),
                     lambda: kv4_attention(x, cache, table)):
            with pytest.raises(ValueError):
                call()
    assert not lib.calls


def test_kv8_tensors_that_were_changed_where_they_are(lib):
    c = Kv8Cache.empty(2, 64, 2, 32, device="cpu")
    at = c.k.data_ptr()
    c.k.resize_(2, 1, 64, 32), c.v.resize_(2, 1, 64, 32)
    x, start = torch.zeros(2, 3, 1, 32, dtype=BF), torch.zeros(2, dtype=I32)
    calls = (lambda: kv8_read(c, start), lambda: kv8_write(c, x, x, start), lambda: kv8_attention(x, c, start))
    for call in calls:  # the scales and tails are those of two heads
        with pytest.raises(ValueError):
            call()
    c.k_scale.resize_(2, 1, 2), c.v_scale.resize_(2, 1, 2)
    c.k_tail.resize_(2, 1, 32, 32), c.v_tail.resize_(2, 1, 32, 32)
    assert c.k.data_ptr() == at
    for call in calls:
        lib.calls.clear()
        call()
        assert _lib.KV8_CACHE.unpack(lib.calls[-1][1][0])[6:11] == (2, 1, 64, 32, 32)
    assert calls[0]()[0].shape == (2, 64, 1, 32)
    for name in ("k", "k_scale", "k_tail"):
        d = Kv8Cache.empty(2, 64, 2, 32, device="cpu")
        getattr(d, name).transpose_(0, 1)  # the same shape, in another order
        lib.calls.clear()
        y = torch.zeros(2, 3, 2, 32, dtype=BF)
        for call in (lambda: kv8_read(d, start), lambda: kv8_write(d, y, y, start), lambda: kv8_attention(y, d, start)):
            with pytest.raises(ValueError):
                call()
        assert not lib.calls


def test_changes_in_place_move_the_versions(lib):
    """A backward that saved a tensor which a call has changed since says so."""
    c4, c8 = Kv4Cache.empty(4, 1, 32, page=32, device="cpu"), Kv8Cache.empty(2, 64, 1, 32, device="cpu")
    x, state = torch.zeros(2, 3, 1, 32, dtype=BF), torch.zeros(2, 1, 32, 32)
    at, slots = torch.zeros(2, dtype=I32), torch.zeros(2, 3, dtype=I32)
    pages = PageTable.empty(2, 64, 8, device="cpu")
    step, out = x[:, 0].float(), state.clone()
    for call, changed, kept in (
            (lambda: kv4_write(c4, x, x, slots), (c4.k, c4.v, c4.k_scale, c4.v_scale), (x, slots)),
            (lambda: kv8_write(c8, x, x, at), (c8.k, c8.v, c8.k_scale, c8.v_scale, c8.k_tail, c8.v_tail), (x, at)),
            (lambda: pages_resize(pages, at, at), (pages.table, pages.free, pages.n_free), (at,)),
            (lambda: decay_attention_step(step, step, step, torch.zeros(1), state), (state,), (step,)),
            (lambda: decay_attention_step(step, step, step, torch.zeros(1), state, out=out), (out,), (step, state))):
        before, others = [t._version for t in changed], [t._version for t in kept]
        call()
        assert all(t._version > n for t, n in zip(changed, before))
        assert [t._version for t in kept] == others
        with torch.inference_mode():
            call()
    w = torch.ones(1, requires_grad=True, dtype=BF)
    y = (w * c4.k_scale).sum()
    kv4_read(c4, slots), kv4_attention(x, c4, slots)
    y.backward(retain_graph=True)
    kv4_write(c4, x, x, slots)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


# ---- lengths next to 2^31 -------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [_lib.F32, _lib.BF16])
@pytest.mark.parametrize("D", [1, 8, 64, 128])
def test_decay_plans_of_lengths_up_to_31_bits(dtype, D):
    """A long history is cut into segments, the longest ones as those a little shorter: their parts' bytes are the same."""
    lib, some = _lib.load(), 1 << 20  # an aligned address that no query looks at

    def bytes_of(query, L, H=1):
        view = (some, L * H * D, H * D, D)
        return query(_lib.DECAY_ARGS.pack(*view * 4, *(some,) * 4, some, 0, 0, 0, 0, 0, 1, L, H, D, D, dtype, 1.0))

    for query in (lib.hclsm_decay_attn_fwd_workspace_size, lib.hclsm_decay_attn_bwd_workspace_size):
        want = bytes_of(query, (1 << 31) - 1000)
        assert want > 0
        for L in (1 << 31) - 200, (1 << 31) - 128, (1 << 31) - 127, (1 << 31) - 64, (1 << 31) - 63, (1 << 31) - 1:
            assert bytes_of(query, L) == want, L
