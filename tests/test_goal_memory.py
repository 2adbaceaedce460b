"""The example that runs the attention operators together, a captured training step of it, the operators as
dispatcher operators, and (on the CPU) the layout of the argument structs."""
import importlib.util
import os
import shutil
import subprocess

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import hclsm_b200.torch_ops  # noqa: F401  (registers the ops)
from hclsm_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OPS = torch.ops.hclsm_b200


def _example():
    spec = importlib.util.spec_from_file_location("goal_memory", os.path.join(ROOT, "examples", "goal_memory.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_struct_layouts_match_the_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "hclsm_b200.h"\nint main(void) { printf("%zu %zu %zu %zu\\n", '
                   'sizeof(hclsm_view), sizeof(hclsm_rope_side), sizeof(hclsm_xattn_args), sizeof(hclsm_kv8_cache)); '
                   'return 0; }\n')
    subprocess.check_call([cc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")])
    sizes = [int(v) for v in subprocess.check_output([str(tmp_path / "s")]).split()]
    assert sizes == [_lib.VIEW.size, _lib.ROPE_SIDE.size, _lib.XATTN_ARGS.size, _lib.KV8_CACHE.size]


def test_c_entries_refuse_without_a_gpu():
    """Argument checks return a status before anything touches a device."""
    lib = _lib.load()

    def xattn(**kw):
        a = dict(q=(16, 0, 0, 0), k=(16, 0, 0, 0), v=(16, 0, 0, 0), do=(0, 0, 0, 0), o=16, B=1, Lq=1, Lk=1, H=1, Hkv=1,
                 D=64, dtype=0, scale=1.0, lo=0)
        a.update(kw)
        return _lib.XATTN_ARGS.pack(*a["q"], *a["k"], *a["v"], *a["do"], a["o"], 0, 0, 0, 0, a["lo"], 0, 0, 0, a["B"],
                                    a["Lq"],
                                    a["Lk"], a["H"], a["Hkv"], a["D"], a["dtype"], a["scale"])

    for want, kw in ((2, dict(dtype=7)), (1, dict(D=129)), (1, dict(D=0)), (1, dict(H=3, Hkv=2)), (1, dict(B=-1)),
                     (1, dict(scale=0.0)), (1, dict(scale=float("nan"))), (3, dict(lo=8)), (8, dict(o=0)),
                     (8, dict(k=(0, 0, 0, 0)))):
        assert lib.hclsm_xattn_fwd(xattn(**kw), None, 0, None) == want, kw
    assert lib.hclsm_xattn_fwd(xattn(B=0), None, 0, None) == 0
    assert lib.hclsm_xattn_bwd(xattn(), None, 0, None) == 8
    assert lib.hclsm_xattn_fwd(None, None, 0, None) == 8

    def kv8(**kw):
        a = dict(p=16, B=1, Hkv=1, T=64, D=64, block=32, dtype=1)
        a.update(kw)
        return _lib.KV8_CACHE.pack(*[a["p"]] * 6, a["B"], a["Hkv"], a["T"], a["D"], a["block"], a["dtype"])

    view = _lib.VIEW.pack(16, 64, 64, 64)
    for want, kw in ((1, dict(D=48)), (1, dict(block=24)), (1, dict(T=40)), (2, dict(dtype=3)), (3, dict(p=8)),
                     (8, dict(p=0))):
        assert lib.hclsm_kv8_write(kv8(**kw), view, view, 1, 16, None, None) == want, kw
        assert lib.hclsm_kv8_attn(kv8(**kw), view, 16, None, 1, 1, 1.0, None, 0, None) == want, kw
    assert lib.hclsm_kv8_attn(kv8(), view, 16, None, 1, 1, -1.0, None, 0, None) == 1
    assert lib.hclsm_kv8_write(kv8(), view, _lib.VIEW.pack(18, 64, 64, 64), 1, 16, None, None) == 3

    def rope(**kw):
        a = dict(x=16, dy=0, y=16, w=0, pos=0, dw=0, s=(64, 64, 64), L=1, H=1)
        a.update(kw)
        return _lib.ROPE_SIDE.pack(a["x"], a["dy"], a["y"], a["w"], a["pos"], a["dw"], *a["s"], a["L"], a["H"])

    def call(side, rot=0, D=64, dtype=0, flags=0, P=4, tab=16):
        return lib.hclsm_qk_norm_rope(side, None, tab, tab, P, rot, 1, D, 1e-6, dtype, flags, None)

    assert call(rope(), D=12) == 1 and call(rope(), rot=24) == 1 and call(rope(), rot=128) == 1
    assert call(rope(), dtype=5) == 2 and call(rope(x=8)) == 3 and call(rope(s=(64, 3, 64))) == 3
    assert call(rope(x=0)) == 8 and call(rope(), rot=32, tab=None) == 8
    assert call(rope(w=16), flags=2) == 7 and call(rope(L=9), rot=32) == 1
    assert call(rope(L=0, x=0)) == 0


def test_ops_registered_and_fake_shapes():
    with FakeTensorMode():
        q = torch.empty(2, 5, 6, 64, dtype=torch.bfloat16, device="cuda")
        k = torch.empty(2, 9, 3, 64, dtype=torch.bfloat16, device="cuda")
        o, lse, lo = OPS.cross_attention_fwd(q, k, k, None, None, 0.1)
        assert o.shape == q.shape and o.dtype == q.dtype and lse.shape == (2, 6, 5) and lse.dtype == torch.float32
        assert lo.shape == q.shape and OPS.cross_attention_fwd(q.float(), k.float(), k.float(), None, None,
                                                               0.1)[2].numel() == 0
        assert [t.shape for t in OPS.cross_attention_bwd(q, k, k, o, lse, lo, o, None, None, 0.1)] == [q.shape, k.shape,
                                                                                               k.shape]
        yq, yk = OPS.qk_norm_rope_fwd(q, k, None, None, None, None, None, None, 1e-6, False)
        assert yq.shape == q.shape and yk.shape == k.shape
    x = torch.zeros(1, 2, 1, 64)
    with pytest.raises(ValueError):
        OPS.cross_attention_fwd(x, x, x, None, None, 0.1)


@pytest.mark.gpu
def test_example_trains_and_rolls_out():
    """The 8-bit cache: values and keys are off by at most half a step, 1/254 of a block's largest (3.5 standard
    deviations: 0.8 percent rms), which weights and values carry once each; with bf16's 0.4 percent well below 5."""
    losses, far = _example().main(steps=20, B=4, K=10, N=16, G=3)
    assert losses[-1] < 0.5 * losses[0]
    assert 0 < far < 0.05


@pytest.mark.gpu
def test_training_step_captures_as_a_graph():
    import hclsm_b200

    torch.manual_seed(1)
    model = _example().GoalMemory(256, heads=4, kv_heads=2)
    goals, states = (torch.randn(*s, device="cuda").bfloat16() for s in ((2, 3, 256), (2, 6, 8, 256)))
    counts = torch.tensor([6, 3], device="cuda", dtype=torch.int32)
    alive = torch.rand(2, 8, device="cuda") > 0.2

    def step():
        model(goals, states, counts - 1, counts, alive).float().square().sum().backward()

    step()
    eager = [p.grad.clone() for p in model.parameters()]
    for p in model.parameters():
        p.grad = None
    graphed = hclsm_b200.GraphedStep(step, params=list(model.parameters()))
    graphed.replay()
    for p, g in zip(model.parameters(), eager):
        assert torch.equal(p.grad, g)
    assert hclsm_b200.device_error() == 0


@pytest.mark.gpu
def test_ops_match_direct_calls_and_autograd():
    from hclsm_b200.kernels import Kv8Cache, cross_attention, kv8_attention, kv8_write, qk_norm_rope, rope_tables

    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(2, n, h, 64, generator=g, device="cuda").bfloat16().requires_grad_()
               for n, h in ((7, 4), (50, 2), (50, 2)))
    lens = torch.tensor([50, 31], device="cuda", dtype=torch.int32)
    w = torch.ones(64, device="cuda", requires_grad=True)
    cos, sin = rope_tables(64, 32)

    def direct():
        a, b = qk_norm_rope(q, k, w, w, cos, sin)
        return cross_attention(a, b, v, kv_lens=lens)

    def ops():
        a, b = OPS.qk_norm_rope_fwd(q, k, w, w, cos, sin, None, None, 1e-6, False)
        return OPS.cross_attention_fwd(a, b, v, lens, None, 64 ** -0.5)[0]

    o1, o2 = direct(), ops()
    do = torch.randn(o1.shape, generator=g, device="cuda").bfloat16()
    assert torch.equal(o1, o2)
    for a, b in zip(torch.autograd.grad(o1, (q, k, v, w), do), torch.autograd.grad(o2, (q, k, v, w), do)):
        assert torch.equal(a, b)
    caches = [Kv8Cache.empty(2, 64, 2, 64) for _ in range(2)]
    start = torch.zeros(2, device="cuda", dtype=torch.int32)
    kv8_write(caches[0], k.detach(), v.detach(), start, lens)
    c = caches[1]
    OPS.kv8_write(c.k, c.v, c.k_scale, c.v_scale, c.k_tail, c.v_tail, k.detach(), v.detach(), start, lens)
    got = OPS.kv8_attention(q.detach(), c.k, c.v, c.k_scale, c.v_scale, c.k_tail, c.v_tail, lens, 64 ** -0.5)
    assert torch.equal(got, kv8_attention(q.detach(), caches[0], lens))
