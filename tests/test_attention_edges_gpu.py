"""Further edges of the attention operators: long sweeps with part-filled query tiles, layouts with free strides,
accuracy that only the right intermediate types give, and derivatives that are refused instead of dropped.

Errors are 2-norms relative to the result's, u = 2^-8 is bf16's unit roundoff.
"""
import pytest
import torch

import hclsm_b200
from hclsm_b200.kernels import cross_attention
from test_attention_ops_gpu import BF16, U, _allowed, _attn_ref, _err, _gen, _randn

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
