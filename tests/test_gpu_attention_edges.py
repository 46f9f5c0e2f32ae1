"""Attention operators on a B200 where calls leave the ordinary: weights without
a norm, impossible values in device memory, given-back pages, very many tiles
and shares.  Against 64-bit references and sentinels."""
from __future__ import annotations

import pytest
import torch

import attn_cases as ac

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("layout", [None, "half", "interleaved"])
def test_a_weight_is_the_norms(ctx, dtype, layout):
    """Without a norm its weights have no part in the result: rotation only,
    or the elements as they are."""
    from turbocider_b200 import cuda as tcc
    g = ac.gen(21)
    q, k = ac.normal(g, (37, 5, 64), dtype), ac.normal(g, (37, 2, 64), dtype)
    wq, wk = (1 + 0.5 * torch.randn(64, device="cuda", generator=g) for _ in range(2))
    rope = None
    if layout:
        f = 1e4 ** (-torch.arange(16, dtype=torch.float64, device="cuda") / 16)
        rope = tcc.Rope(f, torch.arange(37, dtype=torch.int32, device="cuda"), layout=layout)
    want = tcc.qk_norm_rope(ctx, q, k, rope)
    got = tcc.qk_norm_rope(ctx, q, k, rope, q_weight=wq, k_weight=wk)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    if rope is None:
        assert torch.equal(got[0], q) and torch.equal(got[1], k)
    if dtype == FP:
        return
    lens = [(30, 40), (7, 7)]
    offsets, lengths = ac.offsets_of(lens)
    table = torch.arange(6, dtype=torch.int32, device="cuda").view(2, 3)
    rope = tcc.Rope(f, layout=layout) if layout else None
    v, kept = ac.normal(g, (37, 2, 64), dtype), []
    for weights in (dict(), dict(q_weight=wq, k_weight=wk)):
        cache = [torch.zeros((6, 2, 16, 64), dtype=dtype, device="cuda") for _ in range(2)]
        y = tcc.kv_append(ctx, tcc.PagedCache(*cache), tcc.PagedBatch(offsets, lengths, table, 30, 40), k, v, rope, q=q,
                          **weights)
        kept.append([y] + cache)
    assert all(torch.equal(a, b) for a, b in zip(*kept))
    assert ctx.status() == 0
