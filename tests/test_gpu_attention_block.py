"""The attention block (quantised projections, cache, attention) on a B200
against the same mathematics in 64 bits on the dequantised weights."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, DIM, PAGE = 512, 4, 2, 128, 16


def build(ctx, pages):
    from turbocider_b200 import cuda as tcc
    from turbocider_b200.attention import AttentionBlock, PagePool
    rng = np.random.default_rng(7)

    def weight(n, k):
        raw = tcc.quantize(tcc.Q4_K, (rng.standard_normal((n, k)) * k ** -0.5).astype(np.float32))
        return tcc.Weight.upload(ctx, tcc.Q4_K, n, k, raw)
    k, v = (torch.full((pages, KV, PAGE, DIM), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    norms = [1 + 0.2 * torch.randn(DIM, device="cuda", generator=g) for _ in range(2)]
    freq, _ = tcc.rope_freqs(DIM, 1e4, device="cuda")
    block = AttentionBlock(ctx, weight((HEADS + 2 * KV) * DIM, HIDDEN), weight(HIDDEN, HEADS * DIM),
                           tcc.PagedCache(k, v), HEADS, *norms, freq=freq)
    return block, PagePool(pages, PAGE), norms, freq


def reference(block, norms, freq, x):
    """The block over one whole request in 64 bits."""
    from turbocider_b200 import cuda as tcc
    w, wo = (tcc.dequant(block.ctx, m, tcc.F32).double() for m in (block.qkv, block.out))
    n = x.shape[0]
    heads = (x.double() @ w.T).view(n, HEADS + 2 * KV, DIM)
    t = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * freq
    turn = torch.polar(torch.ones_like(t), t)[:, None]

    def place(h, norm):
        h = h / (h.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * norm.double()
        z = torch.complex(h[..., :DIM // 2], h[..., DIM // 2:]) * turn
        return torch.cat((z.real, z.imag), -1)
    q, k, v = place(heads[:, :HEADS], norms[0]), place(heads[:, HEADS:HEADS + KV], norms[1]), heads[:, HEADS + KV:]
    k, v = (a.repeat_interleave(HEADS // KV, 1) for a in (k, v))
    s = torch.einsum("ihd,jhd->hij", q, k) * DIM ** -0.5
    s = s.masked_fill(torch.ones((n, n), dtype=torch.bool, device="cuda").triu(1), -torch.inf)
    return torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v).reshape(n, -1) @ wo.T


def test_prompts_and_steps(ctx):
    """Prompts in uneven parts, then single tokens, of requests that come and
    go.  Roundings to bf16 on the way (weights, projections, heads,
    probabilities, attention, result): six of relative size 2^-9 rms at most
    each; 2^-9 * sqrt(6) * 2 = 1e-2 in the 2-norm."""
    block, pool, norms, freq = build(ctx, 80)
    g = torch.Generator(device="cuda")
    g.manual_seed(6)
    xs = {r: torch.randn((n, HIDDEN), device="cuda", generator=g).bfloat16() for r, n in
          ((0, 150), (1, 37), (2, 300), (3, 5))}
    got = {r: [] for r in xs}
    plan = [([0, 1], [130, 36]), ([2, 0], [260, 3]), ([0, 1, 2, 3], [1, 1, 1, 0]), ([3], [4]),
            ([2, 3, 0], [39, 1, 16])]
    for requests, new in plan:
        at = [pool.length(r) for r in requests]
        step = pool.step(requests, new, "cuda")
        x = torch.cat([xs[r][a:a + n] for r, a, n in zip(requests, at, new)])
        y = block(x, step)
        for r, part in zip(requests, y.split(new)):
            got[r].append(part)
    assert ctx.status() == 0
    for r, x in xs.items():
        y = torch.cat(got[r])
        assert y.shape[0] == x.shape[0]
        want = reference(block, norms, freq, x)
        err = float((y.double() - want).norm() / want.norm())
        assert err <= 1e-2, f"request {r}: rel-L2 {err:.2e}"


def test_steps_in_a_graph(ctx):
    """A captured step (fixed batch places, device values updated in place)
    gives the same bits as the calls."""
    from turbocider_b200 import cuda as tcc
    block, pool, _, _ = build(ctx, 40)
    for r in range(3):
        pool.grow(r, 60 + 5 * r)
    block.cache.k.normal_()
    block.cache.v.normal_()
    x = torch.randn((3, HIDDEN), device="cuda").bfloat16()
    offsets = torch.arange(4, dtype=torch.int32, device="cuda")
    lengths = torch.zeros(3, dtype=torch.int32, device="cuda")
    table = torch.full((3, 8), -1, dtype=torch.int32, device="cuda")
    step = tcc.PagedBatch(offsets, lengths, table, 1, 8 * PAGE)
    block(x, step)                                   # workspaces
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block(x, step)
    for _ in range(3):
        n = [pool.grow(r, 1) for r in range(3)]
        rows = torch.tensor(pool.table(range(3)), dtype=torch.int32)
        lengths.copy_(torch.tensor(n, dtype=torch.int32))
        table[:, :rows.shape[1]] = rows.cuda()
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        again = block(x, step)
        assert torch.equal(y, again) and not bool(torch.isnan(y).any())
    # the workspace outgrown by a larger call stays valid for the graph
    big = torch.randn((40, HEADS, DIM), device="cuda").bfloat16()
    k = torch.zeros((400, KV, PAGE, DIM), dtype=torch.bfloat16, device="cuda")
    wide = torch.arange(400, dtype=torch.int32, device="cuda")[None].expand(40, 400).contiguous()
    tcc.paged_attention(ctx, tcc.PagedCache(k, k.clone()),
                        tcc.PagedBatch(torch.arange(41, dtype=torch.int32, device="cuda"),
                                       torch.full((40,), 6400, dtype=torch.int32, device="cuda"), wide, 1, 6400), big)
    before = block(x, step)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, before) and ctx.status() == 0
