"""Norm and rotation of heads, and appending to the paged cache, on a B200
against 64-bit references."""
from __future__ import annotations

import pytest
import torch

import attn_cases as ac

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def freqs(pairs, theta=1e4):
    return theta ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,hq,hk,dim,rotary", [(1, 32, 8, 128, 128), (37, 5, 1, 64, 32), (700, 30, 30, 128, 128),
                                                     (3, 1, 0, 256, 256), (19, 7, 7, 96, 64), (5, 3, 2, 8, 8),
                                                     (11, 2, 2, 72, 40), (4, 9, 3, 200, 16)])
def test_norm_and_rotation(ctx, dtype, layout, tokens, hq, hk, dim, rotary):
    from turbocider_b200 import cuda as tcc
    g = ac.gen(tokens + dim)
    row = ac.normal(g, (tokens, (hq + hk) * dim), dtype, 2.0)
    q, k = row[:, :hq * dim].view(tokens, hq, dim), row[:, hq * dim:].view(tokens, hk, dim) if hk else None
    wq, wk = (1 + 0.3 * torch.randn(dim, device="cuda", generator=g) for _ in range(2))
    pos = torch.randint(-5, 2 ** 20, (tokens,), dtype=torch.int32, device="cuda", generator=g)
    f = freqs(rotary // 2)
    where = pos[:, None].expand(-1, rotary // 2)
    for eps, weights, turn in ((1e-6, True, True), (None, False, True), (1e-3, False, False), (1e-6, True, False)):
        rope = tcc.Rope(f, pos, layout=layout, amplitude=1.25) if turn else None
        yq, yk = tcc.qk_norm_rope(ctx, q, k, rope, q_weight=wq if weights else None, k_weight=wk if weights else None,
                                  eps=eps)
        for x, y, w in ((q, yq, wq), (k, yk, wk)):
            if x is not None:
                want, tol = ac.heads_ref(x, w if weights else None, eps, f if turn else None, 1.25, layout, where)
                ac.close(y, want, tol, f"eps {eps} turn {turn}")
    assert (yk is None) == (hk == 0) and ctx.status() == 0


def test_positions_to_the_end_of_int32(ctx):
    from turbocider_b200 import cuda as tcc
    pos = torch.tensor([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 10 ** 9 + 7, 2 ** 24 + 1], dtype=torch.int32, device="cuda")
    # frequencies whose products with any int32 are exact in float64 up to the
    # reference's own cos: multiples of 2^-20 radians
    f = torch.round(freqs(32) * 2 ** 20) / 2 ** 20
    g = ac.gen(1)
    q = ac.normal(g, (7, 2, 64), FP)
    y, _ = tcc.qk_norm_rope(ctx, q, None, tcc.Rope(f, pos))
    want, tol = ac.heads_ref(q, None, None, f, 1.0, "half", pos[:, None].expand(-1, 32))
    ac.close(y, want, tol)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_position_axes(ctx, layout):
    from turbocider_b200 import cuda as tcc
    g = ac.gen(2)
    sections = [8, 28, 28]
    f = torch.cat([freqs(n, 256.0) for n in sections])
    pos = torch.randint(0, 500, (50, 3), dtype=torch.int32, device="cuda", generator=g)
    q = ac.normal(g, (50, 4, 128), HF)
    y, _ = tcc.qk_norm_rope(ctx, q, None, tcc.Rope(f, pos, layout=layout, sections=sections), eps=1e-6)
    where = torch.cat([pos[:, a:a + 1].expand(-1, n) for a, n in enumerate(sections)], 1)
    want, tol = ac.heads_ref(q, None, 1e-6, f, 1.0, layout, where)
    ac.close(y, want, tol)


def test_in_place_strides_and_alignment(ctx):
    from turbocider_b200 import cuda as tcc
    g = ac.gen(3)
    f = freqs(32)
    pos = torch.arange(20, dtype=torch.int32, device="cuda")
    where = pos[:, None].expand(-1, 32)
    for dtype in (BF, FP):
        x = ac.normal(g, (20, 3, 64), dtype)
        want, tol = ac.heads_ref(x, None, 1e-5, f, 1.0, "half", where)
        odd = torch.full((20, 3, 67), 7.0, dtype=dtype, device="cuda")      # no chunk of it is aligned
        odd[..., 1:65] = x
        heads_first = x.transpose(0, 1).contiguous().transpose(0, 1)
        for view in (x.clone(), odd[..., 1:65], heads_first):
            y, _ = tcc.qk_norm_rope(ctx, view, None, tcc.Rope(f, pos), eps=1e-5, q_out=view)
            assert y is view
            ac.close(y, want, tol)
        assert bool((odd[..., 0] == 7).all()) and bool((odd[..., 65:] == 7).all())
    # broadcast input: the same row for every token
    one = ac.normal(g, (1, 3, 64), BF).expand(20, 3, 64)
    y, _ = tcc.qk_norm_rope(ctx, one, None, tcc.Rope(f, pos))
    want, tol = ac.heads_ref(one, None, None, f, 1.0, "half", where)
    ac.close(y, want, tol)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("page,token_major", [(8, False), (16, True), (128, False)])
@pytest.mark.parametrize("hq,hk,dim,rotary,norm", [(8, 2, 128, 128, True), (0, 3, 64, 32, False), (4, 4, 80, 80, True),
                                                   (6, 1, 256, 0, False)])
def test_append(ctx, dtype, page, token_major, hq, hk, dim, rotary, norm):
    from turbocider_b200 import cuda as tcc
    g = ac.gen(page + dim)
    lens = [(1, 1), (5, 40), (0, 7), (1, 0), (70, 70), (3, 129), (2, 17)] + [(1, 9)] * 40
    kc, vc, table, ks, vs = ac.paged(lens, page, hk, dim, dtype, g, token_major)
    offsets, lengths = ac.offsets_of(lens)
    tokens = int(offsets[-1])
    extra = 2   # rows that belong to no request
    row = ac.normal(g, (tokens + extra, (hq + 2 * hk) * dim), dtype, 1.5)
    q = row[:, :hq * dim].view(-1, hq, dim) if hq else None
    k, v = (row[:, (hq + i * hk) * dim:(hq + (i + 1) * hk) * dim].view(-1, hk, dim) for i in range(2))
    wq, wk = (1 + 0.3 * torch.randn(dim, device="cuda", generator=g) for _ in range(2))
    f = freqs(rotary // 2) if rotary else None
    before = kc.clone(), vc.clone()
    q_out = torch.full((tokens + extra, hq, dim), 9.0, dtype=dtype, device="cuda") if hq else None
    got = tcc.kv_append(ctx, tcc.PagedCache(kc, vc, token_major),
                        tcc.PagedBatch(offsets, lengths, table, 70, 129), k, v, tcc.Rope(f) if rotary else None, q=q,
                        q_weight=wq if norm else None, k_weight=wk if norm else None, eps=1e-6 if norm else None,
                        q_out=q_out)
    assert ctx.status() == 0 and got is q_out
    place = torch.tensor([n - new + i for new, n in lens for i in range(new)], device="cuda")
    where = place.clamp(min=0)[:, None].expand(-1, rotary // 2)
    args = (1e-6 if norm else None, f, 1.0, "half", where)
    want_k, tol_k = ac.heads_ref(k[:tokens], wk if norm else None, *args)
    if hq:
        want_q, tol_q = ac.heads_ref(q[:tokens], wq if norm else None, *args)
        ac.close(got[:tokens], want_q, tol_q, "q")
        assert bool((got[tokens:] == 9).all())
    table = table.cpu()
    t = 0
    for b, (new, n) in enumerate(lens):
        for i in range(new):
            p = n - new + i
            if n and p >= 0:
                pg, r = int(table[b, p // page]), p % page
                kk, vv, k0, v0 = ((c[pg, r] if token_major else c[pg, :, r]) for c in (kc, vc, *before))
                ac.close(kk, want_k[t], tol_k[t], "k")
                assert torch.equal(vv.view(torch.int16), v[t].view(torch.int16))
                k0.copy_(kk)
                v0.copy_(vv)
            t += 1
    for c, c0 in zip((kc, vc), before):   # every other place is as it was, bit for bit
        assert torch.equal(c.view(torch.int16), c0.view(torch.int16))


def test_append_many_requests_and_given_positions(ctx):
    """More requests than one search step covers, empty ones among them."""
    from turbocider_b200 import cuda as tcc
    g = ac.gen(4)
    lens = [(i % 3, 3 + i % 50) for i in range(1500)]
    kc, vc, table, _, _ = ac.paged(lens, 64, 1, 64, BF, g, fill=0.0)
    offsets, lengths = ac.offsets_of(lens)
    tokens = int(offsets[-1])
    k, v = ac.normal(g, (tokens, 1, 64), BF), ac.normal(g, (tokens, 1, 64), BF)
    pos = torch.randint(0, 1000, (tokens,), dtype=torch.int32, device="cuda", generator=g)
    f = freqs(32)
    tcc.kv_append(ctx, tcc.PagedCache(kc, vc), tcc.PagedBatch(offsets, lengths, table, 2, 52), k, v, tcc.Rope(f, pos))
    want, tol = ac.heads_ref(k, None, None, f, 1.0, "half", pos[:, None].expand(-1, 32))
    b = torch.repeat_interleave(torch.arange(1500), torch.tensor([n for n, _ in lens]))
    place = torch.tensor([n - new + i for new, n in lens for i in range(new)])
    pg, r = table.cpu()[b, place // 64].long().cuda(), (place % 64).cuda()
    ac.close(kc[pg, :, r], want, tol)
    assert torch.equal(vc[pg, :, r], v) and ctx.status() == 0


def test_append_reports_impossible_pages(ctx):
    from turbocider_b200 import cuda as tcc
    g = ac.gen(5)
    lens = [(1, 20), (1, 30)]
    kc, vc, table, _, _ = ac.paged(lens, 16, 2, 64, BF, g, fill=0.0)
    offsets, lengths = ac.offsets_of(lens)
    k, v = ac.normal(g, (2, 2, 64), BF), ac.normal(g, (2, 2, 64), BF)
    before = kc.clone()
    for bad in (-1, kc.shape[0], 2 ** 31 - 1):
        t = table.clone()
        t[:, 1] = bad
        tcc.kv_append(ctx, tcc.PagedCache(kc, vc), tcc.PagedBatch(offsets, lengths, t, 1, 30), k, v)
        assert ctx.status() == tcc.STATUS_GEOMETRY
    assert torch.equal(kc, before)
    for n in (10 ** 6, -3):
        tcc.kv_append(ctx, tcc.PagedCache(kc, vc), tcc.PagedBatch(offsets, torch.full_like(lengths, n), table, 1, 30),
                      k, v)
        assert ctx.status() == tcc.STATUS_GEOMETRY
    assert torch.equal(kc, before)


def test_refusals(ctx):
    from turbocider_b200 import cuda as tcc
    g = ac.gen(6)
    x = ac.normal(g, (4, 2, 64), BF)
    pos = torch.arange(4, dtype=torch.int32, device="cuda")
    f = freqs(32)

    def refused(match, fn, *a, **kw):
        with pytest.raises(tcc.BackendError, match=match):
            fn(*a, **kw)

    refused("multiple of 8", tcc.qk_norm_rope, ctx, ac.normal(g, (4, 2, 60), BF))
    refused("at most 256", tcc.qk_norm_rope, ctx, ac.normal(g, (4, 2, 264), BF))
    refused("rotary_dim", tcc.qk_norm_rope, ctx, x, None, tcc.Rope(freqs(48), pos))
    refused("rotary_dim", tcc.qk_norm_rope, ctx, x, None, tcc.Rope(freqs(10), pos))
    refused("needs positions", tcc.qk_norm_rope, ctx, x, None, tcc.Rope(f))
    refused("one position", tcc.qk_norm_rope, ctx, x, None, tcc.Rope(f, pos[:3]))
    refused("sections must add up", tcc.qk_norm_rope, ctx, x, None,
            tcc.Rope(f, torch.zeros((4, 2), dtype=torch.int32, device="cuda"), sections=[16, 15]))
    refused("section", tcc.Rope, f, pos, sections=[16, 16])
    refused("layout", tcc.Rope, f, pos, layout="other")
    refused("float64", tcc.Rope, f.float(), pos)
    refused("int32", tcc.Rope, f, pos.long())
    refused("eps", tcc.qk_norm_rope, ctx, x, eps=-1.0)
    refused("f32, f16 or bf16", tcc.qk_norm_rope, ctx, x.double())
    refused("share", tcc.qk_norm_rope, ctx, x, x[:3])
    refused("norm weights", tcc.qk_norm_rope, ctx, x, q_weight=torch.ones(32, device="cuda"), eps=1e-6)
    refused("overlapping head", tcc.qk_norm_rope, ctx, x, q_out=x[:1].expand(4, 2, 64))
    kc = torch.zeros((4, 2, 16, 64), dtype=BF, device="cuda")
    cache = tcc.PagedCache(kc, kc.clone())
    batch = tcc.PagedBatch(torch.tensor([0, 4], dtype=torch.int32, device="cuda"), pos[:1] + 4,
                           torch.zeros((1, 1), dtype=torch.int32, device="cuda"), 4, 4)
    refused("cache's heads", tcc.kv_append, ctx, cache, batch, x[:, :1], x[:, :1])
    refused("cache's type", tcc.kv_append, ctx, cache, batch, x.half(), x.half())
    refused("one row for each key", tcc.kv_append, ctx, cache, batch, x, x, q=x[:2])
    assert tcc.qk_norm_rope(ctx, x[:0])[0].shape == (0, 2, 64)
    assert ctx.status() == 0


def test_refuses_other_ranks_and_wide_bounds(ctx):
    """Tensors that are not three-dimensional and bounds past 32 bits are refused, not read or cut off."""
    from turbocider_b200 import cuda as tcc
    x = ac.normal(ac.gen(7), (4, 2, 64), BF)
    kc = torch.zeros((4, 2, 16, 64), dtype=BF, device="cuda")
    cache = tcc.PagedCache(kc, kc.clone())
    offsets = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    length, table = offsets[1:], torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    batch = tcc.PagedBatch(offsets, length, table, 4, 4)
    flat = x.reshape(4, 128)
    for call in (lambda: tcc.qk_norm_rope(ctx, flat), lambda: tcc.qk_norm_rope(ctx, x, flat),
                 lambda: tcc.kv_append(ctx, cache, batch, flat, flat),
                 lambda: tcc.kv_append(ctx, cache, batch, x, flat),
                 lambda: tcc.kv_append(ctx, cache, batch, x, x, q=flat),
                 lambda: tcc.paged_attention(ctx, cache, batch, flat),
                 lambda: tcc.PagedBatch(offsets, length, table, 2**32 + 4, 4),
                 lambda: tcc.PagedBatch(offsets, length, table, 4, 2**32 + 4)):
        with pytest.raises(tcc.BackendError):
            call()
    assert not kc.any() and ctx.status() == 0
