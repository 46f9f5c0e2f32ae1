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


def _sentinels(ctx, lens, seen_lens, max_new, max_length, hq, hk, dim, dtype, seed):
    """Attention and append of requests `lens` into outputs filled with 7,
    bounded by max_new and max_length; (attention's out, lse, its reference
    over seen_lens, append's q_out, cache before, cache after, status bits)."""
    from turbocider_b200 import cuda as tcc
    g = ac.gen(seed)
    k, v, table, ks, vs = ac.paged([(0, max(n, 1)) for _, n in lens], 16, hk, dim, dtype, g, fill=0.0)
    offsets, lengths = ac.offsets_of(lens)
    tokens = int(offsets[-1])
    q = ac.normal(g, (tokens, hq, dim), dtype)
    batch = tcc.PagedBatch(offsets, lengths, table, max_new, max_length)
    out = torch.full_like(q, 7.0)
    _, lse = tcc.paged_attention(ctx, tcc.PagedCache(k, v), batch, q, out=out, return_lse=True)
    bits = ctx.status()
    want = ac.attention_ref(q, seen_lens, ks, vs, dim ** -0.5, True, 0)
    turned = torch.full_like(q, 7.0)
    k2, v2 = k.clone(), v.clone()
    nk, nv = (ac.normal(g, (tokens, hk, dim), dtype) for _ in range(2))
    tcc.kv_append(ctx, tcc.PagedCache(k2, v2), batch, nk, nv, q=q, q_out=turned)
    assert ctx.status() == bits
    return tcc, bits, q, out, want, turned, (k, v), (k2, v2), (nk, nv), table


@pytest.mark.parametrize("dim,hq,hk", [(128, 8, 2), (64, 4, 4), (256, 2, 1)])
@pytest.mark.parametrize("new,most,length", [(3, 1, 30), (5, 4, 5), (200, 100, 300), (130, 129, 130)])
def test_a_request_past_max_new_is_cut(ctx, dim, hq, hk, new, most, length):
    """It counts as one of length 0, reported, and its rows past max_new are
    left alone; the other request is served."""
    lens = [(new, length), (1, 20)]
    tcc, bits, q, out, (want, _, tol, _), turned, old, fresh, (nk, nv), table = _sentinels(
        ctx, lens, [(new, 0), (1, 20)], most, max(length, 20), hq, hk, dim, BF, seed=new)
    assert bits == tcc.STATUS_GEOMETRY
    assert bool((out[most:new] == 7).all()) and float(out[:most].abs().max()) == 0.0
    ac.close(out[new:], want[new:], tol[new:])
    assert bool((turned[most:new] == 7).all()) and torch.equal(turned[:most], q[:most])
    assert torch.equal(turned[new:], q[new:])
    page = int(table[1, 1])
    for a, b, x in zip(old, fresh, (nk, nv)):
        assert torch.equal(b[page, :, 3], x[new])
        a[page, :, 3] = b[page, :, 3]
        assert torch.equal(a, b)


@pytest.mark.parametrize("dim,hq,hk", [(128, 8, 2), (64, 4, 4), (256, 2, 1)])
@pytest.mark.parametrize("new,length", [(2, 1), (7, 3), (200, 199), (300, 40)])
def test_a_request_shorter_than_its_new_tokens_is_impossible(ctx, dim, hq, hk, new, length):
    """Lengths count the new tokens: less than them, but not 0, is reported and
    treated as length 0."""
    lens = [(new, length), (1, 20)]
    tcc, bits, q, out, (want, _, tol, _), turned, old, fresh, (nk, nv), table = _sentinels(
        ctx, lens, [(new, 0), (1, 20)], new, max(length, 20), hq, hk, dim, HF, seed=new)
    assert bits == tcc.STATUS_GEOMETRY
    assert float(out[:new].abs().max()) == 0.0
    ac.close(out[new:], want[new:], tol[new:])
    page = int(table[1, 1])
    for a, b, x in zip(old, fresh, (nk, nv)):
        assert torch.equal(b[page, :, 3], x[new])
        a[page, :, 3] = b[page, :, 3]
        assert torch.equal(a, b)


@pytest.mark.parametrize("bad", [-1, -77, 10 ** 6, 2 ** 31 - 1])
@pytest.mark.parametrize("dim,page", [(64, 8), (128, 16), (128, 256), (256, 32), (80, 64)])
@pytest.mark.parametrize("new", [1, 5, 150])
def test_a_page_outside_the_cache_reads_as_zeros(ctx, new, dim, page, bad):
    """An impossible page number is reported, and no other page's tokens stand
    in for its own."""
    from turbocider_b200 import cuda as tcc
    g = ac.gen(new + page)
    lens = [(new, 700), (new, 300)]
    k, v, table, ks, vs = ac.paged(lens, page, 2, dim, BF, g, fill=50.0)
    first = int((table == 0).nonzero()[0, 0]) if bool((table == 0).any()) else -1   # whose tokens page 0 holds
    which = 0 if first == 1 else 1
    table[which, 1] = bad
    for d in (ks, vs):
        d[which][page:2 * page] = 0
    offsets, lengths = ac.offsets_of(lens)
    q = ac.normal(g, (2 * new, 4, dim), BF)
    y = tcc.paged_attention(ctx, tcc.PagedCache(k, v), tcc.PagedBatch(offsets, lengths, table, new, 700), q)
    assert ctx.status() == tcc.STATUS_GEOMETRY
    want, _, tol, _ = ac.attention_ref(q, lens, ks, vs, dim ** -0.5, True, 0)
    ac.close(y, want, tol)


@pytest.mark.parametrize("dim,hq,hk", [(64, 4, 2), (128, 8, 2), (256, 2, 2)])
@pytest.mark.parametrize("page", [8, 16, 64, 128, 512])
@pytest.mark.parametrize("new,window", [(1, 1), (1, 300), (5, 33), (40, 1000), (150, 7), (300, 520)])
def test_pages_behind_a_window_may_be_given_back(ctx, dim, hq, hk, page, new, window):
    """Pages that end before the first position that any new token sees are
    neither looked up nor read."""
    from turbocider_b200 import cuda as tcc
    g = ac.gen(page + window)
    lens = [(new, n) for n in (new, 1500, 2047, 4100)]
    k, v, table, ks, vs = ac.paged(lens, page, hk, dim, BF, g)
    for b, (_, n) in enumerate(lens):
        gone = max(n - new - window + 1, 0) // page
        for d in (k, v):
            d[table[b, :gone].long()] = float("nan")
        table[b, :gone] = -1
    offsets, lengths = ac.offsets_of(lens)
    q = ac.normal(g, (new * len(lens), hq, dim), BF)
    y = tcc.paged_attention(ctx, tcc.PagedCache(k, v), tcc.PagedBatch(offsets, lengths, table, new, 4100), q,
                            window=window)
    assert ctx.status() == 0
    want, _, tol, _ = ac.attention_ref(q, lens, ks, vs, dim ** -0.5, True, window)
    ac.close(y, want, tol)


def test_more_tiles_than_a_grid_dimension(ctx):
    """Heads of 256: 4100 requests of up to 257 rows make 69700 tiles."""
    from turbocider_b200 import cuda as tcc
    g, dim, page = ac.gen(41), 256, 16
    lens = [(1, 1 + i % 16) for i in range(4100)]
    lens[1234] = (257, 300)
    k, v, table, ks, vs = ac.paged(lens, page, 1, dim, BF, g)
    offsets, lengths = ac.offsets_of(lens)
    q = ac.normal(g, (int(offsets[-1]), 1, dim), BF)
    y, lse = tcc.paged_attention(ctx, tcc.PagedCache(k, v), tcc.PagedBatch(offsets, lengths, table, 257, 300), q,
                                 return_lse=True)
    assert ctx.status() == 0
    want, wlse, tol, tol_lse = ac.attention_ref(q, lens, ks, vs, dim ** -0.5, True, 0)
    ac.close(y, want, tol)
    ac.close(lse, wlse, tol_lse)


def test_more_requests_than_a_grid_dimension(ctx):
    """70000 requests of one token over the same two pages."""
    from turbocider_b200 import cuda as tcc
    g, n, dim = ac.gen(42), 70000, 64
    k, v, table, ks, vs = ac.paged([(1, 13)], 8, 2, dim, HF, g)
    q = ac.normal(g, (n, 4, dim), HF)
    y = tcc.paged_attention(ctx, tcc.PagedCache(k, v),
                            tcc.PagedBatch(torch.arange(n + 1, dtype=torch.int32, device="cuda"),
                                           torch.full((n,), 13, dtype=torch.int32, device="cuda"),
                                           table.expand(n, -1).contiguous(), 1, 13), q)
    assert ctx.status() == 0
    want, _, tol, _ = ac.attention_ref(q, [(n, 13)], ks, vs, dim ** -0.5, False, 0)   # every row sees all 13
    ac.close(y, want, tol)


@pytest.mark.parametrize("dim,n,hk,group", [(256, 700, 8, 16), (128, 600, 8, 32)])
def test_partial_results_past_the_workspaces_bound(ctx, dim, n, hk, group):
    """Requests whose partial results together pass the bound of the workspace
    (all over the same pages, so that the cache stays small)."""
    from turbocider_b200 import cuda as tcc
    g, length = ac.gen(43), 4000
    k, v, table, ks, vs = ac.paged([(1, length)], 64, hk, dim, BF, g)
    q = ac.normal(g, (n, hk * group, dim), BF)
    args = (torch.arange(n + 1, dtype=torch.int32, device="cuda"),
            torch.full((n,), length, dtype=torch.int32, device="cuda"), table.expand(n, -1).contiguous(), 1, length)
    y = tcc.paged_attention(ctx, tcc.PagedCache(k, v), tcc.PagedBatch(*args), q)
    again = tcc.paged_attention(ctx, tcc.PagedCache(k, v), tcc.PagedBatch(*args), q)
    assert ctx.status() == 0 and torch.equal(y, again)
    want, _, tol, _ = ac.attention_ref(q, [(n, length)], ks, vs, dim ** -0.5, False, 0)   # every row sees all of them
    ac.close(y, want, tol)


def test_a_loose_bound_on_the_lengths(ctx):
    """max_length far past what the page table covers asks for no more
    workspace than the table can mean."""
    from turbocider_b200 import cuda as tcc
    g = ac.gen(44)
    lens = [(1, 300 - i) for i in range(64)]
    k, v, table, ks, vs = ac.paged(lens, 16, 8, 128, BF, g)
    offsets, lengths = ac.offsets_of(lens)
    q = ac.normal(g, (64, 32, 128), BF)
    y = tcc.paged_attention(ctx, tcc.PagedCache(k, v), tcc.PagedBatch(offsets, lengths, table, 1, 2 ** 30), q)
    assert ctx.status() == 0
    want, _, tol, _ = ac.attention_ref(q, lens, ks, vs, 128 ** -0.5, True, 0)
    ac.close(y, want, tol)


@pytest.mark.parametrize("length", [150001, 140000])
def test_very_many_shares(ctx, length):
    """64 rows of 64 over so long a cache that the statistics of its shares do
    not fit the memory that the last CTA joins them in."""
    from turbocider_b200 import cuda as tcc
    g = ac.gen(45)
    lens = [(4, length)]
    k, v, table, ks, vs = ac.paged(lens, 256, 1, 64, BF, g)
    offsets, lengths = ac.offsets_of(lens)
    q = ac.normal(g, (4, 16, 64), BF)
    y, lse = tcc.paged_attention(ctx, tcc.PagedCache(k, v), tcc.PagedBatch(offsets, lengths, table, 4, length), q,
                                 return_lse=True)
    assert ctx.status() == 0
    want, wlse, tol, tol_lse = ac.attention_ref(q, lens, ks, vs, 64 ** -0.5, True, 0)
    ac.close(y, want, tol)
    ac.close(lse, wlse, tol_lse)
