"""Paged attention on a B200 against a 64-bit reference: head dimensions,
groups, page sizes, layouts, strides, masks that leave rows empty, lengths of
zero and one, splits of long caches, NaN in every unused place of the cache."""
from __future__ import annotations

import math

import pytest
import torch

import attn_cases as ac

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def attend(ctx, lens, page, hq, hk, dim, dtype, seed, causal=True, window=0, token_major=False, scale=None, stream=None,
           q_view=None, out_view=None, fill=float("nan"), slack=0):
    from turbocider_b200 import cuda as tcc
    g = ac.gen(seed)
    k, v, table, ks, vs = ac.paged(lens, page, hk, dim, dtype, g, token_major, fill=fill)
    offsets, lengths = ac.offsets_of(lens)
    tokens = int(offsets[-1])
    q = ac.normal(g, (tokens, hq, dim), dtype, 1.2)
    if q_view:
        q = q_view(q)
    out = out_view(tokens, hq, dim, dtype) if out_view else None
    cache = tcc.PagedCache(k, v, token_major)
    batch = tcc.PagedBatch(offsets, lengths, table, max(n for n, _ in lens) + slack,
                           max(n for _, n in lens) + slack * page)
    torch.cuda.synchronize()
    y, lse = tcc.paged_attention(ctx, cache, batch, q, scale=scale, causal=causal, window=window, out=out,
                                 return_lse=True, stream=stream)
    torch.cuda.synchronize()
    assert ctx.status() == 0
    want, wlse, tol, tol_lse = ac.attention_ref(q, lens, ks, vs, dim ** -0.5 if scale is None else scale, causal, window)
    ac.close(y, want, tol, "out")
    assert torch.equal(torch.isinf(lse), torch.isinf(wlse)) and not bool(torch.isnan(lse).any())
    fine = torch.isfinite(wlse)
    ac.close(lse[fine], wlse[fine], tol_lse[fine], "lse")
    return y, lse


RAGGED = [(1, 1), (1, 17), (1, 0), (1, 700), (1, 64), (0, 50), (1, 128), (1, 1500)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hq,hk,dim,page", [(8, 2, 128, 16), (4, 4, 64, 8), (24, 1, 128, 64), (5, 1, 80, 32),
                                            (6, 2, 96, 256), (3, 3, 40, 16), (16, 2, 256, 16), (2, 1, 160, 128),
                                            (40, 2, 72, 16)])
def test_single_tokens(ctx, dtype, hq, hk, dim, page):
    attend(ctx, RAGGED, page, hq, hk, dim, dtype, seed=dim + page)


CHUNKS = [(3, 3), (7, 120), (33, 33), (0, 9), (130, 611), (1, 300), (5, 0), (64, 64)]


@pytest.mark.parametrize("causal,window", [(True, 0), (True, 1), (True, 37), (False, 0), (False, 20), (True, 5000)])
@pytest.mark.parametrize("hq,hk,dim,page,dtype", [(8, 2, 128, 16, BF), (3, 1, 64, 8, HF), (2, 2, 96, 128, HF),
                                                  (10, 1, 128, 32, HF), (4, 2, 256, 64, BF)])
def test_chunks_and_masks(ctx, causal, window, hq, hk, dim, page, dtype):
    attend(ctx, CHUNKS, page, hq, hk, dim, dtype, seed=window + dim, causal=causal, window=window)


@pytest.mark.parametrize("new,length", [(127, 127), (128, 128), (129, 129), (255, 1000), (256, 513), (257, 257),
                                        (1, 4097), (16, 4096), (300, 2500)])
@pytest.mark.parametrize("hq,hk,dim", [(2, 1, 128), (4, 4, 64)])
def test_sizes_around_the_tiles(ctx, new, length, hq, hk, dim):
    attend(ctx, [(new, length), (max(new - 1, 1), length - 1)], 16, hq, hk, dim, BF, seed=new)


@pytest.mark.parametrize("page", [512, 4096])
@pytest.mark.parametrize("lens", [[(1, 1300), (1, 90)], [(9, 700), (1, 1)], [(200, 1300), (90, 90)]])
def test_pages_larger_than_a_step(ctx, page, lens):
    attend(ctx, lens, page, 4, 2, 128, BF, seed=page)


@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("new", [1, 6, 90])
def test_many_requests(ctx, new, window):
    """More requests than a warp looks up at once, of all sizes, empty ones
    among them."""
    lens = [((i * 7) % (new + 1), (i * 7) % (new + 1) + (i * 13) % 200) for i in range(71)] + [(0, 0), (new, 0), (0, 5)]
    attend(ctx, lens, 16, 6, 2, 64, BF, seed=new, window=window)


def test_rows_that_see_nothing_give_zeros(ctx):
    # more new tokens than cached ones: the first sit before the cache's start
    y, lse = attend(ctx, [(1, 0), (4, 0), (200, 0), (2, 30)], 16, 4, 2, 128, BF, seed=3)
    assert float(y[:205].abs().max()) == 0.0 and bool(torch.isneginf(lse[:205]).all())


@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("lens", [[(1, 333), (1, 20)], [(150, 333), (70, 70)]])
def test_layouts_and_strides(ctx, token_major, lens):
    # q a slice of a wider row, out with a padded row; then both head-major
    def q_slice(q):
        wide = torch.zeros((q.shape[0], q.shape[1] + 3, q.shape[2]), dtype=q.dtype, device="cuda")
        wide[:, 2:-1] = q
        return wide[:, 2:-1]

    def q_heads_first(q):
        return q.transpose(0, 1).contiguous().transpose(0, 1)

    def padded(t, h, d, dtype):
        return torch.empty((t, h, d + 8), dtype=dtype, device="cuda")[..., :d]

    def odd(t, h, d, dtype):
        return torch.empty((t, h, d + 3), dtype=dtype, device="cuda")[..., 1:d + 1]

    def q_odd(q):
        wide = torch.zeros((q.shape[0], q.shape[1], q.shape[2] + 3), dtype=q.dtype, device="cuda")
        wide[..., 1:-2] = q
        return wide[..., 1:-2]

    for qv, ov in ((q_slice, padded), (q_heads_first, padded), (q_odd, odd)):
        attend(ctx, lens, 16, 6, 2, 128, BF, seed=5, token_major=token_major, q_view=qv, out_view=ov)


def test_hints_may_be_larger_than_the_values(ctx):
    attend(ctx, [(1, 100), (1, 5)], 16, 4, 2, 64, BF, seed=6, slack=50)
    attend(ctx, [(140, 200), (1, 5)], 16, 4, 2, 64, BF, seed=6, slack=50)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3, 4.0])
def test_scales(ctx, scale):
    # 4.0: a few keys take all the weight
    attend(ctx, [(1, 900), (40, 90), (300, 700)], 16, 2, 1, 64, BF, seed=8, scale=scale)


@pytest.mark.parametrize("lens", [[(1, 2000), (1, 30)], [(200, 900)]])
def test_own_stream_and_repeats_are_bit_equal(ctx, lens):
    side = torch.cuda.Stream()
    first = attend(ctx, lens, 16, 8, 2, 128, BF, seed=9)
    with torch.cuda.stream(side):
        for _ in range(3):
            again = attend(ctx, lens, 16, 8, 2, 128, BF, seed=9, stream=side)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_a_nan_query_stays_in_its_row(ctx):
    from turbocider_b200 import cuda as tcc
    for lens in ([(1, 300), (1, 40)], [(150, 300), (3, 40)]):
        g = ac.gen(11)
        k, v, table, _, _ = ac.paged(lens, 16, 2, 128, BF, g)
        offsets, lengths = ac.offsets_of(lens)
        q = ac.normal(g, (int(offsets[-1]), 4, 128), BF)
        args = (ctx, tcc.PagedCache(k, v), tcc.PagedBatch(offsets, lengths, table, max(n for n, _ in lens), 300))
        clean = tcc.paged_attention(*args, q)
        q[0, 1, 5] = float("nan")
        y, lse = tcc.paged_attention(*args, q, return_lse=True)
        assert bool(torch.isnan(y[0, 1]).all()) and bool(torch.isnan(lse[0, 1]))
        y[0, 1] = clean[0, 1]
        assert torch.equal(y, clean)


def test_impossible_values_on_the_device_are_reported(ctx):
    from turbocider_b200 import cuda as tcc
    g = ac.gen(12)
    for new in (1, 150):
        lens = [(new, 300), (new, 200)]
        k, v, table, _, _ = ac.paged(lens, 16, 2, 64, HF, g, fill=0.0)
        offsets, lengths = ac.offsets_of(lens)
        q = ac.normal(g, (2 * new, 4, 64), HF)
        cache = tcc.PagedCache(k, v)
        good = tcc.paged_attention(ctx, cache, tcc.PagedBatch(offsets, lengths, table, new, 300), q)
        assert ctx.status() == 0
        bad_page, long, far = table.clone(), lengths.clone(), offsets.clone()
        bad_page[1, 2] = k.shape[0]
        long[1] = 10 ** 6
        far[2] = 10 ** 6
        for o, n, t in ((offsets, lengths, bad_page), (offsets, long, table), (far, lengths, table)):
            y = tcc.paged_attention(ctx, cache, tcc.PagedBatch(o, n, t, new, 300), q)
            assert ctx.status() == tcc.STATUS_GEOMETRY
            assert torch.equal(y[:new], good[:new])   # the other request is untouched
        assert ctx.status() == 0


def test_refusals(ctx):
    from turbocider_b200 import cuda as tcc
    g = ac.gen(13)
    lens = [(2, 30)]
    k, v, table, _, _ = ac.paged(lens, 16, 2, 64, BF, g)
    offsets, lengths = ac.offsets_of(lens)
    batch = tcc.PagedBatch(offsets, lengths, table, 2, 30)
    cache = tcc.PagedCache(k, v)
    q = ac.normal(g, (2, 4, 64), BF)

    def refused(match, fn, *a, **kw):
        with pytest.raises(tcc.BackendError, match=match):
            fn(*a, **kw)

    refused("multiple of the cache's heads", tcc.paged_attention, ctx, cache, batch, q[:, :3])
    refused("cache's type", tcc.paged_attention, ctx, cache, batch, q.half())
    refused("head_dim", tcc.paged_attention, ctx, cache, batch, q[..., :32])
    refused("window", tcc.paged_attention, ctx, cache, batch, q, window=-1)
    refused("scale", tcc.paged_attention, ctx, cache, batch, q, scale=math.inf)
    refused("overlapping head", tcc.paged_attention, ctx, cache, batch, q, out=q.new_empty((1, 4, 64)).expand(2, 4, 64))
    refused("max_new", tcc.paged_attention, ctx, cache, tcc.PagedBatch(offsets, lengths, table, 0, 30), q)
    refused("2\\^30", tcc.paged_attention, ctx, cache, tcc.PagedBatch(offsets, lengths, table, 2, 2 ** 31), q)
    odd = torch.empty((4, 2, 12, 64), dtype=BF, device="cuda")
    refused("power of two", tcc.paged_attention, ctx, tcc.PagedCache(odd, odd), batch, q)
    far = torch.empty(4 * 2 * 16 * 64 + 8, dtype=BF, device="cuda")[4:-4].view(4, 2, 16, 64)
    refused("16-byte aligned", tcc.paged_attention, ctx, tcc.PagedCache(far, far), batch, q)
    shared = torch.empty((1, 2, 16, 64), dtype=BF, device="cuda").expand(4, 2, 16, 64)
    refused("overlapping cache", tcc.paged_attention, ctx, tcc.PagedCache(shared, shared), batch, q)
    refused("f16 or bf16", tcc.paged_attention, ctx, tcc.PagedCache(k.float(), v.float()), batch, q.float())
    refused("same shape", tcc.PagedCache, k, v[:, :, :8])
    refused("device tensors", tcc.PagedCache, k.cpu(), v.cpu())
    refused("device", tcc.PagedBatch, offsets.cpu(), lengths, table, 2, 30)
    refused("device", tcc.PagedBatch, offsets, lengths, table.cpu(), 2, 30)
    refused("context's device", tcc.paged_attention, ctx, cache, batch, q.cpu())
    refused("int32", tcc.PagedBatch, offsets.long(), lengths, table, 2, 30)
    refused("rows", tcc.PagedBatch, offsets[:1], lengths, table, 2, 30)
    assert ctx.status() == 0
    # no tokens, no work
    none = tcc.PagedBatch(torch.zeros(2, dtype=torch.int32, device="cuda"), lengths, table, 0, 30)
    assert tcc.paged_attention(ctx, cache, none, q[:0]).shape == (0, 4, 64)


def test_offsets_past_32_bits(ctx):
    """A cache of more than 2^32 elements: pages at both ends."""
    from turbocider_b200 import cuda as tcc
    pages, page, hk, dim = 2 ** 32 // (2 * 16 * 128) + 40, 16, 2, 128
    k = torch.zeros((pages, hk, page, dim), dtype=BF, device="cuda")
    v = torch.zeros_like(k)
    g = ac.gen(14)
    for new in (1, 150):
        n = 160
        ks, vs = [ac.normal(g, (n, hk, dim), BF)], [ac.normal(g, (n, hk, dim), BF)]
        table = torch.tensor([[pages - 1 - j if j % 2 else j for j in range(n // page)]], dtype=torch.int32)
        for j, pg in enumerate(table[0].tolist()):
            k[pg] = ks[0][j * page:(j + 1) * page].transpose(0, 1)
            v[pg] = vs[0][j * page:(j + 1) * page].transpose(0, 1)
        offsets, lengths = ac.offsets_of([(new, n)])
        q = ac.normal(g, (new, 4, dim), BF)
        y = tcc.paged_attention(ctx, tcc.PagedCache(k, v), tcc.PagedBatch(offsets, lengths, table.cuda(), new, n), q)
        want, _, tol, _ = ac.attention_ref(q, [(new, n)], ks, vs, dim ** -0.5, True, 0)
        ac.close(y, want, tol)
    assert ctx.status() == 0


@pytest.mark.parametrize("window", [2**31 - 1, 2**31 + 5, 2**32 + 3])
@pytest.mark.parametrize("causal", [True, False])
def test_windows_past_32_bits_hide_nothing(ctx, causal, window):
    attend(ctx, [(1, 90), (40, 90)], 16, 4, 2, 64, BF, seed=31, causal=causal, window=window)
