"""How paged attention divides its calls: rules on sizes, no GPU."""
from __future__ import annotations

import pytest

from turbocider_b200 import cuda as tcc

SMS = 148


@pytest.mark.parametrize("dim,rows,places", [(64, 16, 3), (64, 32, 2), (64, 64, 2), (128, 16, 3), (128, 32, 2), (256, 16, 1),
                                             (136, 3, 1), (80, 1, 3)])
def test_rounds_are_counted_by_the_ctas_that_fit(dim, rows, places):
    """An SM holds as many CTAs as their shared memory (64 KB of rings, 128 for
    heads above 128) and registers leave room for."""
    plan = tcc.attention_plan(rows, 1, dim, 8, 8, 1, 6000)
    assert not plan.many_rows and plan.ctas_per_sm == places


@pytest.mark.parametrize("dim,group,new,heads,requests,length", [
    (64, 4, 7, 5, 8, 6000), (64, 8, 4, 8, 1, 20000), (256, 4, 4, 4, 4, 9000), (256, 2, 1, 8, 1, 16000),
    (128, 4, 1, 8, 3, 9000)])
def test_no_last_round_for_a_few(dim, group, new, heads, requests, length):
    """Where one round of CTAs holds the work at the longest share, the shares do
    not start a second one."""
    plan = tcc.attention_plan(group * heads, heads, dim, requests, requests * new, new, length)
    room = SMS * plan.ctas_per_sm
    at_least = requests * heads * -(-length // 1024)
    assert at_least <= room and requests * heads * plan.shares <= room
    assert plan.shares * plan.share_keys >= length


def test_refusals():
    for bad in (dict(head_dim=12), dict(cache_heads=3), dict(page_size=24), dict(max_length=2 ** 30 + 1), dict(window=-1),
                dict(requests=0), dict(sms=0)):
        sizes = dict(n_heads=8, cache_heads=2, head_dim=128, requests=1, tokens=1, max_new=1, max_length=100)
        with pytest.raises(tcc.BackendError, match="would not take"):
            tcc.attention_plan(**{**sizes, **bad})


def test_no_gigabytes_for_a_rounding_of_the_rounds():
    """1 request, 8192 new tokens over 262144 (256 blocks of rows by 8 heads): the
    last round of CTAs is 1 in 14, seven shares would move 1.8 GB to save 0.05 %."""
    plan = tcc.attention_plan(64, 8, 128, 1, 8192, 8192, 262144)
    assert plan.many_rows and plan.shares == 1 and plan.workspace_bytes == 0


@pytest.mark.parametrize("dim", [64, 96, 128, 200, 256])
@pytest.mark.parametrize("heads,group", [(1, 1), (1, 32), (2, 8), (8, 4), (8, 8), (30, 1), (64, 1)])
def test_workspaces_stay_bounded(dim, heads, group):
    """Partial results: never more than 256 MB but for a single request whose one
    tile of rows over its whole cache needs more; many rows' take no longer to
    move than the call's products, or 40 us."""
    for requests in (1, 2, 3, 7, 16, 64, 200, 1000):
        for new in (1, 2, 5, 16, 40, 100, 333, 1000, 4096, 8192):
            for past in (0, 500, 4000, 30000, 262144, 10 ** 6):
                length = new + past
                plan = tcc.attention_plan(heads * group, heads, dim, requests, requests * new, new, length)
                assert plan.shares * plan.share_keys >= length and plan.launches >= 1
                padded = 64 if dim <= 64 else 128 if dim <= 128 else 256
                unit = heads * plan.shares * min(plan.rows, group * new) * (padded + 2) * 4
                assert plan.workspace_bytes <= max(256 << 20, 0 if plan.many_rows else unit + 16), (requests, new, past)
                if plan.many_rows and plan.shares > 1:
                    # written and read at 6.5 TB/s against 4 flops an element of a score at 1.6 PFLOP/s
                    move = 2 * plan.workspace_bytes / 6.5e12
                    compute = 4 * max(requests * new * group, 256 * requests) * heads * length * padded / 1.6e15
                    assert move <= max(compute, 40e-6), (requests, new, past, plan.shares)


@pytest.mark.parametrize("heads,group,new,length,least", [(8, 4, 64, 100000, 8), (8, 4, 300, 30000, 4), (8, 1, 100, 3000, 4),
                                                          (8, 4, 1536, 31537, 2)])
def test_few_blocks_are_split(heads, group, new, length, least):
    assert tcc.attention_plan(heads * group, heads, 128, 1, new, new, length).shares >= least


def test_shares_allow_for_uneven_lengths():
    """Drafted tokens of several requests: a second round that only the longest
    lengths would fill is no reason to split further (three shares of the window
    take 20 us, five 28)."""
    plan = tcc.attention_plan(20, 5, 64, 23, 23 * 4, 7, 6007, window=2048, page_size=32)
    assert plan.rows == 32 and plan.shares == 3
    # one request is as long as it is
    assert tcc.attention_plan(64, 8, 64, 1, 4, 4, 20000).shares * 8 <= SMS * 2
