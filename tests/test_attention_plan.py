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
