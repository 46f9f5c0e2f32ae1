"""Host side of the paged cache (no GPU)."""
from __future__ import annotations

import random

import pytest

from turbocider_b200.attention import PagePool


def test_pages_are_taken_as_requests_grow_and_given_back():
    pool = PagePool(10, 16)
    assert pool.grow("a", 16) == 16 and pool.free_pages == 9
    assert pool.grow("a", 1) == 17 and pool.free_pages == 8
    assert pool.grow("b", 0) == 0 and pool.free_pages == 8
    assert pool.grow("b", 33) == 33 and pool.free_pages == 5
    table = pool.table(["a", "b", "c"])
    assert [len(r) for r in table] == [3, 3, 3] and table[2] == [-1] * 3 and table[0][2] == -1
    assert len({p for r in table for p in r if p >= 0}) == 5
    pool.release("a")
    pool.release("a")
    assert pool.free_pages == 7 and pool.length("a") == 0 and pool.length("b") == 33


def test_a_request_that_does_not_fit_takes_nothing():
    pool = PagePool(3, 8)
    pool.grow(1, 17)
    with pytest.raises(MemoryError):
        pool.grow(2, 1)
    with pytest.raises(MemoryError):
        pool.grow(1, 8)
    with pytest.raises(ValueError):
        pool.grow(1, -1)
    assert pool.length(1) == 17 and pool.length(2) == 0 and pool.free_pages == 0


def test_no_page_is_ever_shared():
    rng, pool, live = random.Random(3), PagePool(64, 4), {}
    for _ in range(2000):
        r = rng.randrange(12)
        if rng.random() < 0.3:
            pool.release(r)
            live.pop(r, None)
        else:
            n = rng.randrange(9)
            try:
                live[r] = pool.grow(r, n)
            except MemoryError:
                pass
        used = [p for row in pool.table(list(live)) for p in row if p >= 0]
        assert len(used) == len(set(used)) == sum(-(-n // 4) for n in live.values())
        assert len(used) + pool.free_pages == 64
