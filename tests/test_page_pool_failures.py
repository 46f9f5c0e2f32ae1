"""A step of the page pool that cannot be had changes nothing."""
from __future__ import annotations

import pytest

from turbocider_b200 import cuda as tcc
from turbocider_b200.attention import PagePool


def state(pool):
    requests = sorted(pool._pages)
    return list(pool._free), requests, pool.table(requests), [pool.length(r) for r in requests]


def pool_with_one():
    pool = PagePool(4, 8)
    pool.grow("a", 3)
    return pool


@pytest.mark.parametrize("requests,new,error", [
    (["a", "b"], [9, 100], MemoryError),         # the second does not fit
    (["b", "a"], [8, 100], MemoryError),
    (["b", "c", "a"], [8, 8, 16], MemoryError),  # together one page too many
    (["a", "a"], [20, 20], MemoryError),         # twice the same one
    (["a", "b"], [9, -1], ValueError),
    (["a", "b"], [9], ValueError),               # lists of different lengths
    (["a"], [9, 1], ValueError),
    ([], [], ValueError),                        # nobody
])
def test_a_failed_step_takes_nothing(monkeypatch, requests, new, error):
    monkeypatch.setattr(tcc, "PagedBatch", lambda *a: a)
    pool = pool_with_one()
    before = state(pool)
    with pytest.raises(error):
        pool.step(requests, new, "cpu")
    assert state(pool) == before


def test_a_step_whose_batch_cannot_be_built_takes_nothing(monkeypatch):
    def refuse(*a):
        raise tcc.BackendError("no device")
    monkeypatch.setattr(tcc, "PagedBatch", refuse)
    pool = pool_with_one()
    before = state(pool)
    with pytest.raises(tcc.BackendError):
        pool.step(["a", "b", "a"], [9, 8, 3], "cpu")
    assert state(pool) == before


def test_a_step_retried_after_an_eviction(monkeypatch):
    monkeypatch.setattr(tcc, "PagedBatch", lambda *a: a)
    pool = pool_with_one()
    pool.grow("old", 16)
    with pytest.raises(MemoryError):
        pool.step(["a", "b"], [3, 9], "cpu")
    pool.release("old")
    offsets, lengths, table, max_new, max_length = pool.step(["a", "b"], [3, 9], "cpu")
    assert offsets.tolist() == [0, 3, 12] and lengths.tolist() == [6, 9]
    assert (max_new, max_length) == (9, 9) and table.shape == (2, 2)


def test_a_request_may_come_twice_in_a_step(monkeypatch):
    """Its second part goes behind the first."""
    monkeypatch.setattr(tcc, "PagedBatch", lambda *a: a)
    pool = pool_with_one()
    offsets, lengths, table, _, _ = pool.step(iter(["a", "a"]), iter([3, 5]), "cpu")
    assert offsets.tolist() == [0, 3, 8] and lengths.tolist() == [6, 11] and table[0].tolist() == table[1].tolist()
