"""The paged cache's accounts beside many open requests (no GPU)."""

from __future__ import annotations

import copy
import sys

import pytest

from leanstack_amd.paged_cache import PagedKVCache


def calls(work) -> int:
    """Python and C functions that `work` calls or resumes: the same on every machine."""
    count = 0

    def seen(frame, event, arg):
        nonlocal count
        count += event in ("call", "c_call")

    sys.setprofile(seen)
    try:
        work()
    finally:
        sys.setprofile(None)
    return count


def opened(n, pages=None):
    cache = PagedKVCache(1, 1, pages or n, page_rows=16)
    return cache, [cache.open() for _ in range(n)]


def test_a_step_costs_in_proportion_to_its_requests():
    def step(cache, requests):
        cache.reserve(requests, 1)
        cache.batch(requests, 1)
        cache.advance(requests, 1)

    costs = {}
    for n in (32, 512):
        cache, requests = opened(n)
        costs[n] = calls(lambda: step(cache, requests))
        assert all(r.rows == 1 for r in requests)
    assert costs[512] <= 16 * costs[32]


def test_one_request_costs_the_same_beside_any_number():
    """In a step, forked, truncated and closed."""
    def life(cache, r):
        cache.reserve([r], 1)
        cache.advance([r], 1)
        other = cache.fork(r)
        cache.truncate(r, 0)
        cache.close(other)
        cache.close(r)

    costs = []
    for n in (4, 512):
        cache, requests = opened(n)
        costs.append(calls(lambda: life(cache, requests[-1])))
        assert cache.free_pages == n
        with pytest.raises(ValueError, match="not open"):
            cache.close(requests[-1])
    assert costs[0] == costs[1]


def test_requests_keep_their_order_when_others_end():
    cache, requests = opened(6)
    for r in requests:
        cache.reserve([r], 16)
        cache.advance([r], 16)
    cache.close(requests[0])
    cache.close(requests[3])
    assert cache.compact() == 4
    assert sorted(requests[i].pages[0] for i in (1, 2, 4, 5)) == [0, 1, 2, 3]
    assert [len(cache.batch([requests[i]])[0][0]) for i in (1, 2, 4, 5)] == [1] * 4


def test_a_copy_with_its_requests():
    """A cache that is copied together with its requests knows the copies, and only them."""
    cache, requests = opened(3, pages=9)
    cache.reserve(requests, 5)
    cache.advance(requests, 5)
    other, theirs = copy.deepcopy((cache, requests))
    other.reserve(theirs, 20)
    other.advance(theirs[:1], 20)
    other.close(theirs[1])
    assert [r.rows for r in requests] == [5] * 3 and theirs[0].rows == 25
    assert cache.free_pages == 6 and cache.batch(requests)[1].tolist() == [5] * 3
    for r in (requests[0], theirs[1]):
        with pytest.raises(ValueError, match="not open"):
            other.batch([r])


@pytest.mark.parametrize("name", [None, 0, [], "a", object()])
def test_what_is_no_request_is_refused(name):
    cache, _ = opened(2)
    with pytest.raises(ValueError, match="not open"):
        cache.batch([name])
