"""Which request has which page (no GPU: a pool in host memory)."""

from __future__ import annotations

import pytest
import torch

from leanstack_amd.paged_cache import PagedKVCache


def cache_of(pages=8, page_rows=16):
    cache = PagedKVCache(2, 1, pages, page_rows=page_rows)
    # every page says which it was
    cache.storage[:] = torch.arange(pages, dtype=torch.uint8)[:, None, None, None]
    cache.exponents[:] = torch.arange(pages, dtype=torch.uint8)[:, None, None] + 100
    return cache


def named(cache, page):
    """Which page's bytes a page holds, the same in all layers."""
    got = set(cache.storage[:, :, page].unique().tolist()) | {e - 100 for e in cache.exponents[:, :, page].unique().tolist()}
    assert len(got) == 1
    return got.pop()


def grow(cache, requests, n):
    cache.reserve(requests, n)
    cache.advance(requests, n)


def test_pages_of_rows():
    cache = cache_of()
    a, b = cache.open(), cache.open()
    grow(cache, [a, b], [1, 17])
    assert (a.pages, b.pages, cache.free_pages) == ([0], [1, 2], 5)
    grow(cache, [a, b], [15, 15])
    assert (a.pages, b.pages) == ([0], [1, 2])
    grow(cache, [a, b], [1, 0])
    assert (a.pages, b.pages, a.rows, b.rows) == ([0, 3], [1, 2], 17, 32)
    table, lens = cache.batch([b, a], [0, 4])
    assert table.tolist() == [[1, 2], [0, 3]] and lens.tolist() == [32, 21] and table.dtype is lens.dtype is torch.int32
    wide, rows = torch.full((2, 5), 9, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    cache.batch([b, a], table=wide, lens=rows)
    assert wide.tolist() == [[1, 2, -1, -1, -1], [0, 3, -1, -1, -1]] and rows.tolist() == [32, 17]
    cache.close(a)
    assert cache.free_pages == 6 and grow(cache, [b], 1) is None and b.pages == [1, 2, 0]  # the lowest free page


def test_reserve_changes_nothing_when_pages_are_short():
    cache = cache_of(pages=3)
    a, b = cache.open(), cache.open()
    grow(cache, [a], 20)
    with pytest.raises(ValueError, match="are free"):
        cache.reserve([a, b], [1, 17])
    assert (a.pages, b.pages, cache.free_pages) == ([0, 1], [], 1)
    grow(cache, [b], 16)
    f = cache.fork(a)
    with pytest.raises(ValueError, match="are free"):  # the copy of the begun page needs one
        cache.reserve([f], 1)
    assert f.pages == a.pages and cache.holders(1) == 2
    grow(cache, [f], 0)


def test_fork_shares_until_one_writes():
    cache = cache_of()
    a = cache.open()
    grow(cache, [a], 20)
    b = cache.fork(a)
    assert b.pages == a.pages and [cache.holders(p) for p in a.pages] == [2, 2] and cache.free_pages == 6
    grow(cache, [b], 3)
    assert b.pages == [0, 2] and a.pages == [0, 1] and named(cache, 2) == 1
    grow(cache, [a], 3)  # a is alone with it now
    assert a.pages == [0, 1] and cache.free_pages == 5
    cache.close(a)
    assert cache.free_pages == 6 and cache.holders(0) == 1 and cache.holders(1) == 0


def test_fork_at_a_page_end_copies_nothing():
    cache = cache_of()
    a = cache.open()
    grow(cache, [a], 32)
    b = cache.fork(a)
    grow(cache, [a, b], 1)
    assert a.pages == [0, 1, 2] and b.pages == [0, 1, 3] and named(cache, 3) == 3


def test_several_forks_in_one_step():
    cache = cache_of()
    a = cache.open()
    grow(cache, [a], 5)
    b, c = cache.fork(a), cache.fork(a)
    grow(cache, [c, a, b], 1)
    assert sorted([a.pages[0], b.pages[0], c.pages[0]]) == [0, 1, 2]
    assert all(cache.holders(p) == 1 and named(cache, p) == 0 for p in (0, 1, 2))


def test_fork_of_reserved_pages():
    """Pages that are reserved and hold no row are not shared."""
    cache = cache_of()
    a = cache.open()
    grow(cache, [a], 16)
    cache.reserve([a], 20)
    b = cache.fork(a)
    assert len(a.pages) == 3 and b.pages == [0]
    grow(cache, [b], 1)
    assert b.pages[1] not in a.pages


def test_rows_for_a_shared_page_are_refused():
    """A fork between reserve() and batch(): the new row would be written into both."""
    cache = cache_of()
    a, full = cache.open(), cache.open()
    grow(cache, [a, full], [5, 16])
    cache.reserve([a], 3)
    b = cache.fork(a)
    cache.fork(full)
    for call in (lambda: cache.batch([a], 1), lambda: cache.batch([full, b], [0, 1])):
        with pytest.raises(ValueError, match="another request holds"):
            call()
    cache.batch([a, b, full])
    cache.reserve([b], 3)
    for r in (a, b):
        assert cache.batch([r], 3)[1].tolist() == [8]
    cache.reserve([full], 1)
    cache.batch([full], 1)


def test_truncate():
    cache = cache_of()
    a = cache.open()
    grow(cache, [a], 40)
    b = cache.fork(a)
    cache.truncate(a, 17)
    assert a.pages == [0, 1] and cache.holders(2) == 1
    cache.truncate(b, 16)
    assert b.pages == [0] and cache.holders(2) == 0
    cache.truncate(b, 0)
    assert b.pages == [] and cache.holders(0) == 1
    with pytest.raises(ValueError):
        cache.truncate(b, 1)
    with pytest.raises(ValueError):
        cache.truncate(a, -1)


def test_truncated_into_a_shared_page():
    """A cut back into a page that another still reads: it is copied before the next row."""
    cache = cache_of()
    a = cache.open()
    grow(cache, [a], 32)
    b = cache.fork(a)
    cache.truncate(b, 20)
    grow(cache, [b], 4)
    assert a.pages == [0, 1] and b.pages == [0, 2] and named(cache, 2) == 1


def test_compact():
    cache = cache_of()
    requests = [cache.open() for _ in range(4)]
    for r in requests:
        grow(cache, [r], 32)
    shared = cache.fork(requests[3])
    cache.close(requests[0])
    cache.close(requests[2])
    assert cache.compact() == 4
    assert requests[1].pages == [2, 3] and requests[3].pages == [0, 1] == shared.pages
    assert [named(cache, p) for p in range(4)] == [6, 7, 2, 3] and cache.holders(0) == 2 and cache.free_pages == 4
    grow(cache, [requests[1]], 1)
    assert requests[1].pages == [2, 3, 4]
    assert cache.compact() == 5 and requests[1].pages == [2, 3, 4]


def test_requests_of_other_caches_and_bad_numbers_are_refused():
    cache, other = cache_of(), cache_of()
    a, b = cache.open(), other.open()
    for call in (lambda: cache.reserve([b], 1), lambda: cache.fork(b), lambda: cache.close(b), lambda: cache.batch([a, b]),
                 lambda: cache.reserve([a, a], 1), lambda: cache.reserve([a], [1, 2]), lambda: cache.reserve([a], -1),
                 lambda: cache.advance([a], 1), lambda: cache.batch([a], 1)):
        with pytest.raises(ValueError):
            call()
    cache.close(a)
    with pytest.raises(ValueError):
        cache.close(a)
    with pytest.raises(ValueError):
        cache.reserve([a], 1)
    b = cache.open()
    for table in (torch.zeros((2, 4), dtype=torch.int32), torch.zeros((1, 4), dtype=torch.long), torch.zeros(4, dtype=torch.int32)):
        with pytest.raises(ValueError):
            cache.batch([b], table=table)
    with pytest.raises(ValueError):
        cache.batch([b], lens=torch.zeros(2, dtype=torch.int32))


def test_no_requests():
    cache = cache_of()
    cache.reserve([], 1)
    table, lens = cache.batch([])
    assert table.shape == (0, 1) and lens.shape == (0,)
    assert cache.compact() == 0


@pytest.mark.parametrize("kwargs", [dict(num_layers=0), dict(num_pages=0), dict(num_key_value_heads=0), dict(page_rows=48),
                                    dict(page_rows=8), dict(page_rows=2048), dict(page_rows=0)])
def test_bad_pools(kwargs):
    with pytest.raises(ValueError):
        PagedKVCache(**(dict(num_layers=1, num_key_value_heads=1, num_pages=1) | kwargs))


def test_existing_pools():
    storage, exponents = torch.zeros((2, 2, 5, 3, 4, 2048), dtype=torch.uint8), torch.zeros((2, 2, 5, 3, 4), dtype=torch.uint8)
    cache = PagedKVCache.of(storage, exponents)
    assert (cache.num_layers, cache.num_pages, cache.num_key_value_heads, cache.page_rows) == (2, 5, 3, 64)
    assert cache.storage.data_ptr() == storage.data_ptr() and cache.free_pages == 5
    for bad in ((storage[:, :1], exponents[:, :1]), (storage[..., :1024], exponents), (storage.to(torch.int8), exponents),
                (storage, exponents[:, :, :4]), (storage[:, :, :, :, :3], exponents[..., :3]), (storage[:, :, ::2], exponents[:, :, ::2]),
                (storage[0], exponents[0])):
        with pytest.raises(ValueError):
            PagedKVCache.of(*bad)
