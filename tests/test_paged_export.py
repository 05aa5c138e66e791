"""Requests of the paged cache that go on in an ArenaKVCache: what does not fit is refused before
anything is written (no GPU)."""

from __future__ import annotations

import pytest

from leanstack_amd.kv_cache import ArenaKVCache
from leanstack_amd.paged_cache import PagedKVCache


@pytest.mark.parametrize("target,names", [
    (dict(num_layers=1), "layers"), (dict(num_layers=3), "layers"), (dict(num_key_value_heads=3), "heads"),
    (dict(head_dim=64), "128"), (dict(capacity=19), "room"),
])
def test_export_refuses_a_cache_that_does_not_fit(target, names):
    cache = PagedKVCache(2, 1, 4, page_rows=16)
    a = cache.open()
    cache.reserve([a], 20)
    cache.advance([a], 20)
    arena = ArenaKVCache(**(dict(num_layers=2, num_key_value_heads=1, head_dim=128, capacity=32) | target))
    with pytest.raises(ValueError, match=names):
        cache.export(a, arena)
    assert not any(arena.layer_seq_lens)


def test_export_refuses_when_a_later_layer_is_full():
    """Nothing is written: the first layers, which have room, neither."""
    cache = PagedKVCache(2, 1, 4, page_rows=16)
    a = cache.open()
    cache.reserve([a], 20)
    cache.advance([a], 20)
    arena = ArenaKVCache(2, 1, 128, 32)
    arena.advance(1, 13)
    with pytest.raises(ValueError, match="room"):
        cache.export(a, arena)
    assert arena.layer_seq_lens == [0, 13]


def test_export_of_a_request_without_rows():
    cache = PagedKVCache(2, 1, 4, page_rows=16)
    arena = ArenaKVCache(2, 1, 128, 32)
    cache.export(cache.open(), arena)
    assert arena.layer_seq_lens == [0, 0]
