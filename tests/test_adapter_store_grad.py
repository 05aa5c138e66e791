"""Adapters under training are loaded as values: a store keeps no graph of them."""

from __future__ import annotations

import pytest
import torch

from leanstack_amd.adapters import AdapterStore
from tests.helpers import seeded_normal


@pytest.mark.parametrize("gate_up", [False, True])
def test_a_store_takes_parameters_without_their_graph(gate_up):
    n, k, r = 64, 96, 5
    a, b = (torch.nn.Parameter(seeded_normal(shape, 1.0, seed)) for shape, seed in (((r, k), 1), ((n, r), 2)))
    plain = AdapterStore(2, n, k, 16, gate_up=gate_up, device="cpu")
    plain.load(0, a.detach(), b.detach(), 0.5)
    plain.load(1, a.detach(), b.detach(), 0.5)
    store = AdapterStore(2, n, k, 16, gate_up=gate_up, device="cpu")
    made = AdapterStore.of(torch.stack((a, a)), torch.stack((b, b)), torch.full((2,), 0.5, requires_grad=True), gate_up=gate_up)
    for _ in range(2):
        store.load(0, a, b, 0.5)
        store.load_parts(1, [(a, b)], 0.5)
    for s in (store, made):
        for x, expect in ((s.a_tiles, plain.a_tiles), (s.b_tiles, plain.b_tiles), (s.scales, plain.scales)):
            assert not x.requires_grad and x.grad_fn is None and torch.equal(x, expect)
    store.clear(0)
    assert store.b_tiles.grad_fn is None and a.grad_fn is None and a.requires_grad
