"""lora_linear refuses before its first launch: a call that raises has written nothing."""

from __future__ import annotations

import pytest
import torch

from leanstack_amd import _lib, kernels
from leanstack_amd.adapters import AdapterStore
from leanstack_amd.layout import PackedWeight
from tests.helpers import seeded_normal

N, K = 64, 32
BAD_INDEX = [torch.zeros(3, dtype=torch.int64), torch.zeros(2, dtype=torch.int32), torch.zeros(6, dtype=torch.int32)[::2],
             torch.zeros(0, dtype=torch.int32)]


def _on(device, index):
    """`index` there, with its stride."""
    return index.to(device) if index.is_contiguous() else index.repeat_interleave(2).to(device)[::2]


def _arguments(device, gate_up=False):
    layout = _lib.LAYOUT_MFMA16X32_GATEUP if gate_up else _lib.LAYOUT_MFMA16X32
    weight = PackedWeight.from_rowmajor(seeded_normal((N, K), 1, 3).to(device), layout)
    return seeded_normal((3, K), 1, 2).to(device), weight, AdapterStore(2, N, K, 8, gate_up=gate_up, device=device)


@pytest.mark.parametrize("index", BAD_INDEX)
@pytest.mark.parametrize("gate_up", [False, True])
def test_the_index_is_checked_first(index, gate_up):
    x, weight, store = _arguments("cpu", gate_up)
    with pytest.raises(ValueError, match="index"):
        kernels.lora_linear(x, weight, store, index, epilogue=_lib.EPI_SILU_MUL if gate_up else _lib.EPI_NONE)


@pytest.mark.gpu
@pytest.mark.parametrize("index", BAD_INDEX)
def test_a_refused_call_leaves_its_output(gpu, index):
    x, weight, store = _arguments(gpu)
    hidden, index = torch.full((3, N), 5.0, device=gpu).bfloat16(), _on(gpu, index)
    with pytest.raises(ValueError, match="index"):
        kernels.lora_linear(x, weight, store, index, out=hidden)
    with pytest.raises(ValueError, match="index"):
        kernels.lora_linear(x, weight, store, index, epilogue=_lib.EPI_RESIDUAL_ADD, residual=hidden, out=hidden)
    assert bool((hidden == 5).all())


@pytest.mark.gpu
def test_tensors_of_another_device_are_refused_first(gpu):
    x, weight, store = _arguments(gpu)
    index = torch.zeros(3, dtype=torch.int32)
    out = torch.full((3, N), 5.0, device=gpu).bfloat16()
    for args, what in (((x, weight, store, index), "index is on"), ((x, weight, _arguments("cpu")[2], index.to(gpu)), "store is on")):
        with pytest.raises(ValueError, match=what):
            kernels.lora_linear(*args, out=out)
    assert bool((out == 5).all())
    assert kernels.lora_linear(x[:0], weight, store, index[:0].to(gpu)).shape == (0, N)
