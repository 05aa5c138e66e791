"""Attention over a shared prefix: row strides that the kernel's 32-bit offsets do not hold."""

from __future__ import annotations

import pytest
import torch

from leanstack_amd import _lib, kernels

D = 128
LENS = torch.zeros(1, dtype=torch.int32)


def _bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("stride", [(1 << 32) + D, (1 << 31) + D, 1 << 22, _lib.MAX_ACTIVATION_STRIDE + 8])
def test_far_rows_are_refused(stride):
    far = torch.empty(stride + 2 * D, dtype=torch.bfloat16)  # (its pages are never touched)
    prefix, own = far.as_strided((1, 2, D), (2 * D, stride, 1)), far.as_strided((1, 1, 2, D), (2 * D, 2 * D, stride, 1))
    q, near = _bf(1, 4, 1, D), _bf(1, 2, D)
    with pytest.raises(ValueError, match="prefix_k / prefix_v.*stride"):
        kernels.shared_prefix_attention(q, prefix, prefix, near[None], near[None], LENS, 0.1)
    with pytest.raises(ValueError, match="k / v.*stride"):
        kernels.shared_prefix_attention(q, near, near, own, own, LENS, 0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("stride", [1 << 22, 1 << 23, (1 << 31) + 8, 1 << 33, 4])
def test_a_single_row_takes_any_stride(gpu, stride):
    gen = torch.Generator(device=gpu).manual_seed(1)
    q, far, near = (torch.randn(s, generator=gen, device=gpu).bfloat16() for s in ((2, 4, 1, D), (2, 1, D), (2, 2, 1, D)))
    lens = torch.tensor([1, 0], dtype=torch.int32, device=gpu)
    expect = kernels.shared_prefix_attention(q, far, far * 2, near, near * 3, lens, 0.1)
    one = [x.as_strided(x.shape, (*x.stride()[:-2], stride, 1)) for x in (far, far * 2, near, near * 3)]
    assert torch.equal(kernels.shared_prefix_attention(q, *one, lens, 0.1), expect)
