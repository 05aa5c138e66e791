"""Rows that do not start on 16 bytes are copied, as rows of any other stride are:
the projections and the greedy head give what they give for the copy."""

from __future__ import annotations

import pytest
import torch

from leanstack_amd import _lib, kernels
from leanstack_amd.layout import PackedWeight
from tests.helpers import seeded_normal

pytestmark = pytest.mark.gpu


def _shifted(t, by):
    """The values of `t`, contiguous, `by` elements past an aligned address."""
    room = torch.full((t.numel() + 16,), 7.0, device=t.device, dtype=t.dtype)
    out = room[by:by + t.numel()].view_as(t)
    out.copy_(t)
    assert out.is_contiguous() and out.data_ptr() % 16
    return out


@pytest.mark.parametrize("by", [1, 4])
@pytest.mark.parametrize("m", [1, 5, 16, 40, 200])
def test_projections_of_misaligned_rows(gpu, m, by):
    n, k = 512, 1024
    x, res = seeded_normal((m, k), 1.0, 1).to(gpu), seeded_normal((m, n), 1.0, 2).to(gpu)
    w = seeded_normal((n, k), 0.02, 3).to(gpu)
    plain, gate_up = PackedWeight.from_rowmajor(w), PackedWeight.from_rowmajor(w, _lib.LAYOUT_MFMA16X32_GATEUP)
    for weight, kw in ((plain, {}), (gate_up, {"epilogue": _lib.EPI_SILU_MUL})):
        assert torch.equal(kernels.linear(_shifted(x, by), weight, **kw), kernels.linear(x, weight, **kw))
    kw = {"epilogue": _lib.EPI_RESIDUAL_ADD}
    expect = kernels.linear(x, plain, residual=res, **kw)
    moved = _shifted(res, by)
    assert torch.equal(kernels.linear(_shifted(x, by), plain, residual=moved, **kw), expect) and torch.equal(moved, res)


@pytest.mark.parametrize("m", [1, 5])
def test_fused_norms_and_the_head_of_misaligned_rows(gpu, m):
    k = 2560
    x, norm = seeded_normal((m, k), 1.0, 1).to(gpu), (1 + seeded_normal((k,), 0.1, 2)).to(gpu)
    weight = PackedWeight.from_rowmajor(seeded_normal((512, k), 0.02, 3).to(gpu))
    moved = _shifted(x, 3)
    assert torch.equal(kernels.rmsnorm_linear(moved, norm, 1e-6, weight), kernels.rmsnorm_linear(x, norm, 1e-6, weight))
    assert torch.equal(kernels.lm_head_argmax(moved, weight), kernels.lm_head_argmax(x, weight))
