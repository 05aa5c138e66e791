"""Attention over a shared prefix at its edges: batches that have nothing to attend."""

from __future__ import annotations

import pytest
import torch

from leanstack_amd import kernels
from tests import test_gpu_prefix_attention as attention_of

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
D = 128
SCALE = D ** -0.5


@pytest.mark.parametrize("b,t,n_q,n_kv", [(32, 1, 32, 8), (33, 1, 32, 8), (300, 1, 4, 1), (64, 1, 32, 8), (9, 40, 32, 8)])
def test_large_batches_without_any_row(gpu, b, t, n_q, n_kv):
    """No prefix and no room for own rows: zeros, however many requests there are."""
    q, pk, pv, k, v, _ = attention_of._request(b, t, n_q, n_kv, 0, 1)
    none = k[:, :, :0]
    for lens in (torch.zeros(b, dtype=torch.int32, device=DEV), torch.full((b,), 7, dtype=torch.int32, device=DEV)):
        out = torch.full((b, t, n_q * D), 9.0, device=DEV).bfloat16()
        assert kernels.shared_prefix_attention(q, pk, pv, none, v[:, :, :0], lens, SCALE, out=out) is out
        assert not bool(out.any())
