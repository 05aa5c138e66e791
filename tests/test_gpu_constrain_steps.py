"""Constrained logits step by step: every value's bits and the token against the
documented fp32 steps, where they reach the ends of the logits' type."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from leanstack_amd import kernels

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _steps(logits, history, prompt, rho, alpha_f, alpha_p, bias, allowed):
    """One row in numpy's float32, one rounding per step, rounded once to the logits' type."""
    z = logits.float().numpy().copy()
    f32 = np.float32
    with np.errstate(over="ignore", invalid="ignore"):
        for v in np.unique(history):
            z[v] = z[v] / f32(rho) if z[v] > 0 else z[v] * f32(rho)
        tokens, count = np.unique(history[prompt:], return_counts=True)
        for v, c in zip(tokens, count):
            z[v] = f32(z[v] - f32(f32(alpha_f) * f32(c))) - f32(alpha_p)
        for v, b in bias.items():
            z[v] = z[v] + f32(b)
    z[~allowed] = -np.inf
    return torch.from_numpy(z).to(logits.dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value", ["lowest", "highest", "smallest", "subnormal", "half"])
@pytest.mark.parametrize("v", [37, 5000])
def test_values_at_the_ends_of_the_type(gpu, dtype, value, v):
    info = torch.finfo(dtype)
    start = {"lowest": info.min, "highest": info.max, "smallest": -info.tiny, "subnormal": info.tiny / 4,
             "half": info.min / 2}[value]
    gen = torch.Generator().manual_seed(v)
    logits = torch.full((4, v), start, dtype=dtype)
    logits[1, ::3] = -start
    logits[2, v - 1] = start / 2
    history = torch.randint(0, v, (4, 40), generator=gen, dtype=torch.int32)
    rho, alpha_f, alpha_p = (torch.tensor(x) for x in ([1.5, 0.75, 2.0, 1.0], [0.5, info.max / 8, -0.25, 0.0], [1.0, 0.5, info.max / 4, 2.0]))
    prompt = torch.tensor([7, 0, 40, 13], dtype=torch.int32)
    ids = torch.stack([torch.randperm(v, generator=gen)[:9] for _ in range(4)]).int()
    values = torch.randn(4, 9, generator=gen) * torch.tensor([1.0, info.max / 2, info.tiny, 100.0])[:, None]
    words = torch.randint(-2**31, 2**31, (4, (v + 31) // 32), generator=gen, dtype=torch.int64).int()
    words[3] = -1
    at = torch.arange(v)
    allowed = (words[:, at // 32] >> (at % 32)) & 1 != 0
    got, tokens = kernels.constrain_logits(
        logits.to(DEV), history=history.to(DEV), prompt_lens=prompt.to(DEV), repetition=rho.to(DEV),
        frequency=alpha_f.to(DEV), presence=alpha_p.to(DEV), bias_ids=ids.to(DEV), bias_values=values.to(DEV),
        allowed=words.to(DEV))
    for r in range(4):
        expect = _steps(logits[r], history[r].numpy(), int(prompt[r]), float(rho[r]), float(alpha_f[r]), float(alpha_p[r]),
                        dict(zip(ids[r].tolist(), values[r].tolist())), allowed[r].numpy())
        assert not bool(expect.isnan().any())
        assert torch.equal(got[r].cpu().float().view(torch.int32), expect.float().view(torch.int32)), f"row {r}"
        best = int(np.argmax(expect.float().numpy()))
        assert int(tokens[r]) == (best if float(expect[best]) > -np.inf else -1), f"row {r}"
