"""Filtered sampling at the ends of the logits' range: temperatures so high that the
lowest logit with weight lies below what the type holds."""

import numpy as np
import pytest
import torch

import _sample_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("temperature", [1000.0, 2000.0, 1e6, 1e30])
@pytest.mark.parametrize("top_p", [1.0, 0.7])
def test_hot_rows_with_banned_tokens(dtype, temperature, top_p):
    """The lowest logit with weight lies below what fp16 holds, and top-k exceeds the
    tokens that are not banned: -inf must not count as one of them."""
    from csaq.sampling import sample_tokens
    rows, V, k = 8, 5003, 3000
    g = torch.Generator().manual_seed(int(np.log10(temperature)))
    x = torch.randn(rows, V, generator=g) * 3
    x[:, torch.randperm(V, generator=g)[:2500]] = float("-inf")
    x = x.to(dtype)
    u = torch.linspace(0.0, 1.0 - 2.0 ** -24, rows)
    out = torch.full((rows,), -7, dtype=torch.int64, device=DEV)
    sample_tokens(x.to(DEV), u.to(DEV), temperature=temperature, top_k=k, top_p=top_p, out=out)
    for r in range(rows):
        want, kept = ref.sample(x[r].double().numpy(), float(u[r]), temperature=temperature, top_k=k, top_p=top_p)
        assert int(out[r]) == want, (r, want, int(out[r]), len(kept))
