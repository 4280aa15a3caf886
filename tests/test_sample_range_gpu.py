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


@pytest.mark.parametrize("temperature", [1.0, 1e29, 1e30])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=40), dict(top_k=1500, top_p=0.9), dict(top_p=0.9), dict(min_p=0.1)],
                         ids=str)
def test_rows_of_nearly_the_lowest_value(temperature, kw):
    """fp32 logits within a hundredth of the range's lower end, banned ones at its end: what has no
    weight beside the largest has none here either."""
    from csaq.sampling import sample_tokens
    lowest = torch.finfo(torch.float32).min
    V = 2003
    x = torch.full((4, V), lowest)
    x[0, 1700] = -3.401e38                            # the rest lies 1.8e35 below
    x[1, ::2] = torch.tensor(lowest) * (1 - 2.0 ** -23)  # two steps of fp32 above, 4e31
    x[2, :] = torch.linspace(-3.4028e38, -3.395e38, V)
    x[3, 5] = -3.3e38
    u = torch.tensor([0.3, 0.6, 0.999, 0.0])
    out = torch.full((4,), -7, dtype=torch.int64, device=DEV)
    sample_tokens(x.to(DEV), u.to(DEV), temperature=temperature, out=out, **kw)
    for r in range(4):
        want, kept = ref.sample(x[r].double().numpy(), float(u[r]), temperature=temperature, **kw)
        assert int(out[r]) == want, (r, want, int(out[r]), len(kept))
