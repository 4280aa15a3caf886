"""Filtered sampling where a rounded difference of logits would draw another token,
against 64 bits."""

import numpy as np
import pytest
import torch

import _sample_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"

# largest logit 17, the others `low`, whose difference needs more than the 24 bits of an
# fp32: 17 - low lies half an ulp, 2^-20, from the nearest
LOW = {torch.float16: 2.0 ** -10 * (1 + 2.0 ** -10), torch.bfloat16: 2.0 ** -14 * (1 + 2.0 ** -6),
       torch.float32: 2.0 ** -10 * (1 + 2.0 ** -10)}


@pytest.mark.parametrize("dtype", list(LOW))
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=120000), dict(top_p=0.9999999), dict(min_p=1e-9)], ids=str)
def test_differences_of_logits_are_exact(dtype, sign, kw):
    """N tokens of weight e^(low - 17) = 4e-8, each a border of the cumulative mass, under
    one of weight 1. A difference off by 2^-20 moves the border of token 100000 by
    100000 * 4e-8 * 2^-20 = 3.9e-9; weights good to 2^-32 by 1e-12. The numbers are the
    two fp32 neighbours of a border, 2^-32 or 2^-31 apart, each at least a tenth of that from it."""
    from csaq.sampling import sample_tokens
    N = 128000
    x = torch.full((N + 1,), sign * LOW[dtype], dtype=torch.float64)
    x[N] = 17.0
    row = x.to(dtype)
    assert torch.equal(row.double(), x)
    w = np.exp(sign * LOW[dtype] - 17.0)
    kept = min(N, kw.get("top_k", N + 1) - 1)  # the first `kept` of the equals beside the largest
    if "top_p" in kw:  # of them while the mass before is at most top_p of the whole
        kept = int((float(np.float32(kw["top_p"])) * (1.0 + N * w) - 1.0) / w) + 1
    total = 1.0 + kept * w
    us, want = [], []
    for k in range(70000, 119000, 331):
        border = k * w / total  # tokens 0 .. k - 1 end here
        below = np.float32(border)
        below = below if float(below) < border else np.nextafter(below, np.float32(0))
        above = np.nextafter(below, np.float32(1))
        if min(border - float(below), float(above) - border) < 0.1 * float(above - below):
            continue
        us += [below, above]
        want += [k - 1, k]
    us, want = us[:128], want[:128]
    u = torch.from_numpy(np.array(us, np.float32))
    got = sample_tokens(row.to(DEV).expand(len(us), N + 1), u.to(DEV), **kw).cpu()
    assert torch.equal(got, torch.tensor(want)), int((got != torch.tensor(want)).sum())
    r = len(us) // 2
    assert ref.sample(x.numpy(), us[r], **kw)[0] == want[r]


@pytest.mark.parametrize("dtype", list(LOW))
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_differences_in_a_sorted_list_are_exact(dtype, sign):
    """The same with the first 1000 ranks alone, which are sorted and cut in one place: a border at
    token 900, 4e-5, moves by 4e-11, ten steps of an fp32 there."""
    from csaq.sampling import sample_tokens
    N, top_k = 40000, 1000
    x = torch.full((N + 1,), sign * LOW[dtype] - 40.0, dtype=torch.float64)
    x[::100] = x[50::100] = sign * LOW[dtype]
    x[7::200] = x[57::200] = x[107::200] = sign * LOW[dtype]
    x[N] = 17.0
    row = x.to(dtype)
    low = torch.nonzero(x == sign * LOW[dtype]).view(-1)[:top_k - 1]
    assert torch.equal(row.double()[low], x[low]) and len(low) == top_k - 1
    w = np.exp(sign * LOW[dtype] - 17.0)
    us, want = [], []
    for k in range(500, 990):
        border = k * w / (1.0 + (top_k - 1) * w)
        below = np.float32(border)
        below = below if float(below) < border else np.nextafter(below, np.float32(0))
        above = np.nextafter(below, np.float32(1))
        if min(border - float(below), float(above) - border) >= 0.1 * float(above - below):
            us += [below, above]
            want += [int(low[k - 1]), int(low[k])]
    us, want = us[:256], want[:256]
    got = sample_tokens(row.to(DEV).expand(len(us), N + 1), torch.from_numpy(np.array(us, np.float32)).to(DEV),
                        top_k=top_k).cpu()
    assert torch.equal(got, torch.tensor(want)), int((got != torch.tensor(want)).sum())
