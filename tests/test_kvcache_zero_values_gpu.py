"""Attention over long stretches of a quantised cache whose values are zero.

A group of zeros has scale 0, so the weights of such keys say nothing about the
products they go into, and the running maximum that they are taken against is kept
by their sum alone. Many of them in one chunk, then keys that score far lower or
that a query does not see, then ordinary keys.

Outputs are compared with 64-bit attention within eps/2 |o| for the output's
rounding, 2^-11 sum_j w_j |v_j| for the fp16 rounding of each weight times its
value's scale, and 2^-12 of it for the scores (fp32 sums of at most 128 products of
size 1, off by 2^-15), the exponential's 2^-22 and the normaliser: sums of up to
12288 equal powers of two are exact in fp32, and the 640 others add 640 2^-24.
"""

import numpy as np
import pytest
import torch

import _kv_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
# bits, D, group, heads: enough heads that at most 8 chunks of 16384 keys cover the cache
LAYOUTS = [(8, 64, 64, 24), (8, 128, 128, 24), (8, 128, 64, 24), (4, 64, 64, 80)]
L, ZEROS = 131072, 12288  # of the first chunk: 384 a lane


def _cache(bits, D, group, heads):
    from csaq._lib import lib
    from csaq.kvcache import QuantizedKVCache
    c = QuantizedKVCache(1, heads, L, D, bits=bits, group_size=group, device=DEV)
    assert lib().csaq_kvq_attention_launches(c._ref, 1, heads, D) == 1  # chunks meet in a cluster of at most 8
    return c


def _place(c, name, start, x):
    """Rows x (n, D) into positions start .. of every head; the fp64 values they stand for."""
    codes, words = ref.quantise(x.numpy(), c.bits, c.group_size)
    packed = ref.pack(codes, c.bits)
    getattr(c, name + "_codes")[:, :, start:start + len(x)] = torch.from_numpy(packed).to(DEV)
    getattr(c, name + "_params")[:, :, start:start + len(x)] = torch.from_numpy(words.view(np.int32)).to(DEV)
    return torch.from_numpy(ref.values(packed, words, c.bits, c.group_size))


@pytest.mark.parametrize("bits,D,group,heads", LAYOUTS)
@pytest.mark.parametrize("drop", [28.0, 75.0, 100.0, 300.0])
@pytest.mark.parametrize("S", [1, 3])
def test_lower_scores_after_zero_values(bits, D, group, heads, drop, S):
    """Every warp meets tiles whose scores all lie `drop` nats below those of the zeros."""
    dtype = torch.bfloat16
    c = _cache(bits, D, group, heads)
    g = torch.Generator().manual_seed(int(drop) + S)
    low = torch.zeros(128, D)
    low[:, 0] = -drop
    last = torch.randn(512, D, generator=g) * 0.25
    k = torch.cat([_place(c, "k", ZEROS, low), _place(c, "k", ZEROS + 128, last)])
    v = _place(c, "v", ZEROS, torch.randn(640, D, generator=g))
    q = (torch.randn(S, D, generator=g) * 0.25).to(dtype)
    q[:, 0] = 1.0
    pos0 = torch.tensor([ZEROS + 640 - S], dtype=torch.int32, device=DEV)
    out = c.attend(q.to(DEV).repeat(1, heads), pos0, scale=1.0).view(S, heads, D)
    assert torch.equal(out, out[:, :1].expand_as(out))  # all heads hold the same
    s = q.double() @ k.t()
    for r in range(S):
        n = 640 - S + 1 + r
        w = s[r, :n].exp()
        w = w / (w.sum() + ZEROS)  # the zeros score 0
        want, mag = w @ v[:n], w @ v[:n].abs()
        tol = torch.finfo(dtype).eps / 2 * want.abs() + (2.0 ** -11 + 2.0 ** -12) * mag
        got = out[r, 0].double().cpu()
        assert ((got - want).abs() <= tol).all(), (r, float((got - want).abs().max()), float(want.abs().max()))


@pytest.mark.parametrize("bits,D,group,heads", LAYOUTS)
@pytest.mark.parametrize("S", [2, 9])
def test_unseen_keys_after_zero_values(bits, D, group, heads, S):
    """A zeroed cache: the first token of the step sees none of the tile that the others see."""
    c = _cache(bits, D, group, heads)
    q = torch.randn(S, heads * D, generator=torch.Generator().manual_seed(S)).to(torch.bfloat16).to(DEV)
    out = c.attend(q, torch.tensor([ZEROS - 1], dtype=torch.int32, device=DEV))
    assert torch.equal(out, torch.zeros_like(out))
