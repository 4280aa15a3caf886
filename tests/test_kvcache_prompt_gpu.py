"""Prompts so large that a warp of the quantised write takes several heads in turn, more
of them than it holds in flight and shares that differ from warp to warp: codes, words
and queries bit for bit, and the other positions as they were."""

import numpy as np
import pytest
import torch

import _kv_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("Hq,Hkv,bits,D,group", [(14, 2, 8, 128, 128), (32, 8, 4, 128, 64), (39, 3, 4, 64, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_large_prompt_is_the_definition(Hq, Hkv, bits, D, group, dtype):
    from csaq.kvcache import QuantizedKVCache
    B, S, at = 2, 1500, (3, 41)
    g = torch.Generator().manual_seed(Hq)
    qkv = torch.randn(B * S, (Hq + 2 * Hkv) * D, generator=g).to(dtype)
    x = qkv.float().numpy().reshape(B, S, Hq + 2 * Hkv, D)
    f = torch.arange(1600).double()[:, None] * (1.0 / (10000.0 ** (torch.arange(0, D, 2).double() / D)))
    cos, sin = (torch.cat([t, t], -1).float().contiguous() for t in (f.cos(), f.sin()))
    c = QuantizedKVCache(B, Hkv, 1600, D, bits=bits, group_size=group, device=DEV)
    before = [t.random_(0, 200).cpu().numpy().copy() for t in c.buffers()]
    on = qkv.to(DEV)
    q = c.write(on[:, Hq * D:(Hq + Hkv) * D], on[:, (Hq + Hkv) * D:], torch.tensor(at, dtype=torch.int32, device=DEV),
                cos.to(DEV), sin.to(DEV), q=on[:, :Hq * D])
    p = np.array(at)[:, None] + np.arange(S)
    cs, sn = cos.numpy()[p][:, :, None], sin.numpy()[p][:, :, None]
    assert torch.equal(q.cpu().view(B, S, Hq, D), torch.from_numpy(ref.rotate(x[:, :, :Hq], cs, sn)).to(dtype))
    for i, y in ((0, ref.rotate(x[:, :, Hq:Hq + Hkv], cs, sn)), (2, x[:, :, Hq + Hkv:])):
        codes, words = ref.quantise(y, bits, group)
        want_c, want_w = before[i], before[i + 1]
        for b in range(B):
            want_c[b, :, at[b]:at[b] + S] = ref.pack(codes[b], bits).swapaxes(0, 1)
            want_w[b, :, at[b]:at[b] + S] = words[b].view(np.int32).swapaxes(0, 1)
        assert np.array_equal(c.buffers()[i].cpu().numpy(), want_c)
        assert np.array_equal(c.buffers()[i + 1].cpu().numpy(), want_w)
