"""Refusals of the quantised KV cache, before anything reaches a GPU: the C entry
points' status codes on dummy pointers, and the Python class's exceptions."""

import ctypes

import pytest
import torch

OK, ARG, BITS, UNSUPPORTED = 0, -1, -2, -5
P = ctypes.c_void_p(256)


def _cache(**kw):
    from csaq._lib import CsaqKvqCache
    f = dict(k_codes=256, k_params=256, v_codes=256, v_params=256, Lmax=64, bits=8, group_size=128)
    f.update(kw)
    return ctypes.byref(CsaqKvqCache(*(f[n] for n, _ in CsaqKvqCache._fields_)))


BAD_CACHES = [(dict(k_codes=None), ARG), (dict(v_params=None), ARG), (dict(Lmax=0), ARG), (dict(bits=2), BITS),
              (dict(bits=16), BITS), (dict(Lmax=60), UNSUPPORTED), (dict(Lmax=1 << 31), UNSUPPORTED),
              (dict(group_size=32), UNSUPPORTED), (dict(group_size=0), UNSUPPORTED),
              (dict(k_params=260), UNSUPPORTED), (dict(v_codes=257), UNSUPPORTED)]


@pytest.mark.parametrize("bad,rc", BAD_CACHES)
def test_cache_descriptor_refused(bad, rc):
    from csaq._lib import lib
    L = lib()
    c = _cache(**bad)
    assert L.csaq_kvq_write(None, 0, P, 1024, P, 1024, P, 1, 1, 0, 8, 128, None, None, 0, None, c, 2, None) == rc
    assert L.csaq_kvq_read(c, 1, 8, 128, 0, 1, P, P, 2, None) == rc
    assert L.csaq_kvq_attention(P, 4096, c, P, 1, 1, 32, 8, 128, 0.1, P, P, 4096, 2, None) == rc
    assert L.csaq_kvq_read(None, 1, 8, 128, 0, 1, P, P, 2, None) == ARG


def test_write_refusals():
    from csaq._lib import lib
    f = lib().csaq_kvq_write

    def call(q=P, ldq=4096, k=P, ldk=1024, v=P, ldv=1024, pos0=P, B=1, S=1, Hq=32, Hkv=8, D=128, cos=P, sin=P, n=64,
             q_out=P, dtype=2):
        return f(q, ldq, k, ldk, v, ldv, pos0, B, S, Hq, Hkv, D, cos, sin, n, q_out, _cache(), dtype, None)

    for bad in (dict(k=None), dict(v=None), dict(pos0=None), dict(S=0), dict(q_out=None), dict(cos=None),
                dict(sin=None), dict(cos=None, sin=None), dict(n=0), dict(dtype=0), dict(dtype=9), dict(ldk=1016),
                dict(ldv=8), dict(ldq=4088), dict(B=0), dict(Hkv=0), dict(Hq=0)):
        assert call(**bad) == ARG, bad
    odd = ctypes.c_void_p(258)
    for bad in (dict(ldk=1028), dict(ldv=1027), dict(ldq=4097), dict(k=odd), dict(v=odd), dict(q=odd),
                dict(q_out=odd), dict(cos=odd), dict(D=96, ldk=1024), dict(B=1 << 20, S=1 << 20)):
        assert call(**bad) == UNSUPPORTED, bad


def test_read_refusals():
    from csaq._lib import lib
    f = lib().csaq_kvq_read
    for start, n in ((-1, 1), (0, -1), (0, 65), (64, 1), (65, 0), (1, 1 << 62)):
        assert f(_cache(), 1, 8, 128, start, n, P, P, 2, None) == ARG
    assert f(_cache(), 1, 8, 128, 0, 1, None, None, 2, None) == ARG
    assert f(_cache(), 1, 8, 128, 0, 1, P, P, 3, None) == ARG
    assert f(_cache(), 1, 8, 128, 0, 1, ctypes.c_void_p(264), P, 2, None) == UNSUPPORTED
    assert f(_cache(), 1, 8, 128, 64, 0, P, P, 2, None) == OK  # nothing to read


def test_attention_refusals():
    from csaq._lib import lib
    L = lib()

    def call(q=P, ldq=4096, pos0=P, B=1, S=1, Hq=32, Hkv=8, D=128, part=P, out=P, ldo=4096, dtype=2, Lmax=64):
        return L.csaq_kvq_attention(q, ldq, _cache(Lmax=Lmax), pos0, B, S, Hq, Hkv, D, 0.1, part, out, ldo, dtype, None)

    for bad in (dict(q=None), dict(pos0=None), dict(part=None, Lmax=1 << 20), dict(out=None), dict(S=0),
                dict(Hq=0), dict(Hq=33), dict(ldq=4095), dict(ldo=4095), dict(dtype=0)):
        assert call(**bad) == ARG, bad
    for bad in (dict(ldo=4097), dict(out=ctypes.c_void_p(258)), dict(part=ctypes.c_void_p(260)), dict(S=70000),
                dict(B=1 << 30), dict(ldq=4098), dict(q=ctypes.c_void_p(264))):
        assert call(**bad) == UNSUPPORTED, bad
    assert L.csaq_kvq_attention_workspace_floats(1, 1, 33, 8, 128, 64) == -1
    assert L.csaq_kvq_attention_workspace_floats(1, 0, 32, 8, 128, 64) == -1


def test_workspace_sizes():
    """None while a head's chunks fit a cluster, else one partial state per (chunk,
    query row): their number stays bounded and does not depend on the step's tokens."""
    from csaq._lib import lib
    f = lib().csaq_kvq_attention_workspace_floats
    assert f(1, 1, 32, 8, 128, 64) == 0 and f(128, 1, 32, 8, 128, 1 << 16) == 0
    long = f(1, 1, 32, 8, 128, 1 << 17)
    assert long > 0 and long % (8 * 4 * 130) == 0 and f(1, 5, 32, 8, 128, 1 << 17) == 5 * long
    for B, Hkv, Lmax in ((1, 8, 1 << 20), (64, 8, 1 << 15), (1, 1, 1 << 24), (2048, 16, 4096)):
        assert f(B, 1, Hkv, Hkv, 64, Lmax) // 66 <= 4 * 148


def test_struct_layout():
    from csaq._lib import CsaqKvqCache as C
    assert ctypes.sizeof(C) == 48 and C.Lmax.offset == 32 and C.bits.offset == 40 and C.group_size.offset == 44


def _buffers(B=2, H=4, L=32, D=128, bits=8, NG=1):
    z = lambda *s, t: torch.zeros(*s, dtype=t)  # noqa: E731
    return [z(B, H, L, D * bits // 8, t=torch.uint8), z(B, H, L, NG, t=torch.int32),
            z(B, H, L, D * bits // 8, t=torch.uint8), z(B, H, L, NG, t=torch.int32)]


def test_class_refusals():
    from csaq.kvcache import QuantizedKVCache, cache_positions
    assert [cache_positions(n) for n in (1, 16, 17)] == [16, 16, 32]
    ok = QuantizedKVCache.from_buffers(*_buffers(), bits=8)
    assert (ok.batch, ok.kv_heads, ok.max_len, ok.head_dim, ok.group_size) == (2, 4, 32, 128, 128)
    assert QuantizedKVCache.from_buffers(*_buffers(bits=4, NG=2), bits=4).group_size == 64
    for kw in (dict(bits=3), dict(head_dim=96), dict(group_size=32), dict(group_size=0), dict(max_len=0),
               dict(batch=0)):
        args = dict(batch=1, kv_heads=2, max_len=32, head_dim=128, bits=8, device="cpu")
        args.update(kw)
        with pytest.raises(ValueError):
            QuantizedKVCache(**args)
    b = _buffers()
    for i, wrong in ((0, b[0].to(torch.int8)), (1, b[1].float()), (2, b[2][:, :, :16]), (3, b[3].expand(2, 4, 32, 2)),
                     (0, b[0].transpose(1, 2)), (1, b[1][0])):
        bufs = list(b)
        bufs[i] = wrong
        with pytest.raises(ValueError):
            QuantizedKVCache.from_buffers(*bufs, bits=8)
    with pytest.raises(ValueError):
        QuantizedKVCache.from_buffers(*_buffers(L=24), bits=8)
    with pytest.raises(ValueError):
        QuantizedKVCache.from_buffers(*_buffers(), bits=2)
    # a cache on the host has no kernels
    k = torch.zeros(2, 512, dtype=torch.bfloat16)
    pos = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ok.write(k, k, pos)
    with pytest.raises(RuntimeError, match="CUDA"):
        ok.attend(k, pos)
    with pytest.raises(ValueError, match="positions"):
        ok.read(0, 33)
    with pytest.raises(ValueError, match="positions"):
        ok.read(5, 4)
    with pytest.raises(ValueError):
        ok.workspace(1, 6)
