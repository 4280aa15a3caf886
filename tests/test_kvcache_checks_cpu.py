"""What the quantised cache's calls check on the host, up to the launch (which a
stand-in takes the place of)."""

import pytest
import torch


def _long_cache(monkeypatch):
    """A cache on the host whose attention leaves partials, and the launches it would make."""
    from csaq.kvcache import QuantizedKVCache
    c = QuantizedKVCache(1, 1, 16384, 64, bits=8, device="cpu")
    launched = []
    monkeypatch.setattr(QuantizedKVCache, "_tokens", lambda self, t, what: (t.shape[0] // self.batch, t.shape[1], 1))
    monkeypatch.setattr(QuantizedKVCache, "_run", lambda self, fn, what, *args: launched.append(what))
    return c, torch.zeros(1, 64, dtype=torch.float16), torch.zeros(1, dtype=torch.int32), launched


def test_attend_wants_scratch_of_contiguous_floats(monkeypatch):
    """The kernel writes 32-bit partials one behind the other."""
    from csaq.kvcache import KVWorkspace
    c, q, pos0, launched = _long_cache(monkeypatch)
    n = c.workspace(1, 1).part.numel()
    assert n > 0
    for part in (torch.zeros(n, dtype=torch.float16), torch.zeros(n, dtype=torch.bfloat16),
                 torch.zeros(n, dtype=torch.uint8), torch.zeros(2 * n)[::2], torch.zeros(1).expand(n),
                 torch.zeros(4, n // 2).t()[:, :2], torch.zeros(n - 1)):
        with pytest.raises(ValueError, match="workspace"):
            c.attend(q, pos0, workspace=KVWorkspace(part))
    assert not launched
    for part in (torch.zeros(n), torch.zeros(n + 5), torch.zeros(2, n)):
        c.attend(q, pos0, workspace=KVWorkspace(part))
    assert launched == ["kvq_attention"] * 3


def test_a_cache_on_the_host_cannot_be_read():
    from csaq.kvcache import QuantizedKVCache
    c = QuantizedKVCache(1, 1, 32, 64, bits=8, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA device"):
        c.read(0, 4, dtype=torch.float16)


def test_buffers_without_a_sequence_are_refused():
    from csaq.kvcache import QuantizedKVCache
    z = lambda *s, t: torch.zeros(*s, dtype=t)  # noqa: E731
    for B, H, L in ((0, 2, 16), (2, 0, 16), (2, 2, 0)):
        with pytest.raises(ValueError):
            QuantizedKVCache.from_buffers(z(B, H, L, 64, t=torch.uint8), z(B, H, L, 1, t=torch.int32),
                                          z(B, H, L, 64, t=torch.uint8), z(B, H, L, 1, t=torch.int32), bits=8)
