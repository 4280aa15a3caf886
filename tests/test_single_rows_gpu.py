"""Calls of one row or one sequence, whose strides say nothing: torch calls such views
contiguous whatever the stride of the axis of size one is."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _row(n, ld, dtype, seed):
    """(1, n) values as the first row of a matrix ld wide, and the same packed."""
    x = torch.randn(2, ld, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)
    return x[:1, :n], x[:1, :n].clone().view(-1).view(1, n)


@pytest.mark.parametrize("ld", [257, 260])
def test_one_token_in_rows_of_any_stride(ld):
    from csaq.kvcache import QuantizedKVCache
    new = lambda: QuantizedKVCache(1, 2, 32, 128, bits=8, device=DEV)  # noqa: E731
    a, b = new(), new()
    at = torch.tensor([9, 3, 9, 3], dtype=torch.int32, device=DEV)
    tables = [torch.rand(32, 128, device=DEV) for _ in range(2)]
    (k, k0), (v, v0), (q, q0) = (_row(256, ld, torch.bfloat16, s) for s in (1, 2, 3))
    assert k.stride(0) == ld and k0.stride(0) == 256
    pos = at[::2][:1]  # one value, two elements from a next one
    assert pos.stride(0) == 2
    ra = a.write(k, v, pos, *tables, q=q)
    rb = b.write(k0, v0, at[:1], *tables, q=q0)
    assert torch.equal(ra, rb) and all(torch.equal(s, t) for s, t in zip(a.buffers(), b.buffers()))
    want = b.attend(q0, at[:1])
    assert torch.equal(a.attend(q, pos), want)
    buf = torch.zeros(1, ld, dtype=torch.bfloat16, device=DEV)
    assert torch.equal(a.attend(q, pos, out=buf[:, :256]), want) and not buf[:, 256:].any()
    # strides shorter than the row
    assert torch.equal(a.attend(q0.as_strided((1, 256), (1, 1)), pos), want)
    out = torch.zeros(256, dtype=torch.bfloat16, device=DEV).as_strided((1, 256), (1, 1))
    assert torch.equal(a.attend(q, pos, out=out), want)
    c = new()
    c.write(k0.as_strided((1, 256), (0, 1)), v0.as_strided((1, 256), (8, 1)), pos, *tables)
    assert all(torch.equal(s, t) for s, t in zip(c.buffers(), b.buffers()))


def test_one_row_of_logits():
    from csaq.sampling import sample_tokens
    x = torch.randn(501, 1, generator=torch.Generator().manual_seed(1)).to(DEV)
    u = torch.rand(3, device=DEV)
    settings = torch.tensor([0.5, 2.0], device=DEV)[::2]  # one value at a stride of two
    want = sample_tokens(x.view(1, 501).clone(), u[:1], temperature=0.5)
    assert x.t().stride() == (1, 1)
    assert torch.equal(sample_tokens(x.t(), u[:1], temperature=0.5), want)
    assert torch.equal(sample_tokens(x.t(), u[:1], temperature=settings), want)
    assert sample_tokens(torch.zeros(3, 2, device=DEV)[:, :1], u).tolist() == [0, 0, 0]  # a vocabulary of one
