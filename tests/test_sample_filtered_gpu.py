"""Filtered sampling on the GPU against the 64-bit reference (tests/_sample_ref.py).

Tokens are compared for equality. Weights and sums of both sides are fp64 with
relative errors near 1e-14, so a row could differ only where a border of the
cumulative mass lies within about 1e-13 of a fixed fp32 random number, or a
filter's bound within as much of a weight; the inputs that put numbers on borders
do so where both sides compute them exactly.
"""

import numpy as np
import pytest
import torch

import _sample_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _logits(rows, V, dtype, seed, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, V, generator=g) * spread
    x.scatter_add_(1, torch.randint(0, V, (rows, 8), generator=g), 5 + 3 * torch.randn(rows, 8, generator=g))
    return x.to(dtype), torch.rand(rows, generator=g)


def _check(x, u, got, **kw):
    xd, ud = x.double().cpu().numpy(), u.cpu().numpy()
    for r in range(x.shape[0]):
        one = {k: (v[r].item() if isinstance(v, torch.Tensor) else v) for k, v in kw.items()}
        want, kept = ref.sample(xd[r], ud[r], **one)
        assert int(got[r]) == want, (r, one, float(ud[r]), want, int(got[r]), len(kept))


SETTINGS = [dict(), dict(temperature=0.6), dict(top_k=1), dict(top_k=7, temperature=1.7), dict(top_k=1000),
            dict(top_p=0.9), dict(top_p=0.3, temperature=0.8), dict(top_p=0.999), dict(min_p=0.05), dict(min_p=1.0),
            dict(top_k=50, top_p=0.95, min_p=0.02, temperature=0.8), dict(top_k=3, top_p=0.5, temperature=5.0),
            dict(top_k=20000, top_p=0.97, temperature=2.0), dict(temperature=0.0), dict(temperature=1e-3, top_p=0.9),
            dict(temperature=100.0, top_k=300, top_p=0.7), dict(top_p=1e-9), dict(top_k=1024, top_p=0.6),
            dict(top_k=1025, min_p=0.001), dict(temperature=50.0, top_p=0.5), dict(temperature=1e-4, top_k=200),
            dict(temperature=0.02, top_p=0.9999999), dict(temperature=1e31, top_k=9), dict(top_k=100, min_p=0.3)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("rows,V", [(1, 128256), (12, 5003), (40, 257)])
def test_matches_reference(dtype, kw, rows, V):
    from csaq.sampling import sample_tokens
    x, u = _logits(rows, V, dtype, seed=V + rows)
    _check(x, u, sample_tokens(x.to(DEV), u.to(DEV), **kw), **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 8, 15, 33, 511, 513, 4097])
def test_small_and_odd_vocabularies(dtype, V):
    from csaq.sampling import sample_tokens
    x, u = _logits(9, V, dtype, seed=V)
    for kw in (dict(), dict(top_k=2), dict(top_p=0.5), dict(top_k=V), dict(top_k=V + 1, top_p=0.8, min_p=0.01)):
        _check(x, u, sample_tokens(x.to(DEV), u.to(DEV), **kw), **kw)


@pytest.mark.parametrize("rows,V,dtype", [(3, 680000, torch.bfloat16), (3, 340000, torch.float32), (160, 151936,
                                          torch.bfloat16), (300, 32003, torch.float16), (200, 70000, torch.float32)])
def test_large(rows, V, dtype):
    """The widest rows, and more rows than SMs: every cluster size."""
    from csaq.sampling import sample_tokens
    x, u = _logits(rows, V, dtype, seed=3)
    some = list(range(0, rows, max(1, rows // 12)))
    for kw in (dict(top_p=0.9), dict(top_k=40, temperature=0.7)):
        got = sample_tokens(x.to(DEV), u.to(DEV), **kw).cpu()
        _check(x[some], u[some], got[some], **kw)


def test_per_row_settings():
    from csaq.sampling import sample_tokens
    rows, V = 64, 3001
    x, u = _logits(rows, V, torch.bfloat16, seed=5)
    g = torch.Generator().manual_seed(6)
    pick = lambda vals, t: torch.tensor(vals, dtype=t)[torch.randint(0, len(vals), (rows,), generator=g)]  # noqa: E731
    kw = dict(temperature=pick([0.0, 0.5, 1.0, 2.0], torch.float32), top_k=pick([0, 1, 30, 5000], torch.int32),
              top_p=pick([1.0, 0.9, 0.4], torch.float32), min_p=pick([0.0, 0.03, 0.3], torch.float32))
    got = sample_tokens(x.to(DEV), u.to(DEV), **{k: v.to(DEV) for k, v in kw.items()})
    _check(x, u, got, **kw)
    # a row's token does not depend on the rows beside it
    for r in (0, 17, 63):
        one = {k: v[r:r + 1].to(DEV) for k, v in kw.items()}
        assert int(sample_tokens(x[r:r + 1].to(DEV), u[r:r + 1].to(DEV), **one)) == int(got[r])


def test_settings_out_of_range_on_the_device():
    """Device arrays are not looked at by the host: what lies outside is read as off
    (top_k < 0, top_p > 1 or NaN, min_p < 0 or NaN), as the first rank (temperature
    below 0 or NaN, top_p <= 0) or as its bound (min_p > 1)."""
    from csaq.sampling import sample_tokens
    nan = float("nan")
    x, u = _logits(9, 999, torch.float32, seed=8)
    t = torch.tensor([1.0, 1, 1, 1, 1, -1, nan, 1, 1])
    k = torch.tensor([-5, 0, 0, 0, 0, 0, 0, 0, 0], dtype=torch.int32)
    p = torch.tensor([1.0, 7, nan, 1, 1, 1, 1, -2, 1])
    m = torch.tensor([0.0, 0, 0, -1, nan, 0, 0, 0, 9])
    got = sample_tokens(x.to(DEV), u.to(DEV), temperature=t.to(DEV), top_k=k.to(DEV), top_p=p.to(DEV), min_p=m.to(DEV))
    for r in range(9):
        kw = dict(temperature=0.0) if r in (5, 6) else dict(top_p=0.0) if r == 7 else dict(min_p=1.0) if r == 8 else {}
        assert int(got[r]) == ref.sample(x[r].double().numpy(), float(u[r]), **kw)[0], r


@pytest.mark.parametrize("dtype", DTYPES)
def test_special_logits(dtype):
    """Banned tokens, NaN, infinities, signed zeros, the type's lowest value, rows of one value."""
    from csaq.sampling import sample_tokens
    V, inf, nan = 1000, float("inf"), float("nan")
    g = torch.Generator().manual_seed(1)
    x = torch.randn(12, V, generator=g).to(dtype)
    x[0, ::2] = -inf
    x[1] = -inf
    x[2] = nan
    x[3, 5:] = nan
    x[4, [17, 400, 999]] = inf
    x[5] = torch.finfo(dtype).min
    x[6] = torch.finfo(dtype).min
    x[6, 77] = -inf
    x[7] = -0.0
    x[7, ::3] = 0.0
    x[8] = -inf
    x[8, 999] = -3.0
    x[9, :] = torch.finfo(dtype).max
    x[10] = nan
    x[10, 3] = -inf
    x[11, 500] = torch.finfo(dtype).max
    for kw in (dict(), dict(top_k=5), dict(top_p=0.5), dict(min_p=0.9), dict(temperature=0.0),
               dict(top_k=400, top_p=0.9, temperature=0.5)):
        for seed in range(3):
            u = torch.rand(12, generator=torch.Generator().manual_seed(seed))
            _check(x, u, sample_tokens(x.to(DEV), u.to(DEV), **kw), **kw)


def test_ties_go_to_the_lowest_index():
    from csaq.sampling import sample_tokens
    V = 4096
    x = torch.zeros(1, V)
    x[0, 100::7] = 1.0                      # 571 equal leaders
    lead = list(range(100, V, 7))
    u = torch.tensor([0.999999])
    for k in (1, 2, 300, 571):              # the first k leaders, the last of them drawn
        assert int(sample_tokens(x.to(DEV), u.to(DEV), top_k=k)) == lead[k - 1]
    _check(x, u, sample_tokens(x.to(DEV), u.to(DEV), top_k=573), top_k=573)
    flat = torch.full((1, 1024), 2.5)
    for p, last in ((0.5, 512), (0.25, 256), (1 / 1024, 1), (0.4999, 511)):  # i/1024 <= p, exactly
        assert int(sample_tokens(flat.to(DEV), u.to(DEV), top_p=p)) == last


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1 << 16, 100003])
def test_flat_rows_hit_every_border_right(dtype, V):
    """Equal logits: the token of u is floor(u V), exactly, wherever u lies."""
    from csaq.sampling import sample_tokens
    rows = 2000
    g = torch.Generator().manual_seed(2)
    u = torch.rand(rows, generator=g)
    u[:500] = torch.randint(0, 1 << 16, (500,), generator=g) / float(1 << 16)  # on borders of the power of two
    u[0], u[1] = 0.0, 1 - 2.0 ** -24
    row = torch.full((1, V), -1.75, dtype=dtype, device=DEV)
    got = sample_tokens(row.expand(rows, V), u.to(DEV)).cpu()
    assert torch.equal(got, torch.floor(u.double() * V).long())


@pytest.mark.parametrize("dtype", DTYPES)
def test_crowded_cuts(dtype):
    """More equal or nearly equal tokens at a cut than a list holds, in one and in many
    CTAs, and cuts on either side of the crowd."""
    from csaq.sampling import sample_tokens
    V = 30000
    g = torch.Generator().manual_seed(9)
    x = torch.randn(6, V, generator=g) * 0.01
    x[0] = 0.0                                    # all equal
    x[1, ::3] = 1.0                               # 10000 equal leaders
    x[2, 100:900] = 4.0                           # 800 leaders in one CTA, a dense crowd below
    x[3] = torch.arange(V) * 1e-5                 # rising, finely
    x[4, :2500] = 0.5
    x[4, 2500:] = torch.randn(V - 2500, generator=g) - 3
    x = x.to(dtype)
    for seed, kw in enumerate((dict(top_k=500), dict(top_k=1000), dict(top_k=900), dict(top_p=0.5), dict(top_p=0.2),
                               dict(top_p=0.95), dict(top_k=20000, top_p=0.4), dict(top_k=1000, top_p=0.999),
                               dict(top_k=801, top_p=0.9999))):
        u = torch.rand(6, generator=torch.Generator().manual_seed(seed))
        _check(x, u, sample_tokens(x.to(DEV), u.to(DEV), **kw), **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,spread,temperature", [(20011, 2.0, 1.0), (20011, 0.3, 0.5), (3001, 4.0, 2.0), (151936, 3.0, 1.0)])
def test_the_last_kept_rank(dtype, V, spread, temperature):
    """Rows sorted downwards, where the largest random number draws the last kept token:
    a cut wrong by one token, or by one of its equals, shows. Cuts fall among large, small,
    negative and subnormal logits and on both sides of zero. (A border lies within the
    weights' 2^-32 of a bound with a chance of about 2^-32 V p per row.)"""
    from csaq.sampling import sample_tokens
    rows = 24
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(rows, V, generator=g) * spread).to(dtype)
    x[rows // 2:] *= torch.logspace(0, -5, rows - rows // 2).to(dtype)[:, None]
    x = x.sort(dim=1, descending=True).values
    w = ((x.double() - x[:, :1].double()) / temperature).exp()
    above = (w * (x > 0)).sum(1) / w.sum(1)  # the cut at zero
    p = torch.linspace(0.02, 0.999, rows).double()
    p[::3] = above[::3].clamp(0.01, 0.999)
    u = torch.full((rows,), 1.0 - 2.0 ** -24)
    p = p.float()
    kw = dict(top_p=p, temperature=temperature)
    _check(x, u, sample_tokens(x.to(DEV), u.to(DEV), top_p=p.to(DEV), temperature=temperature), **kw)


def test_random_numbers_outside():
    """Below 0 and NaN count as 0, 1 and more as the largest number below 1."""
    from csaq.sampling import sample_tokens
    x = torch.zeros(4, 10, device=DEV)
    u = torch.tensor([-3.0, float("nan"), 1.0, float("inf")], device=DEV)
    assert sample_tokens(x, u).tolist() == [0, 0, 9, 9]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ld,off", [(1000, 0), (1003, 0), (1008, 8), (1001, 3)])
def test_row_strides_and_alignment(dtype, ld, off):
    from csaq.sampling import sample_tokens
    x, u = _logits(6, ld, dtype, seed=ld)
    y = x.to(DEV)[:, off:off + 901]
    for kw in (dict(), dict(top_k=20, top_p=0.9)):
        _check(x[:, off:off + 901], u, sample_tokens(y, u.to(DEV), **kw), **kw)
    t = x.to(DEV).t().contiguous().t()  # column-major: copied
    _check(x, u, sample_tokens(t, u.to(DEV), top_k=9), top_k=9)


@pytest.mark.parametrize("part", [128, 401])
def test_vocabulary_slices(part):
    """Tensor-parallel layout: slices of the vocabulary, rows * part apart."""
    import ctypes
    from csaq._lib import check, lib
    from csaq.sampling import sample_params
    rows, W = 5, 4
    x, u = _logits(rows, W * part, torch.bfloat16, seed=part)
    parts = x.view(rows, W, part).permute(1, 0, 2).contiguous().to(DEV)
    out = torch.empty(rows, dtype=torch.int64, device=DEV)
    kw = dict(temperature=0.9, top_k=60, top_p=0.9, min_p=0.01)
    p = sample_params(rows, out.device, **kw)
    check(lib().csaq_sample_filtered(parts.data_ptr(), W, rows * part, part, part, rows, ctypes.byref(p),
                                     u.to(DEV).data_ptr(), out.data_ptr(), 2,
                                     torch.cuda.current_stream().cuda_stream), "sample_filtered")
    _check(x, u, out, **kw)


def test_captured_and_on_another_stream():
    from csaq.sampling import sample_tokens
    x, u = _logits(8, 20000, torch.bfloat16, seed=4)
    xs, us = x.to(DEV), torch.zeros(8, device=DEV)
    out = torch.empty(8, dtype=torch.int64, device=DEV)
    sample_tokens(xs, us, top_k=50, top_p=0.9, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sample_tokens(xs, us, top_k=50, top_p=0.9, out=out)
    side = torch.cuda.Stream()
    for seed in range(4):
        x, u = _logits(8, 20000, torch.bfloat16, seed=100 + seed)
        xs.copy_(x)
        us.copy_(u)
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = sample_tokens(xs, us, top_k=50, top_p=0.9)
        torch.cuda.synchronize()
        assert torch.equal(out, other)
        _check(x, u, out, top_k=50, top_p=0.9)


def test_refusals_on_the_device():
    from csaq.sampling import sample_tokens
    x, u = torch.zeros(2, 8, device=DEV), torch.zeros(2, device=DEV)
    for args, kw, exc in (((x[0], u), {}, ValueError), ((x, u[:1]), {}, ValueError), ((x, u.double()), {}, ValueError),
                          ((x, u.cpu()), {}, ValueError), ((x.double(), u), {}, TypeError), ((x, u), dict(top_p=0.0), ValueError),
                          ((x, u), dict(out=u), ValueError), ((x, u), dict(top_k=u), ValueError),
                          ((x, u), dict(temperature=torch.ones(2)), ValueError), ((x[:, :0], u), {}, ValueError)):
        with pytest.raises(exc):
            sample_tokens(*args, **kw)
    assert sample_tokens(x[:0], u[:0]).shape == (0,)
    with pytest.raises(RuntimeError, match="not supported"):
        sample_tokens(torch.zeros(1, 800000, dtype=torch.bfloat16, device=DEV), u[:1])
