"""Refusals of filtered sampling on the host, and its reference against hand-made cases."""

import ctypes

import numpy as np
import pytest
import torch

import _sample_ref as ref

P = ctypes.c_void_p(256)


def test_c_refusals():
    from csaq._lib import CsaqSampleParams, lib
    f = lib().csaq_sample_filtered
    s = ctypes.byref(CsaqSampleParams(None, None, None, None, 1.0, 0, 1.0, 0.0))
    for args in ((None, 1, 0, 8, 8, 1, s, P, P, 0), (P, 1, 0, 8, 8, 1, None, P, P, 0), (P, 1, 0, 8, 8, 1, s, None, P, 0),
                 (P, 1, 0, 8, 8, 1, s, P, None, 0), (P, 0, 0, 8, 8, 1, s, P, P, 0), (P, 1, 0, 8, 0, 1, s, P, P, 0),
                 (P, 1, 0, 7, 8, 1, s, P, P, 0), (P, 1, 0, 8, 8, -1, s, P, P, 0), (P, 1, 0, 8, 8, 1, s, P, P, 3),
                 (P, 2, -8, 8, 8, 1, s, P, P, 0)):
        assert f(*args, None) == -1, args
    assert f(P, 1, 0, 8, 8, 0, s, P, P, 0, None) == 0  # no rows
    for V, dtype in ((400_000, 0), (700_000, 1), (1 << 31, 2)):  # rows that no cluster holds
        assert f(P, 1, 0, V, V, 1, s, P, P, dtype, None) == -5


def test_struct_layout():
    from csaq._lib import CsaqSampleParams as C
    assert ctypes.sizeof(C) == 48 and C.temperature_all.offset == 32 and C.min_p_all.offset == 44


def test_python_refusals():
    from csaq.sampling import sample_params, sample_tokens
    dev = torch.device("cpu")
    for kw in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_k=-1), dict(top_k=2.5),
               dict(top_k=1 << 31), dict(top_p=0.0), dict(top_p=1.5), dict(min_p=-0.1), dict(min_p=1.1),
               dict(temperature=torch.ones(3)), dict(top_k=torch.ones(2)), dict(top_p=torch.ones(2, dtype=torch.float64)),
               dict(min_p=torch.ones(4)[::2])):
        with pytest.raises(ValueError):
            sample_params(2, dev, **kw)
    p = sample_params(2, dev, temperature=0.5, top_k=torch.tensor([1, 2], dtype=torch.int32), top_p=0.9)
    assert p.temperature is None and p.temperature_all == 0.5 and p.top_k is not None
    with pytest.raises(RuntimeError, match="CUDA"):
        sample_tokens(torch.zeros(1, 4), torch.zeros(1))


def test_reference_by_hand():
    x = np.log(np.array([0.1, 0.4, 0.2, 0.4, 0.3]))
    pick = lambda u, **kw: ref.sample(x, u, **kw)[0]  # noqa: E731
    kept = lambda **kw: ref.sample(x, 0.0, **kw)[1].tolist()  # noqa: E731
    assert [pick(u) for u in (0.0, 0.06, 0.08, 0.36, 0.51, 0.78, 0.8)] == [0, 0, 1, 2, 3, 3, 4]
    assert kept(top_k=1) == [1] and kept(top_k=2) == [1, 3] and kept(top_k=3) == [1, 3, 4]
    assert kept(top_p=0.1) == [1] and kept(top_p=0.3) == [1, 3] and kept(top_p=0.6) == [1, 3, 4]
    assert kept(min_p=0.6) == [1, 3, 4] and kept(min_p=1.0) == [1, 3]
    assert kept(top_k=3, top_p=0.5) == [1, 3]  # of 1.1, preceding 0, 0.36, 0.73
    assert ref.sample([np.nan, -np.inf], 0.5)[0] == -1
    assert ref.sample([np.nan, 1.0, np.inf, 2.0, np.inf], 0.6)[0] == 4
