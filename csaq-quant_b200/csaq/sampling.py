"""csaq.sampling — tokens from logits and given random numbers.

The engine's sampler at temperature > 0 (csaq/inference.py:269-304) knows
temperature and top-p and draws its own numbers. ``sample_tokens`` is the
server's form: temperature, top-k, top-p and min-p, each one value or one per
row, and the caller's random numbers, so that a request's tokens do not depend
on what else was in its batch. ``DecodeRuntime.generate_sampled`` runs a whole
generation with it.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Union

import torch

from . import _lib
from ._lib import CsaqSampleParams, check, dtype_code, lib, raw_stream

__all__ = ["sample_tokens", "sample_params"]

Setting = Union[float, int, torch.Tensor]


def _setting(x: Setting, rows: int, dtype: torch.dtype, device: torch.device, what: str):
    """(device pointer or None, host value) of one sampling setting."""
    if not isinstance(x, torch.Tensor):
        return None, x
    if x.dtype != dtype or x.shape != (rows,) or x.device != device or not x.is_contiguous():
        raise ValueError(f"csaq-b200: {what} must be a number or {rows} contiguous {dtype} values on {device}")
    return x.data_ptr(), 0


def sample_params(rows: int, device: torch.device, temperature: Setting = 1.0, top_k: Setting = 0,
                  top_p: Setting = 1.0, min_p: Setting = 0.0) -> CsaqSampleParams:
    """The settings as csaq_sample_filtered takes them (tensors are used where they
    are: keep them alive while calls or captured graphs read them)."""
    f32 = torch.float32
    t, t_all = _setting(temperature, rows, f32, device, "temperature")
    k, k_all = _setting(top_k, rows, torch.int32, device, "top_k")
    p, p_all = _setting(top_p, rows, f32, device, "top_p")
    m, m_all = _setting(min_p, rows, f32, device, "min_p")
    if t is None and not t_all >= 0:
        raise ValueError(f"csaq-b200: temperature must not be negative, got {t_all}")
    if k is None and (int(k_all) != k_all or not 0 <= k_all < 1 << 31):
        raise ValueError(f"csaq-b200: top_k must be a whole number from 0 (off) up, got {k_all}")
    if p is None and not 0 < p_all <= 1:
        raise ValueError(f"csaq-b200: top_p must be in (0, 1], got {p_all}")
    if m is None and not 0 <= m_all <= 1:
        raise ValueError(f"csaq-b200: min_p must be in [0, 1], got {m_all}")
    return CsaqSampleParams(t, k, p, m, float(t_all), int(k_all), float(p_all), float(m_all))


def sample_tokens(logits: torch.Tensor, random: torch.Tensor, temperature: Setting = 1.0, top_k: Setting = 0,
                  top_p: Setting = 1.0, min_p: Setting = 0.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token (int64) per row of logits (rows, V) in float32, float16 or bfloat16.

    random holds one fp32 number in [0, 1) per row. temperature, top_k, top_p
    and min_p are numbers or device tensors of one value per row (fp32; int32
    for top_k). Tokens are ranked by falling logit, the lower index first among
    equals; top_k (0: off) keeps the first ranks, top_p of those the ranks whose
    preceding mass is at most top_p of theirs, min_p of those the tokens at
    least min_p as likely as the first. The token is the first index whose
    cumulative kept mass, in index order, exceeds random times the whole.
    Temperature 0 takes the first rank. NaN and -inf logits are never drawn; a
    row of nothing else gives -1."""
    if not logits.is_cuda:
        raise RuntimeError("csaq-b200 kernels run on CUDA tensors only (no CPU path)")
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"csaq-b200: logits must be (rows, vocabulary), got {tuple(logits.shape)}")
    code = dtype_code(logits.dtype)
    rows, V = logits.shape
    dev = logits.device
    if random.dtype != torch.float32 or random.shape != (rows,) or random.device != dev or not random.is_contiguous():
        raise ValueError(f"csaq-b200: random must be {rows} contiguous fp32 values on {dev}")
    if out is None:
        out = torch.empty_like(random, dtype=torch.int64)
    elif out.dtype != torch.int64 or out.shape != (rows,) or out.device != dev or not out.is_contiguous():
        raise ValueError(f"csaq-b200: out must be {rows} contiguous int64 values on {dev}")
    params = sample_params(rows, dev, temperature, top_k, top_p, min_p)
    if rows == 0:
        return out
    ld = logits.stride(0) if rows > 1 else V  # of a single row the stride says nothing
    if logits.stride(1) != 1 or ld < V:
        logits, ld = logits.contiguous(), V

    def call() -> int:
        return lib().csaq_sample_filtered(logits.data_ptr(), 1, 0, ld, V, rows, ctypes.byref(params),
                                          random.data_ptr(), out.data_ptr(), code, raw_stream(dev.index))

    if dev.index == torch.cuda.current_device():
        rc = call()
    else:
        with torch.cuda.device(dev):
            rc = call()
    if rc:
        check(rc, "sample_filtered")
    return out
