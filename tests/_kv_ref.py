"""Plain references of the quantised KV cache for the tests: the stored codes in
fp32 numpy operations (the kernel's definition, operation by operation) and the
attention over stored values in 64 bits."""

import numpy as np
import torch

F = np.float32


def quantise(x, bits, group):
    """(codes (..., D) int, words (..., D/group) uint32) of fp32 x (..., D)."""
    n = F(2 ** bits - 1)
    with np.errstate(all="ignore"):
        g = x.astype(F).reshape(*x.shape[:-1], -1, group)
        ok = np.isfinite(g).all(-1)
        lo = np.minimum(np.where(np.isnan(g), F(0), g).min(-1), F(0))
        hi = np.maximum(np.where(np.isnan(g), F(0), g).max(-1), F(0))
        span = (hi - lo).astype(F)
        halves = ((F(0.5) * hi - F(0.5) * lo).astype(F) / (F(0.5) * n)).astype(F)
        s32 = np.where(span <= F(3.4e38), (span / n).astype(F), halves)
        up = (np.where(ok, s32, F(0)).astype(F).view(np.uint32).astype(np.int64) + 0xFFFF) & 0xFFFF0000
        up = np.maximum(up, 0x00800000)
        up = np.where(span > 0, up, 0)
        up = np.where(ok, up, 0x7FC00000).astype(np.uint32)
        s = up.view(F)
        div = np.where(s != 0, s, F(1)).astype(F)
        z = np.clip(np.rint((-lo / div).astype(F)), 0, n)
        z = np.where(ok & (span > 0), z, 0)
        c = np.rint((g / div[..., None]).astype(F)) + z[..., None]
        c = np.clip(np.where(np.isnan(c), 0, c), 0, n)
    return c.reshape(x.shape).astype(np.int64), (up | (0x6400 + z.astype(np.uint32))).astype(np.uint32)


def pack(codes, bits):
    c = codes.astype(np.uint8)
    return c if bits == 8 else c[..., 0::2] | (c[..., 1::2] << 4)


def values(codes, words, bits, group):
    """fp64 values of packed uint8 codes and uint32 words (numpy arrays)."""
    c = codes.astype(np.int64)
    if bits == 4:
        c = np.stack([c & 15, c >> 4], -1).reshape(*c.shape[:-1], -1)
    w = words.astype(np.uint32)
    s = (w & np.uint32(0xFFFF0000)).view(F).astype(np.float64)
    z = (w & np.uint32(0xFFFF)).astype(np.int64) - 0x6400
    return (c.reshape(*c.shape[:-1], -1, group) - z[..., None]).reshape(c.shape) * np.repeat(s, group, -1)


def rotate(x, cos, sin):
    """rotate_half in fp32, every product and sum rounded once."""
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    m = lambda u, v: (u * v).astype(F)  # noqa: E731
    return np.concatenate([(m(a, cos[..., :h]) - m(b, sin[..., :h])).astype(F),
                           (m(b, cos[..., h:]) + m(a, sin[..., h:])).astype(F)], -1)


def attention64(q, k, v, pos0, S, scale):
    """(out, weight of |v|) in fp64: q (B*S, Hq, D), k/v (B, Hkv, L, D) tensors;
    the second is sum_j w_j |v_j|, which every relative error of a weight acts on."""
    B, Hkv, L, D = k.shape
    Hq = q.shape[1]
    q = q.double().view(B, S, Hkv, Hq // Hkv, D)
    k, v = k.double(), v.double()
    out = torch.zeros(B, S, Hkv, Hq // Hkv, D, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    for b in range(B):
        for s in range(S):
            n = min(int(pos0[b]) + s + 1, L)
            if n <= 0:
                continue
            w = torch.softmax(torch.einsum("hgd,hld->hgl", q[b, s], k[b, :, :n]) * scale, -1)
            out[b, s] = torch.einsum("hgl,hld->hgd", w, v[b, :, :n])
            mag[b, s] = torch.einsum("hgl,hld->hgd", w, v[b, :, :n].abs())
    return out.view(B * S, Hq, D), mag.view(B * S, Hq, D)
