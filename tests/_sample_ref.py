"""Filtered sampling in 64-bit numpy, one row at a time."""

import numpy as np


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The token of logits x (1-D, exact in float64) for the random number u, and the
    kept indices. Settings arrive as the 32-bit values that the kernel sees."""
    x = np.asarray(x, np.float64)
    temperature, top_p, min_p = (float(np.float32(v)) for v in (temperature, top_p, min_p))
    ok = ~np.isnan(x) & (x != -np.inf)
    if not ok.any():
        return -1, np.array([], np.int64)
    x = np.where(ok, x, -np.inf)
    rank = np.argsort(-x, kind="stable")
    rank = rank[ok[rank]]
    if not temperature > 0:
        return int(rank[0]), rank[:1]
    with np.errstate(invalid="ignore"):
        w = (x == np.inf).astype(np.float64) if x.max() == np.inf else np.exp((x - x.max()) / temperature)
    if top_k > 0:
        rank = rank[:top_k]
    run = np.cumsum(w[rank])
    if top_p < 1:
        rank = rank[run - w[rank] <= max(top_p, 0.0) * run[-1]]
    rank = np.sort(rank[w[rank] >= min(min_p, 1.0)])
    run = np.cumsum(w[rank])
    u = min(max(float(u), 0.0), 1 - 2.0 ** -53)
    at = np.searchsorted(run, u * run[-1], side="right")
    return int(rank[min(at, len(rank) - 1)]), rank
