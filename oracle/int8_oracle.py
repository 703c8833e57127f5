"""CPU oracle of the 8-bit products and of the sampler on logits (numpy, 64 bits, test-only)."""
from __future__ import annotations

import numpy as np


def quantize_rows(x: np.ndarray):
    """(codes, scales, quotients) of rows x: scale max |x| / 127 in float32, codes rint(x / s) of the quotient in 64
    bits.  x and s have 24 bits, so a quotient that is no half is at least 2^-33 of itself away from one and float64
    tells them apart."""
    x64 = np.asarray(x, dtype=np.float64)
    top = np.abs(x64).max(-1)
    with np.errstate(all="ignore"):
        scale = (top.astype(np.float32) / np.float32(127)).astype(np.float32)
        bad = ~np.isfinite(x64).all(-1)
        scale = np.where(bad, np.float32(np.nan), scale)
        safe = np.where(bad | (scale == 0), 1.0, scale.astype(np.float64))
        quotient = np.where((bad | (scale == 0))[..., None], 0.0, x64 / safe[..., None])
    return np.clip(np.rint(quotient), -127, 127).astype(np.int8), scale, quotient


def add_rmsnorm(h: np.ndarray, r: np.ndarray, w: np.ndarray, eps: float):
    """(normalised rows, h + r) in 64 bits."""
    s = np.asarray(h, np.float64) + np.asarray(r, np.float64)
    return s * (1.0 + np.asarray(w, np.float64)) / np.sqrt((s * s).mean(-1, keepdims=True) + eps), s


def gemm_int8(a, a_scales, w, w_scales):
    """The scaled sums in 64 bits (the integer sum is below 2^53, so it is exact in float64)."""
    total = np.asarray(a, np.float64) @ np.asarray(w, np.float64).T
    return total * np.asarray(w_scales, np.float64) * np.asarray(a_scales, np.float64)[..., None]


def silu(x):
    with np.errstate(over="ignore"):
        return x / (1.0 + np.exp(-x))


def sample(logits, temperature, u, top_k=None, top_p=None, min_p=None):
    """(token, log of its share) of one row, by a sort, sums in extended precision."""
    x = np.asarray(logits, np.float64)
    nan = np.isnan(x)
    if nan.any():
        return int(nan.argmax()), float("nan")
    best = int(x.argmax())
    if not temperature > 1e-10:
        return best, 0.0
    order = np.lexsort((np.arange(x.size), -x))
    with np.errstate(all="ignore"):
        weight = np.exp(np.asarray(x - x[best], np.longdouble) / np.longdouble(np.float32(temperature)))
    weight = np.where(x == x[best], np.longdouble(1), weight)
    if np.isfinite(x[best]):
        weight = np.where(x == -np.inf, np.longdouble(0), weight)
    else:
        weight = np.where(x == x[best], np.longdouble(1), np.longdouble(0))
    weight = np.where(weight < np.longdouble(2.0) ** -64, 0, weight)
    count = x.size
    if top_k is not None and top_k > 0:
        count = min(count, int(top_k))
    if top_p is not None and top_p < 1:
        run = np.cumsum(weight[order[:count]])
        count = min(count, 1 + int(np.searchsorted(run, np.longdouble(np.float32(top_p)) * run[-1])))
    if min_p is not None and min_p > 0:
        count = max(1, min(count, int((weight[order] >= np.longdouble(np.float32(min_p))).sum())))
    chosen = np.sort(order[:count])
    run = np.cumsum(weight[chosen])
    u = float(np.float32(u)) if u > 0 else 0.0
    held = np.nonzero((run > np.longdouble(u) * run[-1]) & (weight[chosen] > 0))[0]
    at = int(held[0]) if held.size else int(np.nonzero(weight[chosen] > 0)[0][-1])
    return int(chosen[at]), float(np.log(weight[chosen[at]] / run[-1]))
