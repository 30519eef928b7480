"""The 8-bit cache, page bounds and page selection of include/drkv.h restated in numpy, and decode attention in 64 bits."""
from __future__ import annotations

import numpy as np

# every e4m3 byte's value; 0x7f and 0xff are NaN
E4M3 = np.array([np.nan if b & 0x7f == 0x7f else (-1.0 if b & 0x80 else 1.0) *
                 ((b & 7) * 2.0 ** -9 if (b >> 3) & 15 == 0 else (8 + (b & 7)) * 2.0 ** (((b >> 3) & 15) - 10)) for b in range(256)])
_POSITIVE = E4M3[:0x7f]                                     # ascending


def exponent_for(amax: np.ndarray, top: float, lo: int, hi: int) -> np.ndarray:
    """Smallest e with amax <= top * 2^e, held within lo..hi (amax finite, float64)."""
    e = np.full(amax.shape, lo, dtype=np.int64)
    pos = amax > 0
    g = np.floor(np.log2(amax[pos] / top)).astype(np.int64) - 1
    for _ in range(3):                                      # the logarithm is a first guess
        g = np.where(top * 2.0 ** g.astype(np.float64) < amax[pos], g + 1, g)
    e[pos] = g
    return np.clip(e, lo, hi)


def round_e4m3(y: np.ndarray) -> np.ndarray:
    """Bytes of y (float64): nearest, ties to even, saturating; NaN is 0x7f."""
    a = np.minimum(np.abs(y), 448.0)
    i = np.clip(np.searchsorted(_POSITIVE, np.where(np.isnan(a), 0, a)), 1, 126)
    lo, hi = _POSITIVE[i - 1], _POSITIVE[i]
    a = np.where(np.isnan(a), 0, a)
    up = (a - lo > hi - a) | ((a - lo == hi - a) & (i % 2 == 0))
    out = np.where(up, i, i - 1).astype(np.uint8)
    out = out | np.where(np.signbit(y), 0x80, 0).astype(np.uint8)
    return np.where(np.isnan(y), out & 0x80 | 0x7f, out).astype(np.uint8)


def quantise(x: np.ndarray):
    """x [..., d] float64 -> (bytes [..., d], exponents [...])."""
    amax = np.where(np.isfinite(x), np.abs(x), 0).max(-1)
    e = exponent_for(amax, 448.0, -127, 120)
    return round_e4m3(x * 2.0 ** (-e.astype(np.float64))[..., None]), e


def stored_values(x: np.ndarray) -> np.ndarray:
    b, e = quantise(x)
    return E4M3[b] * 2.0 ** e.astype(np.float64)[..., None]


def bounds(keys: np.ndarray):
    """keys [n, d] float64 of one page and head -> (b_max, b_min, e)."""
    k = np.where(np.isnan(keys), np.nan, keys)
    with np.errstate(all="ignore"):
        hi, lo = np.nanmax(k, 0), np.nanmin(k, 0)
    e = exponent_for(np.array([max(np.abs(hi).max(), np.abs(lo).max())]), 127.0, -126, 121)[0]
    return np.ceil(hi / 2.0 ** e).astype(int), np.floor(lo / 2.0 ** e).astype(int), int(e)


def page_scores(q: np.ndarray, b_max, b_min, e) -> np.ndarray:
    """q [group, d]; b_max, b_min [pages, d], e [pages] -> exact scores [pages]."""
    f = exponent_for(np.abs(q).max(-1), 127.0, -126, 121).astype(np.float64)
    q8 = np.rint(q / 2.0 ** f[:, None])
    s = np.maximum(q8, 0) @ b_max.T.astype(np.float64) + np.minimum(q8, 0) @ b_min.T.astype(np.float64)
    return (s * 2.0 ** (f[:, None] + np.asarray(e, dtype=np.float64)[None, :])).max(0)


def select(scores: np.ndarray, resident: np.ndarray, top: int, first: int, last: int) -> list:
    n = len(scores)
    key = scores.copy()
    key[:first] = np.inf
    key[max(0, n - last):] = np.inf
    order = [p for p in np.argsort(-key, kind="stable") if resident[p]]
    return sorted(int(p) for p in order[:top])


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float):
    """q [group, d], k, v [n, d] in float64 -> (out, sum p|v|, largest score magnitude sum scale |q||k|) per head."""
    s = (q @ k.T) * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    return p @ v, p @ np.abs(v), ((np.abs(q) @ np.abs(k).T) * scale).max(-1, keepdims=True)


def attend_tolerance(out, pv_abs, mag, half_step, weight_step):
    """One rounding of the output (fp16 subnormals: 2^-25); weights rounded by weight_step; scores accumulated in fp32:
    2^-20 of the magnitude they are summed at, in nats, acting on numerator and denominator; fp32 sums and ex2: 2^-18."""
    return np.abs(out) * half_step + 2.0 ** -25 + pv_abs * (weight_step + 2.0 ** -18 + 2 * 2.0 ** -20 * mag)
