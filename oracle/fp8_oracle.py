"""Float64 restatement of the 8-bit block-scaled projection, the routing of
frames to experts and the experts' FeedForward, from their definitions.

A value is an e4m3 code (sign, 4 exponent bits with bias 7, 3 mantissa bits; 0x7F
and 0xFF are NaN, the largest is 448) times 2^(s - 127) of its block of 128.
"""
from __future__ import annotations

import numpy as np

BLOCK = 128


def code_values() -> np.ndarray:
    """The value of each of the 256 codes."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, np.ldexp(8.0 + m, e - 10), np.ldexp(m.astype(np.float64), -9))
    v[(c & 127) == 127] = np.nan
    return np.where(c >> 7, -v, v)


VALUES = code_values()
POSITIVE = VALUES[:127]  # ascending, 0 .. 448


def scale_byte(amax: np.ndarray) -> np.ndarray:
    """The smallest s >= 0 with amax <= 448 * 2^(s - 127); 127 for 0."""
    amax = np.asarray(amax, np.float64)
    m, x = np.frexp(np.where(amax > 0, amax, 1.0))
    e = np.where(m <= 0.875, x - 9, x - 8)  # 448 = 0.875 * 2^9
    return np.where(amax > 0, np.maximum(e + 127, 0), 127).astype(np.int64)


def encode(v: np.ndarray) -> np.ndarray:
    """Codes of |v| <= 448 rounded to nearest, ties to even; NaN and infinity
    as 0x7F."""
    v = np.asarray(v, np.float64)
    a = np.where(np.isfinite(v), np.abs(v), 0.0)
    hi = np.clip(np.searchsorted(POSITIVE, a), 1, 126)
    lo = hi - 1
    dl, dh = a - POSITIVE[lo], POSITIVE[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.isfinite(v), code | (np.signbit(v).astype(np.int64) << 7), 127)
    return code.astype(np.uint8)


def _finite_max(b, axis):
    return np.max(np.where(np.isfinite(b), np.abs(b), 0.0), axis=axis)


def round_rows(x: np.ndarray) -> np.ndarray:
    """Values that the codes of x [rows, K] stand for."""
    x = np.asarray(x, np.float64)
    out = np.empty_like(x)
    for lo in range(0, x.shape[1], BLOCK):
        b = x[:, lo:lo + BLOCK]
        s = scale_byte(_finite_max(b, 1))[:, None] - 127
        with np.errstate(invalid="ignore"):
            out[:, lo:lo + BLOCK] = np.ldexp(VALUES[encode(np.ldexp(b, -s))], s)
    return out


def quantize_weight(w: np.ndarray):
    """Codes [N, K] and scale bytes [ceil(N/128), ceil(K/128)] of w [N, K]."""
    n, k = w.shape
    codes = np.empty((n, k), np.uint8)
    scales = np.empty((-(-n // BLOCK), -(-k // BLOCK)), np.uint8)
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            at = np.s_[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK]
            b = np.asarray(w[at], np.float64)
            scales[i, j] = scale_byte(_finite_max(b, None))
            codes[at] = encode(np.ldexp(b, 127 - int(scales[i, j])))
    return codes, scales


def weight_values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    n, k = codes.shape
    s = np.ldexp(1.0, scales.astype(np.int64) - 127)
    s = np.where(scales == 255, np.nan, s)
    return VALUES[codes] * np.repeat(np.repeat(s, BLOCK, 0)[:n], BLOCK, 1)[:, :k]


def linear(x, codes, scales, bias=None):
    """(y, sum of the products' magnitudes), both [rows, N]."""
    q, w = round_rows(x), weight_values(codes, scales)
    with np.errstate(invalid="ignore"):
        y, mag = q @ w.T, np.abs(q) @ np.abs(w).T
    return (y if bias is None else y + np.asarray(bias, np.float64)), mag


def route(logits, top_k, score="softmax", bias=None, n_groups=1, topk_groups=1, renormalize=False, scale=1.0):
    """(indices, weights) [rows, top_k]."""
    x = np.asarray(logits, np.float64)
    rows, n = x.shape
    x = np.where(np.isnan(x), -np.inf, x)
    idx = np.full((rows, top_k), -1, np.int32)
    w = np.zeros((rows, top_k))
    size = n // n_groups
    for r in range(rows):
        there = x[r] > -np.inf
        s = np.zeros(n)
        with np.errstate(over="ignore"):
            if score == "softmax":
                if there.any():
                    mx = x[r].max()
                    s[there] = np.where(x[r][there] == mx, 1.0, np.exp(np.where(x[r][there] == mx, 0.0, x[r][there] - mx)))
                    s /= s.sum()
            else:
                s[there] = 1.0 / (1.0 + np.exp(-x[r][there]))
        c = s if bias is None else s + np.asarray(bias, np.float64)
        c = np.where(there & (c > -np.inf), c, -np.inf)
        if n_groups > 1:
            two = -np.sort(-c.reshape(n_groups, size), axis=1)[:, :2]
            best = two[:, 0].copy()
            if size > 1:
                best = np.where(two[:, 1] > -np.inf, two[:, 0] + np.where(two[:, 1] > -np.inf, two[:, 1], 0.0), best)
            kept = np.argsort(-best, kind="stable")[:topk_groups]
            c = np.where(np.isin(np.arange(n) // size, kept), c, -np.inf)
        order = [e for e in np.argsort(-c, kind="stable")[:top_k] if c[e] > -np.inf]
        idx[r, :len(order)] = order
        w[r, :len(order)] = s[order]
        if renormalize and w[r].sum() > 0:
            w[r] /= w[r].sum()
    return idx, w * scale


def silu(v):
    with np.errstate(over="ignore", invalid="ignore"):
        return np.where(v > -700, v / (1.0 + np.exp(-v)), 0.0 * v)


def experts(x, idx, w, lin1, lin2, b1=None, b2=None, residual=None, res_scale=1.0, sum_err=0.0):
    """lin1, lin2: per expert (codes, scales). Returns (y, bound): bound is how
    far a result may be whose sums are off by sum_err of their terms'
    magnitudes, before its own rounding. A hidden value so far off may round to
    another code, and the bound counts the codes it may round to."""
    x = np.asarray(x, np.float64)
    y, bound = np.zeros_like(x), np.zeros_like(x)
    q = round_rows(x)
    for e in sorted(set(int(v) for v in np.unique(idx) if 0 <= v < len(lin1))):
        w1, w2 = weight_values(*lin1[e]), weight_values(*lin2[e])
        c1 = 0.0 if b1 is None else np.asarray(b1[e], np.float64)
        c2 = 0.0 if b2 is None else np.asarray(b2[e], np.float64)
        for j in range(idx.shape[1]):
            r = np.nonzero(idx[:, j] == e)[0]
            if not len(r):
                continue
            wj = np.asarray(w[r, j], np.float64)[:, None]
            h = q[r] @ w1.T + c1
            dh = sum_err * (np.abs(q[r]) @ np.abs(w1).T + np.abs(c1))
            g = silu(h)
            dg = 1.1 * dh + 2.0 ** -20 * np.abs(g)  # |silu'| < 1.1; exp and reciprocal
            hq = round_rows(g)
            step = np.maximum(np.abs(round_rows_like(g + dg, g) - hq), np.abs(round_rows_like(g - dg, g) - hq))
            o = hq @ w2.T + c2
            y[r] += wj * o
            bound[r] += np.abs(wj) * (step @ np.abs(w2).T + sum_err * ((np.abs(hq) + step) @ np.abs(w2).T + np.abs(c2)))
    y, bound = res_scale * y, abs(res_scale) * bound
    if residual is not None:
        y = y + np.asarray(residual, np.float64)
    return y, bound


def round_rows_like(x, like):
    """x rounded in the steps of `like`'s blocks (past their largest code: to it)."""
    out = np.empty_like(x)
    for lo in range(0, x.shape[1], BLOCK):
        s = scale_byte(_finite_max(like[:, lo:lo + BLOCK], 1))[:, None] - 127
        t = np.ldexp(x[:, lo:lo + BLOCK], -s)
        out[:, lo:lo + BLOCK] = np.ldexp(VALUES[encode(np.clip(t, -448, 448))], s)
    return out
