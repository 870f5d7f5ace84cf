"""Float64 restatement of the operators on rows, from their definitions: a
residual's addition with its norm, low-rank adapters, log probabilities."""
from __future__ import annotations

import numpy as np


def norm(x, delta=None, scale=1.0, weight=None, bias=None, kind="rms", eps=1e-5):
    """(y, v, size): size is what y's rounding errors are relative to, the
    magnitudes that enter it."""
    v = np.asarray(x, np.float64)
    if delta is not None:
        v = v + np.float64(np.float32(scale)) * np.asarray(delta, np.float64)
    w = 1.0 if weight is None else np.asarray(weight, np.float64)
    b = 0.0 if bias is None else np.asarray(bias, np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        u, spread = v, 0.0
        if kind == "layer":
            u, spread = v - v.mean(-1, keepdims=True), np.abs(v).mean(-1, keepdims=True)
        r = 1.0 / np.sqrt((u * u).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
        y = u * r * w + b
        return y, v, np.abs(b) + np.abs(w) * r * (np.abs(u) + spread) + 0.0 * y


def adapted(x, which, adapters):
    """The adapters' part of a projection and the sums of its products'
    magnitudes: adapters [(a [rank, in], b [out, rank], scale)] as held (bf16
    values); rows of no adapter 0. The third result: the magnitudes that enter
    through the inner sums' size alone, sum |b| |t|."""
    x = np.asarray(x, np.float64)
    n = adapters[0][1].shape[0]
    y, mag, inner = np.zeros((len(x), n)), np.zeros((len(x), n)), np.zeros((len(x), n))
    for d, (a, b, s) in enumerate(adapters):
        at = np.nonzero(which == d)[0]
        if not len(at):
            continue
        s = np.float64(np.float32(s))
        with np.errstate(invalid="ignore"):
            t = s * (x[at] @ a.T)
            y[at] = t @ b.T
            mag[at] = (abs(s) * (np.abs(x[at]) @ np.abs(a).T)) @ np.abs(b).T
            inner[at] = np.abs(t) @ np.abs(b).T
    return y, mag, inner


def scores(logits, tokens, top_k, temperature=1.0):
    """Per row: log p of tokens [rows, n], entropy, the top_k tokens and their
    log p, and what the errors of f32 sums are relative to: (|z - M|'s mean
    under p, its square's, log sum)."""
    x = np.asarray(logits, np.float64)
    rows, v = x.shape
    t = 1.0 / np.float64(np.float32(temperature))
    lp = np.zeros(tokens.shape)
    h, idx, top = np.zeros(rows), np.full((rows, top_k), -1, np.int32), np.full((rows, top_k), -np.inf)
    sizes = np.zeros((rows, 3))
    for r in range(rows):
        there = x[r] > -np.inf
        if np.isnan(x[r]).any() or (x[r] == np.inf).any():
            full = np.full(v, np.nan)
            h[r] = np.nan
        elif not there.any():
            full = np.full(v, -np.inf)
        else:
            with np.errstate(over="ignore"):
                d = (x[r] - x[r].max()) * t
                e = np.exp(d)
            ls = np.log(e.sum())
            full, p = d - ls, e / e.sum()
            on = p > 0
            h[r] = -(p[on] * full[on]).sum()
            sizes[r] = (p[on] * -d[on]).sum(), (p[on] * d[on] ** 2).sum(), ls
        order = [i for i in np.argsort(-np.where(there, x[r], -np.inf), kind="stable")[:top_k] if there[i]]
        idx[r, :len(order)] = order
        top[r, :len(order)] = full[order]
        for j, tok in enumerate(tokens[r]):
            lp[r, j] = full[tok] if 0 <= tok < v else 0.0
    return lp, h, idx, top, sizes
