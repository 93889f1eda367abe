"""64-bit references of the norm, the attention over a paged cache and the log probabilities, and the error bounds that
their types and orders of addition give (see token_ops_ref for the types).

A sum in fp32 is off by 2^-24 of the sum of magnitudes for each addition that a term passes: the kernels add at most 64
terms in a row (those of a thread, then of a wavefront and of a workgroup) where not said otherwise.
"""
import numpy as np

import token_ops_ref as R

ULP = 2.0 ** -24


# --------------------------------------------------------------------- norm --
def rms_norm(x, residual, weight, epsilon):
    """(normalised, sum) in 64 bits."""
    s = x if residual is None else x + residual
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        y = s / np.sqrt(np.mean(s * s, axis=-1, keepdims=True) + epsilon)
    return (y if weight is None else y * weight), s


def norm_slack(k):
    """Relative error of a normalised value in fp32: half of that of the sum of squares, and eight more roundings."""
    return (32 + k / 1024 + 8) * ULP


# --------------------------------------------------------------- attention --
def paged_attention(q, k, v, key_cache, value_cache, table, cached, starts=None, scale=1.0, window=0, kind="fp32"):
    """(result, bound of its error, key cache, value cache) in 64 bits; q [T, Hq, D], k and v [T, H, D] or None."""
    t, hq, d = q.shape
    pages, page, h, _ = key_cache.shape
    kc, vc = key_cache.copy(), value_cache.copy()
    b, reach = len(cached), table.shape[1] * page
    starts = np.arange(b + 1) * (t // b) if starts is None else starts
    y, bound = np.zeros(q.shape), np.zeros(q.shape)

    def where(i, place):
        at = table[i, place // page]
        return (at, place % page) if 0 <= at < pages else None

    for i in range(b):
        first, last = int(starts[i]), int(starts[i + 1])
        before = min(max(int(cached[i]), 0), reach)
        if k is not None:
            for j in range(first, last):
                place = before + j - first
                at = where(i, place) if place < reach else None
                if at is not None:
                    kc[at], vc[at] = k[j], v[j]
    for i in range(b):
        first, last = int(starts[i]), int(starts[i + 1])
        before = min(max(int(cached[i]), 0), reach)
        n = min(before + last - first, reach)
        spots = [(p, where(i, p)) for p in range(n)]
        places = np.array([p for p, s in spots if s is not None], np.int64)
        if len(places) == 0:
            continue
        at = np.array([s for _, s in spots if s is not None])
        keys, vals = kc[at[:, 0], at[:, 1]], vc[at[:, 0], at[:, 1]]
        for j in range(first, last):
            p = before + j - first
            seen = (places <= p) & ((places > p - window) if window else True)
            if not seen.any():
                continue
            for c in range(hq):
                kk, vv = keys[seen][:, c // (hq // h)], vals[seen][:, c // (hq // h)]
                with np.errstate(invalid="ignore", over="ignore"):
                    s = scale * (kk @ q[j, c])
                    w = np.exp(s - s.max())
                    total = w.sum()
                    w = w / total
                    y[j, c] = w @ vv
                    # scores: d products added in fp32, twice for matrix instructions that truncate; the exponential of a
                    # distance; the weights' type; n products added
                    off = d * 2 * ULP * abs(scale) * (np.abs(kk) @ np.abs(q[j, c])) + 4 * ULP * np.abs(s) + 4 * ULP * np.abs(s - s.max()) + 8 * ULP
                    rel = off + off.max() + (R.EPS[kind] / 2 if kind != "fp32" else 0) + 4 * len(s) * ULP
                    bound[j, c] = (w * rel) @ np.abs(vv) + (2.0 ** -25 / total if kind == "fp16" else 0) * np.abs(vv).sum(0) + R.EPS[kind] / 2 * np.abs(y[j, c]) + R.LEAST[kind]
                    bound[j, c] *= 1.001     # (terms of second order)
    return y, bound, kc, vc


# ---------------------------------------------------------- log probabilities --
def log_probs(logits, tokens, top):
    """(log p, its bound, entropy, its bound, top log p, its bound, top indices) in 64 bits; logits [rows, V], tokens [rows, n]."""
    rows, v = logits.shape
    l = np.where(np.isnan(logits), -np.inf, logits)
    lp, lpb = np.full(tokens.shape, -np.inf), np.zeros(tokens.shape)
    ent, entb = np.zeros(rows), np.zeros(rows)
    tl, tb, ti = np.full((rows, top), -np.inf), np.zeros((rows, top)), np.full((rows, top), -1, np.int64)
    for r in range(rows):
        most = l[r].max()
        if most == -np.inf:
            continue
        with np.errstate(invalid="ignore"):
            away = np.where(l[r] == most, 0.0, most - l[r])
        w = np.exp(-away)
        rest = w[away > 0].sum() + (np.sum(away == 0) - 1)
        log_sum = np.log1p(rest)
        wd = np.where(w > 0, w * np.where(w > 0, away, 0), 0)
        # a weight is off by 4 + 2 d parts of 2^-24; so are the sums by 64 + 4 and the weighted mean of that
        mean_away = wd.sum() / max(rest, 1e-300)
        off_log = rest / (1 + rest) * (70 + 2 * mean_away) * ULP + 4 * ULP * log_sum
        ent[r] = log_sum + wd.sum() / (1 + rest)
        entb[r] = off_log + 2 * (80 * wd.sum() + 2 * (wd * np.where(w > 0, away, 0)).sum()) / (1 + rest) * ULP + 4 * ULP * ent[r] + 1e-37

        def of(x):
            if x == -np.inf:
                return -np.inf, 0.0
            a = 0.0 if x == most else most - x
            return -a - log_sum, off_log + 4 * ULP * (a + log_sum) + 1e-37

        for j, t in enumerate(tokens[r]):
            if 0 <= t < v:
                lp[r, j], lpb[r, j] = of(l[r, t])
        order = np.lexsort((np.arange(v), -l[r]))[:top]
        for j, t in enumerate(order):
            if l[r, t] > -np.inf:
                ti[r, j] = t
                tl[r, j], tb[r, j] = of(l[r, t])
    return lp, lpb, ent, entb, tl, tb, ti
