"""The token scores and the top-k distillation in 64 bits, row by row, and the
bounds that 32-bit arithmetic on them has. Test infrastructure only.

u = 2^-24 is half a step of float32. A kernel's term exp((x - m) / T) is off by
at most u (4 + 3 |d|) of itself, d = (x - m) / T in base 2: u |d| for the
difference, u |d| for the product, u |d| for reading both back in a sum, and one
step of the exponential with its rounding. Sums are held in at least 32 bits over
at most 64 sequential terms of one sign per thread (64 u) or in 64 bits."""
import math

import numpy as np

U = 2.0 ** -24
TINY = 2.0 ** -125  # smaller magnitudes may be flushed
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
SMALLEST = {"f32": TINY, "bf16": 2.0 ** -125, "f16": 2.0 ** -25}


def softmax_row(x, T):
    """dict of a row's distribution: d, p, log p, ln of the sum, kind."""
    x = np.asarray(x, np.float64)
    if np.isnan(x).any() or (x == np.inf).any():
        return dict(kind="bad")
    if (x == -np.inf).all():
        return dict(kind="empty")
    m = x.max()
    with np.errstate(over="ignore"):
        d = (x - m) / T
    e = np.exp(d)
    s = e.sum()
    lp = d - math.log(s)
    p = e / s
    dd = np.where(p > 0, d, 0.0)
    # how far ln s, and sums weighted with |d|, may be off
    ls_err = U * (70.0 + 5.0 * (p * -dd).sum())
    return dict(kind="ok", d=d, p=p, lp=lp, ls=math.log(s), m=m, ls_err=ls_err,
                h_err=ls_err + U * ((p * (-dd) * (74.0 + 5.0 * -dd)).sum()))


def score_row(x, T, target, k):
    """logp, entropy, [(id, logp)] * k, and how far logp and entropy may be off."""
    r = softmax_row(x, T)
    nan = math.nan
    if r["kind"] == "bad":
        return (0.0 if target < 0 else nan), nan, [(-1, nan)] * k, 0.0, 0.0
    C = len(x)
    if r["kind"] == "empty":
        lp = 0.0 if target < 0 else nan if target >= C else -math.inf
        return lp, 0.0, [(-1, -math.inf)] * k, 0.0, 0.0
    p, lp = r["p"], r["lp"]
    plp = np.zeros(C)
    np.multiply(p, lp, out=plp, where=p > 0)
    order = np.lexsort((np.arange(C), -np.asarray(x, np.float64)))[:k]
    top = [(int(j), float(lp[j])) if x[j] > -np.inf else (-1, -math.inf) for j in order]
    top += [(-1, -math.inf)] * (k - len(top))
    got = 0.0 if target < 0 else nan if target >= C else float(lp[target])
    return got, float(-plp.sum()), top, r["ls_err"], r["h_err"]


def score_grad_row(x, T, target, dlogp, dentropy):
    """dlogits and the elementwise bound of a float32 computation of it."""
    C = len(x)
    r = softmax_row(x, T)
    if r["kind"] == "bad" or target >= C:
        return np.full(C, math.nan), np.zeros(C)
    if r["kind"] == "empty":
        return np.zeros(C), np.zeros(C)
    p = r["p"]
    lp = np.where(p > 0, r["lp"], 0.0)
    h = -(p * lp).sum()
    up = dlogp if target >= 0 else 0.0
    g = -up * p - dentropy * p * (lp + h)
    mag = p * (abs(up) + abs(dentropy) * (np.abs(lp) + h))
    if target >= 0:
        g[target] += up
        mag[target] += abs(up)
    d = np.where(p > 0, -r["d"], 0.0)
    tol = U * (16.0 + 6.0 * d) * mag + mag * r["ls_err"] + \
        p * abs(dentropy) * (r["ls_err"] + r["h_err"])
    return g / T, tol / T


def teacher_row(ids, v, C, tail):
    """q by entry, the rest's mass, S; None where the list is bad."""
    ids, v = np.asarray(ids), np.asarray(v, np.float64)
    keep = ids >= 0
    named = ids[keep]
    if (named >= C).any() or len(set(named.tolist())) != len(named) or \
            np.isnan(v[keep]).any() or (v[keep] == np.inf).any():
        return None
    q = np.where(keep, np.exp(np.where(keep, v, 0.0)), 0.0)
    if not keep.any():
        return q, 0.0, 0.0
    if tail:
        left = max(0.0, 1.0 - q.sum())
        return q, left, q.sum() + left
    total = q.sum()
    return (q / total, 0.0, 1.0) if total > 0 else (q, 0.0, 0.0)


def distill_row(x, ids, v, T, tail):
    """row loss, dlogits of it, and their bounds."""
    C = len(x)
    t, r = teacher_row(ids, v, C, tail), softmax_row(x, T)
    if t is None or r["kind"] == "bad":
        return math.nan, np.full(C, math.nan), 0.0, np.zeros(C)
    q, left, S = t
    ids = np.asarray(ids)
    if r["kind"] == "empty":
        return (math.inf if q.sum() > 0 else 0.0), np.zeros(C), 0.0, np.zeros(C)
    listed = np.zeros(C, bool)
    listed[ids[ids >= 0]] = True
    rest = ~listed & (np.asarray(x, np.float64) > -np.inf)
    if not rest.any():
        S, left = S - left, 0.0
    d = r["d"]
    L = 0.0
    for i, j in enumerate(ids):
        if j >= 0 and q[i] > 0:
            L += q[i] * (math.log(q[i]) - r["lp"][j])
    lt_err = share = 0.0
    if left > 0:
        md = d[rest].max()
        e = np.exp(d[rest] - md)
        lt = md + math.log(e.sum())
        L += left * (math.log(left) - (lt - r["ls"]))
        share = np.zeros(C)
        share[rest] = np.exp(d[rest] - lt)
        lt_err = U * (70.0 + 5.0 * (e / e.sum() * -(d[rest] - md)).sum())
    p = r["p"]
    g = S * p - left * share
    mag = S * p + left * share
    for i, j in enumerate(ids):
        if j >= 0:
            g[j] -= q[i]
            mag[j] += q[i] * (1.0 + abs(float(v[i]) if np.isfinite(v[i]) else 0.0))
    dd = np.where(np.isfinite(d), -d, 0.0)
    # S p_j and left's share of it are each a product of factors right to a few u
    # and an exponential's (16 + 6 |d|) u; their difference adds one rounding.
    tol = mag * (U * (24.0 + 6.0 * dd) + 2 * r["ls_err"] + 2 * lt_err)
    L_tol = (S + 1.0) * (r["ls_err"] + lt_err) + U * abs(L) + U * 4.0
    return L, g / T, L_tol, tol / T
