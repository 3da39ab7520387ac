"""Plain numpy forms of attention over packed sequences, its gradients and rotary positions, in 64 bits, and how far a kernel may be off."""
import numpy as np

from paged_util import sees

BF16_HALF, F32_HALF = 2.0 ** -8, 2.0 ** -24   # half a step, relative to the value


def visible(nq, nk, causal, block=1, window=0, sink=0):
    """[nq, nk]: what the rows of a sequence see of its keys."""
    if not causal:
        return np.ones((nq, nk), dtype=bool)
    return sees(np.arange(nq) + nk - nq, np.arange(nk), block, window, sink)


def _products(a, b):   # [n, m] of a [n, d] and b [m, d]; what no mask shows may be anything
    with np.errstate(all="ignore"):
        return a @ b.T


def _score_error(q, k, scale, seen):
    """How far a score in f32 may be off, absolutely: d products and as many sums, and the multiplication by scale log2 e."""
    s = np.where(seen, _products(np.abs(q), np.abs(k)), 0.0)
    return (q.shape[-1] + 4) * F32_HALF * s * scale


def attention(q, k, v, seen, scale, out_bf16):
    """One head of one sequence: (out, lse, bounds of both)."""
    n, d = q.shape
    if k.shape[0] == 0 or n == 0:
        return np.zeros((n, d)), np.full(n, -np.inf), np.full((n, d), 1e-30), np.full(n, 1e-30)   # (zeros, and no sum)
    some = seen.any(1)
    s = np.where(seen, np.where(seen, _products(q, k), 0.0) * scale, -np.inf)
    top = np.where(some, s.max(1), 0.0)
    e = np.exp(s - top[:, None])
    total = e.sum(1)
    p = e / np.where(some, total, 1.0)[:, None]
    with np.errstate(divide="ignore"):
        lse = np.where(some, top + np.log(np.where(some, total, 1.0)), -np.inf)
    cols = seen.any(0)
    values = np.where(cols[:, None], v, 0.0)
    out, mag = p @ values, p @ np.abs(values)
    off = _score_error(q, k, scale, seen).max(1, initial=0.0)
    sums = F32_HALF * (k.shape[0] / 16 + 64)        # a lane's sums of a row, then sixteen of them
    # weights rounded to bf16, their scores' error (twice: the row sum has it too), the exponential's and the sums' own
    terms = BF16_HALF + 2 * off + sums + 2.0 ** -18
    bound = terms[:, None] * mag + (BF16_HALF if out_bf16 else F32_HALF) * np.abs(out) + 1e-30
    return out, lse, bound, off + sums + 2.0 ** -18 + 4 * F32_HALF * np.abs(np.where(some, lse, 0.0))


def gradients(q, k, v, dout, out, lse, seen, scale, few=0):
    """One head of one sequence, with the result and the logarithms that the kernels are given: (dq, dk, dv, bounds of each before the
    results' own rounding). Rows that see up to `few` keys: with sum_j p_j dp_j in place of sum(dout out)."""
    n, m, d = q.shape[0], k.shape[0], q.shape[1]
    if m == 0 or n == 0:
        z = np.zeros((n, d)), np.zeros((m, d)), np.zeros((m, d))
        return (*z, *z)
    s = np.where(seen, _products(q, k), 0.0) * scale
    p = np.where(seen, np.exp(s - np.where(np.isfinite(lse), lse, 0.0)[:, None]), 0.0)
    dp = _products(dout, v)
    some = seen.sum(1, keepdims=True) <= few
    delta = np.where(some, np.where(seen, p * dp, 0.0).sum(1, keepdims=True), (dout * out).sum(1, keepdims=True))
    ds = p * (dp - delta)
    # a row that sees one key: its weight is 1 whatever the score, so dS is 0, where the rounding of the given result would leave some 2^-8 of dp
    ds = np.where(seen.sum(1, keepdims=True) == 1, 0.0, ds)
    dq, dk, dv = ds @ k * scale, ds.T @ q * scale, p.T @ dout
    # P: its score's error, -lse's rounding and the exponential's; dP - D: products in f32
    off = _score_error(q, k, scale, seen) + 2 * F32_HALF * np.abs(np.where(np.isfinite(lse), lse, 0.0))[:, None] + 2.0 ** -20
    off_dp = (d + 4) * F32_HALF * (_products(np.abs(dout), np.abs(v)) + (np.abs(dout) * np.abs(out)).sum(1, keepdims=True))
    # (few keys: each p_j of their sum is off as P is, each dp_j as dP)
    off_dp = off_dp + np.where(some, np.where(seen, p * (off * np.abs(dp) + (d + 4 + few) * F32_HALF * _products(np.abs(dout), np.abs(v))), 0.0).sum(1, keepdims=True), 0.0)
    ep = p * (off + BF16_HALF)
    es = np.abs(ds) * (off + BF16_HALF + 2 * F32_HALF) + p * off_dp
    acc = F32_HALF * (max(n, m) / 16 + 64)          # f32 sums of the products over rows, or keys
    bq = (es + acc * np.abs(ds)) @ np.abs(k) * scale
    bk = (es + acc * np.abs(ds)).T @ np.abs(q) * scale
    bv = (ep + acc * p).T @ np.abs(dout)
    return dq, dk, dv, bq, bk, bv


TURN = np.longdouble("6.28318530717958647692528676655900577")


def frequencies(n, base=10000.0, scaling=None):
    """Radians a position of n pairs."""
    i = np.arange(n, dtype=np.longdouble)
    if scaling and scaling[0] == "base":
        base = np.longdouble(base) * np.longdouble(scaling[1]) ** (np.longdouble(n) / (n - 1))
    theta = np.longdouble(base) ** (-i / n)
    if scaling and scaling[0] == "linear":
        theta = theta / scaling[1]
    if scaling and scaling[0] == "parts":
        _, factor, original, low, high = scaling
        kept = np.clip((original * theta / TURN - low) / (high - low), 0, 1)
        theta = theta * (kept + (1 - kept) / factor)
    return theta


def rotate(x, positions, theta, halves, amplitude=1.0, inverse=False):
    """x [tokens, heads, d] with its first 2 len(theta) channels turned by positions [tokens, len(theta)] * theta."""
    n = len(theta)
    angle = (positions.astype(np.longdouble) * theta[None, :]) % TURN
    c, s = (np.asarray(f(angle), dtype=np.float64)[:, None, :] * amplitude for f in (np.cos, np.sin))
    s = -s if inverse else s
    y = x.astype(np.float64).copy()
    a, b = (x[..., :n], x[..., n:2 * n]) if halves else (x[..., 0:2 * n:2], x[..., 1:2 * n:2])
    a, b = a.astype(np.float64), b.astype(np.float64)
    u, w = a * c - b * s, a * s + b * c
    if halves:
        y[..., :n], y[..., n:2 * n] = u, w
    else:
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = u, w
    return y
