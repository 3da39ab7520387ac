"""Plain numpy forms of the paged KV cache: where tokens lie, the rotation, the 4-bit format, the attention in 64 bits."""
import numpy as np

LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)


def bf16(x):
    """f32 -> the nearest bf16 value (ties to even), as f32."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)
    return np.where(np.isfinite(x), r, x).astype(np.float32)


def rotate(x, cos, sin, rows, halves):
    """x [n, heads, d] f32 turned by rows `rows` of the tables, every product and sum rounded to f32."""
    x = x.astype(np.float32)
    half = x.shape[-1] // 2
    if halves:
        c, s = cos[rows][:, None, :half], sin[rows][:, None, :half]
        a, b = x[..., :half], x[..., half:]
        return np.concatenate([a * c - b * s, a * s + b * c], -1)
    c, s = cos[rows][:, None, 0::2], sin[rows][:, None, 0::2]
    a, b = x[..., 0::2], x[..., 1::2]
    return np.stack([a * c - b * s, a * s + b * c], -1).reshape(x.shape)


def quantize4(x):
    """x [.., d] f32 -> (codes [.., d/2] u8, scales [.., d/32] u8): by search over the levels, in 64 bits."""
    shape = x.shape
    b = x.astype(np.float64).reshape(-1, 32)
    good = np.isfinite(b).all(1)
    b = np.where(good[:, None], b, 0.0)
    top = np.abs(b).max(1)
    byte = np.ones(len(b), dtype=np.int64)
    for e in range(1, 255):                      # the smallest power of two with top <= 6 * 2^(byte - 127)
        byte = np.where(top > 6.0 * 2.0 ** (byte - 127), byte + 1, byte)
    a = np.abs(b) / 2.0 ** (byte - 127)[:, None]
    dist = np.abs(a[..., None] - LEVELS)
    near = dist.min(-1, keepdims=True)
    tie = dist == near                           # one level, or two neighbours: then the even code
    first = tie.argmax(-1)
    two = tie.sum(-1) == 2
    code = np.where(two & (first % 2 == 1), first + 1, first)
    code = (code + 8 * np.signbit(b)).astype(np.uint8).reshape(shape)
    scales = np.where(good, byte, 255).astype(np.uint8).reshape(*shape[:-1], shape[-1] // 32)
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def values4(codes, scales):
    """The f64 values that codes and scales stand for."""
    v = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], 2 * codes.shape[-1])
    x = LEVELS[v & 7] * np.where(v & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return x * np.repeat(s, 32, -1)


def sees(p, j, block, window, sink):
    """Whether positions p (column) see keys j (row)."""
    tp, tj = p[:, None] // block, j[None, :] // block
    m = (tj <= tp) & (p[:, None] >= 0)
    if window:
        m &= (tp - tj < window) | (tj < sink)
    return m


def attention(q, keys, values, first_pos, scale, block=1, window=0, sink=0, usable=None):
    """One sequence in 64 bits: q [n, heads, d] at positions first_pos .., keys / values [len, kv_heads, d]; usable [len]: keys
    that lie in a page of the pool. Returns (out [n, heads, d], weights' sum of |v| likewise)."""
    n, heads, d = q.shape
    length, kvh = keys.shape[0], keys.shape[1] if keys.ndim == 3 else 1
    out, mag = np.zeros((n, heads, d)), np.zeros((n, heads, d))
    if length == 0 or n == 0:
        return out, mag
    m = sees(np.arange(n) + first_pos, np.arange(length), block, window, sink)
    if usable is not None:
        m &= usable[None, :]
    any_row = m.any(1)
    for h in range(heads):
        kv = h * kvh // heads
        cols = m.any(0)                          # what no row sees is not touched, whatever it holds
        s = np.full((n, length), -np.inf)
        s[:, cols] = (q[:, h].astype(np.float64) @ keys[cols, kv].astype(np.float64).T) * scale
        s = np.where(m, s, -np.inf)
        top = np.where(any_row, s.max(1, initial=-np.inf), 0.0)
        w = np.where(m, np.exp(s - top[:, None]), 0.0)
        w /= np.where(any_row, w.sum(1), 1.0)[:, None]
        v = np.where(cols[:, None], values[:, kv].astype(np.float64), 0.0)
        out[:, h], mag[:, h] = w @ v, w @ np.abs(v)
    return out, mag


def attention_bound(out, mag, out_bf16, worst_score):
    """How far a kernel may be off, element by element: the probabilities rounded to bf16 (2^-8 of each term), the result's own
    rounding (bf16 2^-8, f32 2^-24), scores in f32 (a product of d terms is off by at most (d + 2) 2^-24 of the sum of their
    magnitudes, `worst_score` in units of the exponent; a weight by twice that), and f32 sums of up to 2^17 terms in blocks."""
    terms = 2.0 ** -8 + 2.0 * 130 * 2.0 ** -24 * worst_score + 2.0 ** -12
    return terms * mag + (2.0 ** -8 if out_bf16 else 2.0 ** -24) * np.abs(out) + 1e-30
