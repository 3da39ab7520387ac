"""Inputs of the paged attention on which no key can be missing, or count twice, unnoticed. With random keys each of n weighs 1 / n,
less than a tolerance that allows for rounded probabilities.

marked: all scores are alike and the values mark classes of keys, so a result is the share of each class among the keys seen.
planted: single keys, at the borders of everything that a walk is cut into, are aligned with a query each, which they decide."""
import numpy as np

import paged_util as pu

# marked: probabilities of 1 and sums of up to 2^24 ones are exact; what is left is 1 / sum and its product (2^-24 each), and where shares
# are joined the logarithms of their sums (off by 2^-20 of up to 17: ln 2 times that of each weight, below 2^-19) and the weights'
# exp2 (2^-22), product and sum. 2^-16 of a result is eight times all of it; one key of a class of at most 200 is 2^-8.
MARK_TOLERANCE = 2.0 ** -16


def marks(length, kvh, d, way):
    """Values [length, kvh, d] of zeros and ones: key j is of class j % d (way 0: of neighbours one each) or (j / 32) % d (steps)."""
    v = np.zeros((length, kvh, d), dtype=np.float32)
    j = np.arange(length)
    v[j, :, (j if way == 0 else j // 32) % d] = 1.0
    return v


def mark_shares(length, n, d, way, mask, usable=None):
    """f64 [n, d]: of the keys that row i (position length - n + i) sees, the share of each class."""
    seen = pu.sees(np.arange(n) + length - n, np.arange(length), *mask)
    if usable is not None:
        seen &= usable[None, :]
    out = seen.astype(np.float64) @ marks(length, 1, d, way)[:, 0]
    return out / np.maximum(seen.sum(1), 1)[:, None]


def borders(length, first, mask):
    """Positions on both sides of every multiple of 128 keys (the shares begin at some) and of a few 16, the first and last keys, and
    where window and sinks of the rows at first .. length - 1 begin and end."""
    block, window, sink = mask
    at = {0, 1, length - 1, length - 2}
    edges = list(range(128, length + 1, 128)) + [16, 32, 48, 64, length // 32 * 32, length // 16 * 16, sink * block]
    for p in {first, length - 1}:
        edges.append(p + 1)
        if window:
            edges.append((p // block - window + 1) * block)
    for e in edges:
        at |= {e - 1, e}
    return np.array(sorted(x for x in at if 0 <= x < length))


def plant(rng, keys, at):
    """Puts rows of +-4 with signs of their own at positions `at` of keys [length, kvh, d], and returns them [len(at), d] (a query of
    one scores 16 sqrt(d) with it, some 50 with another at most, 20 with the rest)."""
    rows = rng.choice(np.array([-4.0, 4.0], dtype=np.float32), (len(at), keys.shape[-1]))
    keys[at] = rows[:, None, :]
    return rows
