"""That the planted and marked inputs see what they are for: a definition with one key left out, a step, or one counted twice is past
the tolerance of the device's tests. No GPU."""
import numpy as np
import pytest

import paged_planted as pp
import paged_util as pu
import util  # noqa: F401

CASES = [(9001, 1, (1, 0, 0)), (20000, 2, (1, 0, 0)), (7000, 64, (1, 4500, 70)), (4680, 1560, (1560, 0, 0)), (8000, 3, (100, 40, 2))]


@pytest.mark.parametrize("length,n,mask", CASES)
@pytest.mark.parametrize("d", [64, 128])
def test_marked(length, n, mask, d):
    rng = np.random.Generator(np.random.PCG64(length + d))
    seen = np.nonzero(pu.sees(np.array([length - 1]), np.arange(length), *mask)[0])[0]   # of the last row
    n = min(n, 3)
    for way in (0, 1):
        out = pp.mark_shares(length, n, d, way, mask)[-1]
        for lost in [[x] for x in (*rng.choice(seen, 6), seen[0], seen[-1])] + [seen[-32:], seen[:32]]:
            usable = np.ones(length, dtype=bool)
            usable[lost] = False
            off = np.abs(pp.mark_shares(length, n, d, way, mask, usable)[-1] - out)
            assert (off > 16 * pp.MARK_TOLERANCE * out).any(), (way, lost)
        twice = out * len(seen)
        twice[int(rng.choice(seen)) // (1 if way == 0 else 32) % d] += 1
        assert (np.abs(twice / (len(seen) + 1) - out) > 16 * pp.MARK_TOLERANCE * out).any()


@pytest.mark.parametrize("length,n,mask", CASES)
@pytest.mark.parametrize("d,four", [(64, False), (128, False), (128, True)])
def test_planted(length, n, mask, d, four):
    """Every planted key that a row sees: without it the row is off by more than the bound."""
    rng = np.random.Generator(np.random.PCG64(length + d + four))
    keys, values = (pu.bf16(rng.standard_normal((length, 1, d))) for _ in range(2))
    at = pp.borders(length, length - n, mask)
    rows = pp.plant(rng, keys, at)
    if four:
        keys, values = (pu.values4(*pu.quantize4(x)) for x in (keys, values))
        assert np.array_equal(keys[at, 0], rows)                 # 4 is a code
    seen = pu.sees(np.array([length - 1]), at, *mask)[0]
    assert seen.sum() >= 8
    visible = pu.sees(np.array([length - 1]), np.arange(length), *mask)
    scores = rows.astype(np.float64) @ keys[:, 0].astype(np.float64).T * d ** -0.5   # the last position, a head a target
    v = values[:, 0].astype(np.float64)

    def attend(keep):
        s = np.where(keep, scores, -np.inf)
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        return p @ v, p @ np.abs(v)

    out, mag = attend(visible)
    bound = pu.attention_bound(out, mag, True, d ** -0.5 * 1.45 * 4 * np.abs(keys).max() * d)
    alone = np.abs(out[seen] - v[at[seen]]).max()
    assert alone < 1e-6, alone                                   # the target is all of the result
    for lost in (np.arange(length)[None] == at[:, None], np.isin(np.arange(length), at)[None]):   # a row's own target; all of them
        without, _ = attend(visible & ~lost)
        off = (np.abs(without - out) / bound)[seen].max(1)
        assert off.min() > 20, off.min()
