"""Packed sequences far from the usual shapes, against their definitions in 64 bits: groups of more heads than a step has rows, more sequences than the
gradients' plan holds starts of."""
import numpy as np
import pytest

from test_gpu_packed import MASKS, Case, run_both
from util import announce

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("mask", ["causal", "window", "full", "blocks"])
@pytest.mark.parametrize("heads", [(32, 1, 64), (40, 1, 128), (130, 1, 64), (66, 2, 128)], ids=str)
def test_wide_groups(heads, mask):
    """A step of 32 rows holds one token's heads, or a part of them; a tile of 128 rows begins within a token."""
    announce(f"{heads} {mask}")
    c = Case([(5, 5), (1, 1), (37, 37), (0, 0), (20, 64), (50, 3)], *heads, MASKS[mask], seed=14)
    out, lse, grads = run_both(c)
    c.check_forward(out, lse, f"{heads} {mask}")
    c.check_backward(out, lse, grads, f"{heads} {mask} backward")


@pytest.mark.parametrize("heads", [(2, 1, 64), (3, 3, 128)], ids=str)
@pytest.mark.parametrize("long", [0, 700])
def test_a_thousand_sequences(heads, long):
    rng = np.random.Generator(np.random.PCG64(41))
    counts = [(int(a), int(a)) for a in rng.integers(0, 10, 1100)]
    if long:
        counts[600] = (long, long)
    announce(f"1100 sequences, {heads}, the longest {max(counts)}")
    c = Case(counts, *heads, MASKS["causal"], seed=15)
    out, lse, grads = run_both(c)
    c.check_forward(out, lse, "1100 sequences")
    c.check_backward(out, lse, grads, "1100 sequences backward")
