"""Packed sequences at the borders of what a call describes: bounds that leave nothing, sequences longer than the bounds."""
import numpy as np
import pytest

from test_gpu_packed import MASKS, Case, raw_backward
from util import announce

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

if torch.cuda.is_available():
    import fv_sdpa


@pytest.mark.parametrize("keys", [9, 0])
def test_bounds_of_nothing(keys):
    """A padded buffer whose sequences are all empty: forward and backward run, and leave what they are given."""
    announce(f"9 rows, {keys} keys, no sequence with any")
    zeros = torch.zeros(3, dtype=torch.int32, device="cuda")
    batch = fv_sdpa.PackedSeqs(zeros, 0)
    q, dout = (torch.ones(9, 4, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    k, v = (torch.ones(keys, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    out = torch.full_like(q, 7.0)
    _, lse = fv_sdpa.packed_attention(q, k, v, batch, out=out, with_lse=True)
    grads = fv_sdpa.packed_attention_backward(dout, q, k, v, out, lse, batch)
    torch.cuda.synchronize()
    assert (out == 7).all() and [g.shape[0] for g in grads] == [9, keys, keys]


class Bounded(Case):
    """Of sequences longer than max_q rows or max_k keys the first ones, at the positions that they have in the whole."""

    def __init__(self, seqs, heads, mask, max_q, max_k, **kw):
        super().__init__(seqs, *heads, mask, **kw)
        self.batch = fv_sdpa.PackedSeqs(self.batch.q_start, max_q, self.batch.k_start, max_k)

    def heads_of(self):
        for rows, keys, h, y, seen in super().heads_of():
            a, b = min(rows.stop - rows.start, self.batch.max_q), min(keys.stop - keys.start, self.batch.max_k)
            yield slice(rows.start, rows.start + a), slice(keys.start, keys.start + b), h, y, seen[:a, :b]

    def left_out(self):
        """Of all rows, of all keys: those that no sequence's bounds hold."""
        rest = [np.ones(self.nq, dtype=bool), np.ones(self.nk, dtype=bool)]
        for rows, keys, *_ in self.heads_of():
            rest[0][rows] = rest[1][keys] = False
        return [torch.from_numpy(x).cuda() for x in rest]


@pytest.mark.parametrize("heads", [(6, 2, 64), (5, 1, 128)], ids=str)
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("bounds", [(200, 300), (300, 100), (5, 90), (130, 130)], ids=str)
def test_sequences_longer_than_the_bounds(bounds, mask, heads):
    """(The result in f32: rows that see one of the kept keys alone, whose gradient is nothing, would else have the rounding of the result in it.)"""
    tag = f"bounds {bounds} {mask} {heads}"
    announce(tag)
    c = Bounded([(300, 300), (10, 500), (64, 64), (150, 40)], heads, MASKS[mask], *bounds, seed=21)
    out = torch.full((c.nq, c.heads, c.d), 7.0, device="cuda")
    _, lse = fv_sdpa.packed_attention(c.q, c.k, c.v, c.batch, out=out, out_bf16=False, with_lse=True, **c.how)
    torch.cuda.synchronize()
    rows, keys = c.left_out()
    assert (out[rows] == 7).all()
    c.check_forward(out, lse, tag, out_bf16=False)
    grads = fv_sdpa.packed_attention_backward(c.dout, c.q, c.k, c.v, out, lse, c.batch, **c.how)
    torch.cuda.synchronize()
    for x, rest in zip(grads, (rows, keys, keys)):
        x[rest] = 0       # (not written, and no gradient of the plain form)
    c.check_backward(out, lse, grads, tag)


def test_rows_and_keys_past_the_bounds_are_left():
    c = Bounded([(300, 300), (10, 500)], (4, 2, 128), MASKS["causal"], 130, 200, seed=22)
    announce("gradients into given tensors")
    out, lse = fv_sdpa.packed_attention(c.q, c.k, c.v, c.batch, with_lse=True)
    grads = [torch.full_like(x, 7.0) for x in (c.dout, c.k.contiguous(), c.k.contiguous())]
    assert raw_backward(c, out, lse, *grads)[0] == 0
    torch.cuda.synchronize()
    rows, keys = c.left_out()
    for x, rest in zip(grads, (rows, keys, keys)):
        assert (x[rest] == 7).all() and torch.isfinite(x).all()


def test_heads_of_no_channels():
    """Refused by the library, as every head dim but 64 and 128 is."""
    none = torch.zeros(5, 2, 0, dtype=torch.bfloat16, device="cuda")
    starts = torch.tensor([0, 5], dtype=torch.int32, device="cuda")
    lse = torch.zeros(5, 2, device="cuda")
    for call in (lambda: fv_sdpa.packed_attention(none, none, none, fv_sdpa.PackedSeqs(starts, 5)),
                 lambda: fv_sdpa.packed_attention_backward(none, none, none, none, none, lse, fv_sdpa.PackedSeqs(starts, 5))):
        with pytest.raises(fv_sdpa.FvDeclined, match="head dim"):
            call()
