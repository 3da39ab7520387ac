"""Packed sequences at the borders of what a call describes: bounds that leave nothing."""
import pytest

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
