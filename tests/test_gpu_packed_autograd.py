"""The packed calls beside torch's autograd: they record no graph, so a gradient asked for through their results is an error, and what they write into
tensors of the caller's is known to have changed."""
import pytest

import util  # noqa: F401  (puts the package on the path)
from util import announce

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

if torch.cuda.is_available():
    import fv_sdpa


def make(requires_grad=False):
    gen = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(40, h, 64, device="cuda", generator=gen).bfloat16().requires_grad_(requires_grad) for h in (4, 2, 2))
    starts = torch.tensor([0, 13, 40], dtype=torch.int32, device="cuda")
    return q, k, v, fv_sdpa.PackedSeqs(starts, 27), torch.arange(40, dtype=torch.int32, device="cuda"), fv_sdpa.Rope(64)


def refused(t):
    with pytest.raises(RuntimeError, match="records no graph"):
        t.float().sum().backward()


def test_watched_tensors():
    """The same results as without autograd; a gradient through each of them is refused."""
    announce("watched tensors")
    q, k, v, seqs, positions, rope = make()
    want = fv_sdpa.packed_attention(q, k, v, seqs, with_lse=True)
    turned = fv_sdpa.rope_tokens(rope, positions, q, k)
    for which in range(3):
        watched = [x.detach().requires_grad_(i == which) for i, x in enumerate((q, k, v))]
        got = fv_sdpa.packed_attention(*watched, seqs, with_lse=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        for x in got:
            refused(x)
        refused(fv_sdpa.packed_attention(*watched, seqs))
        held = torch.empty_like(want[0])
        assert fv_sdpa.packed_attention(*watched, seqs, out=held) is held and torch.equal(held, want[0])
        refused(held)
        if which < 2:
            got = fv_sdpa.rope_tokens(rope, positions, *watched[:2])
            assert all(torch.equal(a, b) for a, b in zip(got, turned))
            for x in got:
                refused(x)
    refused(fv_sdpa.rope_tokens(rope, positions, q.detach().requires_grad_()))


def test_gradients_of_gradients():
    announce("gradients of gradients")
    q, k, v, seqs, _, _ = make()
    out, lse = fv_sdpa.packed_attention(q, k, v, seqs, with_lse=True)
    dout = torch.ones_like(out)
    want = fv_sdpa.packed_attention_backward(dout, q, k, v, out, lse, seqs)
    got = fv_sdpa.packed_attention_backward(dout.clone().requires_grad_(), q, k, v, out, lse, seqs)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for x in got:
        refused(x)
    # a function's own way back (the leaves are watched, the gradient is not): plain tensors
    q, k, v, *_ = make(requires_grad=True)
    assert not any(x.requires_grad for x in fv_sdpa.packed_attention_backward(dout, q, k, v, out, lse, seqs))


def test_without_autograd_nothing_is_recorded():
    announce("no_grad and inference_mode")
    q, k, v, seqs, positions, rope = make(requires_grad=True)
    for off in (torch.no_grad, torch.inference_mode):
        with off():
            out, lse = fv_sdpa.packed_attention(q, k, v, seqs, out=torch.empty_like(q), with_lse=True)
            turned = fv_sdpa.rope_tokens(rope, positions, q, k)
            fv_sdpa.rope_tokens(rope, positions, *turned, in_place=True)
            assert not any(x.requires_grad for x in (out, lse, *turned))


def test_written_tensors():
    """In place over watched tensors: refused. Over others, and into `out`: a tensor that was saved for a gradient is known to be another."""
    announce("written tensors")
    q, k, v, seqs, positions, rope = make()
    for i in range(2):
        watched = [x.detach().requires_grad_(i == j) * 1 for j, x in enumerate((q, k))]   # (no leaves)
        before = [x.detach().clone() for x in watched]
        with pytest.raises(ValueError, match="in place"):
            fv_sdpa.rope_tokens(rope, positions, *watched, in_place=True)
        assert all(torch.equal(a, b) for a, b in zip(watched, before))

    def turn(saved):
        fv_sdpa.rope_tokens(rope, positions, saved, in_place=True)

    def turn_second(saved):
        fv_sdpa.rope_tokens(rope, positions, q.clone(), saved, in_place=True)

    def attend(saved):
        fv_sdpa.packed_attention(q, k, v, seqs, out=saved)

    for write in (turn, turn_second, attend):
        w = torch.ones((), device="cuda", dtype=torch.bfloat16, requires_grad=True)
        saved = torch.randn_like(q)
        loss = (w * saved).sum()          # (the product keeps `saved` for w's gradient)
        write(saved)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
