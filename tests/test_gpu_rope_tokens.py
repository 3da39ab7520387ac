"""Rotary positions without tables against the definition in extended precision: both pairings, part of the head, scaled frequencies, far
positions, several axes, both ways, types, strides; and the run of a training step, rotation to rotation."""
import numpy as np
import pytest

import util  # noqa: F401  (puts the package on the path)
import packed_util as pu
from util import announce

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

if torch.cuda.is_available():
    import fv_sdpa

SCALINGS = [None, ("linear", 4.0), ("base", 8.0), ("parts", 8.0, 8192, 1.0, 32.0)]


def positions_of(rope, positions):
    """[tokens, pairs]: the position that each pair goes by."""
    p = positions.cpu().numpy().reshape(len(positions), -1)
    return p[:, [a for a, n in enumerate(rope.axes) for _ in range(n)]]


def check(rope, x, y, positions, theta, inverse, out_bf16, tag):
    """Each output within the sines' error, 2^-22 of the pair's magnitudes (angle: 2^-33 turns of frequency and 2^-24 of an eighth turn in f32; the
    series 2^-24; two products and a sum in f32), and half a step."""
    got, xin = y.double().cpu().numpy(), x.double().cpu().numpy()
    want = pu.rotate(xin, positions_of(rope, positions), theta, rope.halves, rope.amplitude, inverse)
    n = len(theta)
    mag = np.zeros_like(want)
    a, b = (np.abs(xin[..., :n]), np.abs(xin[..., n:2 * n])) if rope.halves else (np.abs(xin[..., 0:2 * n:2]), np.abs(xin[..., 1:2 * n:2]))
    m = (a + b) * rope.amplitude
    if rope.halves:
        mag[..., :n] = mag[..., n:2 * n] = m
    else:
        mag[..., 0:2 * n:2] = mag[..., 1:2 * n:2] = m
    bound = mag * 2.0 ** -22 + np.abs(want) * (pu.BF16_HALF if out_bf16 else pu.F32_HALF) * (1 + 2.0 ** -10) + 1e-30
    worst = (np.abs(got - want) / bound).max()
    print(f"[rope] {tag}: {worst:.3f} of the bound", flush=True)
    assert worst <= 1, (tag, worst)
    if not out_bf16 or x.dtype is torch.bfloat16:
        rest = slice(2 * n, None)
        assert (got[..., rest] == xin[..., rest]).all(), tag


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("scaling", SCALINGS, ids=str)
@pytest.mark.parametrize("d,rot,heads,kvh", [(128, 128, 4, 2), (128, 64, 5, 1), (64, 64, 3, 3), (80, 16, 2, 1), (96, 48, 1, 1), (256, 256, 2, 2)])
def test_against_the_definition(d, rot, heads, kvh, scaling, halves):
    announce(f"{d} {rot} {heads} {kvh} {scaling} {halves}")
    rope = fv_sdpa.Rope(d, rot=rot, halves=halves, scaling=scaling, amplitude=1.25)
    theta = pu.frequencies(rot // 2, 10000.0, scaling)
    gen = torch.Generator().manual_seed(d + rot)
    positions = torch.cat((torch.arange(20), torch.tensor([8191, 8192, 131071, 10_000_019, 2**31 - 1, -1, -77, -2**31]))).to(torch.int32).cuda()
    n = len(positions)
    for in16 in (True, False):
        wide = torch.randn(n, heads + kvh + 1, d, generator=gen).to(torch.bfloat16 if in16 else torch.float32).cuda()
        q, k = wide[:, :heads], wide[:, heads:heads + kvh]
        for out16 in (True, False):
            for inverse in (False, True):
                qo, ko = fv_sdpa.rope_tokens(rope, positions, q, k, inverse=inverse, out_bf16=out16)
                assert qo.is_contiguous() and qo.dtype is (torch.bfloat16 if out16 else torch.float32)
                check(rope, q, qo, positions, theta, inverse, out16, f"q in16 {in16} out16 {out16} inverse {inverse}")
                check(rope, k, ko, positions, theta, inverse, out16, f"k in16 {in16} out16 {out16} inverse {inverse}")
        alone = fv_sdpa.rope_tokens(rope, positions, q)
        both = fv_sdpa.rope_tokens(rope, positions, q, k)
        assert torch.equal(alone, both[0])
        # in place, strided, the neighbours left as they were
        copy = wide.clone()
        got = fv_sdpa.rope_tokens(rope, positions, copy[:, :heads], copy[:, heads:heads + kvh], in_place=True)
        assert got[0].data_ptr() == copy.data_ptr() and torch.equal(copy[:, :heads], both[0]) and torch.equal(copy[:, heads:heads + kvh], both[1])
        assert torch.equal(copy[:, -1], wide[:, -1])


def test_axes():
    """A video's frame, row and column, each a rotation of its own."""
    axes, d = (22, 21, 21), 128
    rope = fv_sdpa.Rope(d, axes=axes)
    theta = np.concatenate([pu.frequencies(n) for n in axes])
    t = torch.arange(3000, dtype=torch.int32, device="cuda")
    positions = torch.stack((t // 1560, t % 1560 // 52, t % 52), 1).contiguous()
    q = torch.randn(3000, 3, d, device="cuda")
    announce("axes")
    out = fv_sdpa.rope_tokens(rope, positions, q)
    check(rope, q, out, positions, theta, False, False, "axes")
    back = fv_sdpa.rope_tokens(rope, positions, out, inverse=True)
    assert (back - q).abs().max() <= 2.0 ** -20 * q.abs().max()     # twice the bound of one way, on pairs


def test_frequencies():
    """The turns of the host's table, to half a unit; the scaled ones' defining properties."""
    for scaling in SCALINGS:
        for n, base in ((64, 10000.0), (8, 500000.0)):
            rope = fv_sdpa.Rope(2 * n, base=base, scaling=scaling)
            got = np.array([int(x) for x in rope.turns], dtype=np.float64) / 2.0 ** 64 * (2 * np.pi)
            want = np.asarray(pu.frequencies(n, base, scaling), dtype=np.float64)
            # a whole number of 2^-64 turns is off by half of one, 2^-65 turns (of a pair that makes 2^-23 turns a position that is 2^-42 of it); what is
            # compared here goes through doubles, a few roundings of 2^-53
            assert (np.abs(got - want) / (2 * np.pi) <= 2.0 ** -65 + 8 * 2.0 ** -53 * want / (2 * np.pi)).all()
    plain, far = (np.array(fv_sdpa.Rope(128, scaling=s).turns, dtype=np.float64) for s in (None, ("base", 8.0)))
    assert plain[0] == far[0] and abs(plain[-1] / far[-1] - 8) < 1e-12     # (half units of numbers of 2^48: 2^-46 of the ratio)


def test_many_tokens():
    """Whole launches of many blocks, few heads and many, against one another."""
    rope = fv_sdpa.Rope(128, halves=True)
    n = 40_001
    q = torch.randn(n, 17, 128, device="cuda").bfloat16()
    positions = torch.randint(0, 100_000, (n,), device="cuda", dtype=torch.int32)
    announce("many tokens")
    whole = fv_sdpa.rope_tokens(rope, positions, q)
    for part in (slice(0, 1), slice(1, 40), slice(17_000, 17_333), slice(n - 1, n)):
        for heads in (slice(0, 1), slice(3, 17)):
            assert torch.equal(fv_sdpa.rope_tokens(rope, positions[part], q[part, heads]), whole[part, heads])


def test_refusals():
    rope = fv_sdpa.Rope(128)
    q, k, p = torch.zeros(4, 2, 128, device="cuda"), torch.zeros(4, 1, 128, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    for call in (lambda: fv_sdpa.rope_tokens(rope, p.long(), q), lambda: fv_sdpa.rope_tokens(rope, p[:3], q), lambda: fv_sdpa.rope_tokens(rope, p.cpu(), q),
                 lambda: fv_sdpa.rope_tokens(rope, p, q.half()), lambda: fv_sdpa.rope_tokens(rope, p, q, k.bfloat16()), lambda: fv_sdpa.rope_tokens(rope, p, q[..., :64]),
                 lambda: fv_sdpa.rope_tokens(rope, p, q, k[:3]), lambda: fv_sdpa.rope_tokens(rope, p, q, in_place=True, out_bf16=True),
                 lambda: fv_sdpa.rope_tokens(rope, p, q.transpose(0, 1)), lambda: fv_sdpa.rope_tokens(rope, torch.stack((p, p), 1), q),
                 lambda: fv_sdpa.Rope(128, rot=24), lambda: fv_sdpa.Rope(128, rot=160), lambda: fv_sdpa.Rope(128, axes=(32, 33)),
                 lambda: fv_sdpa.Rope(128, scaling=("spline", 2.0)), lambda: fv_sdpa.Rope(128, scaling=("parts", 2.0)), lambda: fv_sdpa.Rope(128, axes=(16, 16, 16, 8, 8))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(fv_sdpa.FvError, match="factor"):
        fv_sdpa.Rope(128, scaling=("linear", 0.5))
    assert fv_sdpa.rope_tokens(rope, p[:0], q[:0]).shape == (0, 2, 128)


class Attend(torch.autograd.Function if torch.cuda.is_available() else object):
    """As a training program wraps the calls."""

    @staticmethod
    def forward(ctx, q, k, v, seqs, mask):
        out, lse = fv_sdpa.packed_attention(q, k, v, seqs, mask=mask, with_lse=True)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.seqs, ctx.mask = seqs, mask
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse = ctx.saved_tensors
        return (*fv_sdpa.packed_attention_backward(dout.contiguous(), q, k, v, out, lse, ctx.seqs, mask=ctx.mask), None, None)


class Turn(torch.autograd.Function if torch.cuda.is_available() else object):
    @staticmethod
    def forward(ctx, q, k, rope, positions):
        ctx.rope, ctx.positions = rope, positions
        return fv_sdpa.rope_tokens(rope, positions, q, k)

    @staticmethod
    def backward(ctx, dq, dk):
        return (*fv_sdpa.rope_tokens(ctx.rope, ctx.positions, dq.contiguous(), dk.contiguous(), inverse=True), None, None)


def test_a_training_step():
    """Projection, rotation, attention under a window, loss, and the way back through torch's autograd, against the same in 64 bits on the host: each
    gradient off by a few roundings to bf16 of what it is made from (relative to its norm: q, k, out, dout, P and dS, dq and its rotation, the
    projection's operands; each 2^-9.. 2^-8 at most, independent, ten of them: 10 * 2^-8 at the very worst)."""
    heads, kvh, d, width = 4, 2, 64, 96
    lens = [70, 1, 33]
    n = sum(lens)
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(n, width, generator=gen).bfloat16()
    w = (torch.randn((heads + 2 * kvh) * d, width, generator=gen) / width ** 0.5).bfloat16()
    target = torch.randn(n, heads * d, generator=gen).bfloat16()
    starts = np.concatenate([[0], np.cumsum(lens)])
    pos = torch.cat([torch.arange(m) for m in lens]).to(torch.int32)
    mask = fv_sdpa.BlockCausal(1, 20, 2)

    xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    rope = fv_sdpa.Rope(d, halves=True)
    seqs = fv_sdpa.PackedSeqs(torch.tensor(starts, dtype=torch.int32, device="cuda"), max(lens))
    announce("a training step")
    qkv = (xg @ wg.t()).unflatten(1, (-1, d))
    q, k = Turn.apply(qkv[:, :heads].contiguous(), qkv[:, heads:heads + kvh].contiguous(), rope, pos.cuda())
    out = Attend.apply(q, k, qkv[:, heads + kvh:].contiguous(), seqs, mask)
    (out.flatten(1).float() * target.cuda().float()).sum().backward()
    torch.cuda.synchronize()

    x64, w64 = x.double().requires_grad_(), w.double().requires_grad_()
    qkv = (x64 @ w64.t()).unflatten(1, (-1, d))
    theta = torch.from_numpy(np.asarray(pu.frequencies(d // 2), dtype=np.float64))
    angle = (pos.double()[:, None] * theta)[:, None]
    turn = lambda t: torch.cat((t[..., :d // 2] * angle.cos() - t[..., d // 2:] * angle.sin(), t[..., :d // 2] * angle.sin() + t[..., d // 2:] * angle.cos()), -1)  # noqa: E731
    q, k, v = turn(qkv[:, :heads]), turn(qkv[:, heads:heads + kvh]), qkv[:, heads + kvh:]
    total = 0.0
    for s, m in enumerate(lens):
        at = slice(int(starts[s]), int(starts[s + 1]))
        seen = torch.from_numpy(pu.visible(m, m, True, 1, 20, 2))
        for h in range(heads):
            y = h * kvh // heads
            p = torch.softmax((q[at, h] @ k[at, y].t() / d ** 0.5).masked_fill(~seen, -np.inf), -1)
            total = total + (p @ v[at, y] * target.double()[at, h * d:(h + 1) * d]).sum()
    total.backward()
    for name, a, b in (("x", xg.grad, x64.grad), ("w", wg.grad, w64.grad)):
        rel = float((a.double().cpu() - b).norm() / b.norm())
        print(f"[rope] training step, gradient of {name}: {rel:.5f}", flush=True)
        assert rel <= 10 * 2.0 ** -8
