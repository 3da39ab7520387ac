"""Attention over packed sequences and its gradients against their definitions in 64 bits, at lengths and masks where a kernel can go
wrong; strides, types, what lies outside the sequences, streams, graphs."""
import copy

import numpy as np
import pytest

import packed_util as pu
from util import announce

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

if torch.cuda.is_available():
    import fv_sdpa

SEQS = {   # (rows, keys) of each sequence
    "one": [(1, 1)],
    "short": [(1, 1), (0, 0), (7, 7), (64, 64), (31, 31), (2, 2)],
    "tails": [(127, 127), (129, 129), (33, 33), (65, 65)],
    "long": [(700, 700), (5, 5), (321, 321)],
    "cross": [(200, 77), (3, 130), (90, 1), (0, 40), (40, 0), (129, 64)],     # causal: rows before the first key, sequences without rows or keys
    "ends": [(1, 1500), (5, 999), (17, 64)],
}
MASKS = {   # causal, block, window, sink
    "full": (False, 1, 0, 0),
    "causal": (True, 1, 0, 0),
    "window": (True, 1, 37, 3),
    "band": (True, 1, 64, 0),
    "blocks": (True, 48, 0, 0),
    "block_window": (True, 20, 2, 1),
    "sinks": (True, 1, 5, 100),
}
HEADS = [(2, 2, 128), (6, 2, 64), (5, 1, 128), (3, 3, 64), (16, 2, 128)]


class Case:
    def __init__(self, seqs, heads, kvh, d, mask, seed=0, lead=3, trail=5, sharp=1.0, fused=True):
        self.seqs, self.heads, self.kvh, self.d = seqs, heads, kvh, d
        self.causal, self.block, self.window, self.sink = mask
        rng = np.random.Generator(np.random.PCG64(seed))
        self.q0 = np.concatenate([[0], np.cumsum([a for a, _ in seqs])]) + lead
        self.k0 = np.concatenate([[0], np.cumsum([b for _, b in seqs])]) + lead
        self.nq, self.nk = int(self.q0[-1]) + trail, int(self.k0[-1]) + trail
        outside = [np.array([not (lead <= i < n - trail) for i in range(n)]) for n in (self.nq, self.nk)]

        def make(n, h, out, scale=1.0):   # rows of no sequence hold anything
            x = torch.from_numpy((rng.standard_normal((n, h, d)) * scale).astype(np.float32)).bfloat16()
            x[torch.from_numpy(out)] = float("nan")
            return x

        q, k, v = make(self.nq, heads, outside[0], sharp), make(self.nk, kvh, outside[1]), make(self.nk, kvh, outside[1])
        self.dout = make(self.nq, heads, outside[0])
        self.np = [x.double().numpy() for x in (q, k, v, self.dout)]
        kv = torch.cat((k, v), 1).cuda()             # tokens of k and v lie apart
        self.q, self.k, self.v, self.dout = q.cuda(), kv[:, :kvh], kv[:, kvh:], self.dout.cuda()
        if fused:
            wide = torch.cat((q, q), 1).cuda()
            self.q = wide[:, heads:]
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        self.batch = fv_sdpa.PackedSeqs(i32(self.q0), max(a for a, _ in seqs), i32(self.k0), max(b for _, b in seqs))
        self.how = {"causal": self.causal, "mask": fv_sdpa.BlockCausal(self.block, self.window, self.sink) if self.causal and (self.block, self.window, self.sink) != (1, 0, 0) else None}
        self.scale = 1.0 / np.sqrt(d)

    def few(self):
        """Rows that see up to so many keys have their sum of p dp made from these (where no row sees more than 64)."""
        band = (self.window + self.sink) * self.block if self.causal and self.window else 1 << 40
        return 8 if min(self.batch.max_k, self.nk, band) <= 64 else 0

    def heads_of(self):
        """(rows, keys, head, key head, mask) of every head of every sequence."""
        for s, (a, b) in enumerate(self.seqs):
            seen = pu.visible(a, b, self.causal, self.block, self.window, self.sink)
            for h in range(self.heads):
                yield slice(self.q0[s], self.q0[s + 1]), slice(self.k0[s], self.k0[s + 1]), h, h * self.kvh // self.heads, seen

    def check_forward(self, out, lse, tag, out_bf16=True):
        q, k, v, _ = self.np
        o, l = out.double().cpu().numpy(), lse.double().cpu().numpy()
        worst = 0.0
        for rows, keys, h, y, seen in self.heads_of():
            want, want_l, bound, bound_l = pu.attention(q[rows, h], k[keys, y], v[keys, y], seen, self.scale, out_bf16)
            got, got_l = o[rows, h], l[rows, h]
            assert np.isfinite(got).all(), f"{tag}: not finite, head {h}"
            none = np.isneginf(want_l)
            assert np.array_equal(none, np.isneginf(got_l)), f"{tag}: rows without a key, head {h}"
            assert (got[none] == 0).all(), f"{tag}: rows without a key, head {h}"
            d = np.abs(got - want) / bound
            dl = np.abs(got_l[~none] - want_l[~none]) / bound_l[~none]
            worst = max(worst, d.max(initial=0.0), dl.max(initial=0.0))
            assert d.max(initial=0.0) <= 1, f"{tag}: head {h} rows {rows}: {d.max()} of the bound at {np.unravel_index(d.argmax(), d.shape)}"
            assert dl.max(initial=0.0) <= 1, f"{tag}: lse, head {h} rows {rows}: {dl.max()} of the bound"
        print(f"[packed] {tag}: {worst:.3f} of the bound", flush=True)

    def check_backward(self, out, lse, grads, tag, bf16=True, dout=None):
        q, k, v, g = self.np
        g = g if dout is None else dout
        o, l = out.double().cpu().numpy(), lse.double().cpu().numpy()
        dq, dk, dv = (np.zeros((n, h, self.d)) for n, h in ((self.nq, self.heads), (self.nk, self.kvh), (self.nk, self.kvh)))
        bq, bk, bv = np.zeros_like(dq), np.zeros_like(dk), np.zeros_like(dv)
        for rows, keys, h, y, seen in self.heads_of():
            r = pu.gradients(q[rows, h], k[keys, y], v[keys, y], g[rows, h], o[rows, h], l[rows, h], seen, self.scale, self.few())
            dq[rows, h], bq[rows, h] = r[0], r[3]
            for to, x in ((dk, r[1]), (dv, r[2]), (bk, r[4]), (bv, r[5])):
                to[keys, y] += x
        inside = [slice(self.q0[0], self.q0[-1]), slice(self.k0[0], self.k0[-1]), slice(self.k0[0], self.k0[-1])]
        for name, got, want, bound, at in zip(("dq", "dk", "dv"), grads, (dq, dk, dv), (bq, bk, bv), inside):
            got, want, bound = got.double().cpu().numpy()[at], want[at], bound[at]
            assert np.isfinite(got).all(), f"{tag}: {name} not finite"
            x = np.abs(got - want) / (bound + (pu.BF16_HALF if bf16 else pu.F32_HALF) * np.abs(want) + 1e-30)
            print(f"[packed] {tag}: {name} {x.max(initial=0.0):.3f} of the bound", flush=True)
            assert x.max(initial=0.0) <= 1, f"{tag}: {name} {x.max()} of the bound at {np.unravel_index(x.argmax(), x.shape)}"


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("seqs", SEQS)
@pytest.mark.parametrize("heads", HEADS[:3], ids=str)
def test_against_64_bits(seqs, mask, heads):
    tag = f"{seqs} {mask} {heads}"
    announce(tag)
    c = Case(SEQS[seqs], *heads, MASKS[mask], seed=len(seqs))
    out, lse = fv_sdpa.packed_attention(c.q, c.k, c.v, c.batch, with_lse=True, **c.how)
    torch.cuda.synchronize()
    c.check_forward(out, lse, tag)
    announce(tag + " backward")
    grads = fv_sdpa.packed_attention_backward(c.dout, c.q, c.k, c.v, out, lse, c.batch, **c.how)
    torch.cuda.synchronize()
    c.check_backward(out, lse, grads, tag)


@pytest.mark.parametrize("heads", [HEADS[1], HEADS[2]], ids=str)
def test_many_sequences(heads):
    """More than a wave's lanes have starts, some without rows, some without keys."""
    rng = np.random.Generator(np.random.PCG64(31))
    counts = [(int(a), int(a + b)) for a, b in zip(rng.integers(0, 50, 150), rng.integers(-20, 20, 150).clip(0))]
    announce(f"150 sequences, {heads}")
    for mask in ("causal", "full"):
        c = Case(counts, *heads, MASKS[mask], seed=8)
        out, lse, grads = run_both(c)
        c.check_forward(out, lse, f"150 sequences {mask}")
        c.check_backward(out, lse, grads, f"150 sequences {mask} backward")


def test_starts_outside_the_tensors():
    """Starts are bounded to the tensors: the same bits as from starts that end with them."""
    c = Case([(90, 90), (310, 310), (205, 205)], 6, 2, 64, MASKS["causal"], seed=10, lead=0, trail=0)
    announce("starts before and behind the tensors")
    out, lse, grads = run_both(c)
    starts = torch.tensor([-7, 90, 400, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    c.batch = fv_sdpa.PackedSeqs(starts, 310)
    again, lse2, grads2 = run_both(c)
    torch.cuda.synchronize()
    assert torch.equal(out, again) and torch.equal(lse, lse2) and all(torch.equal(a, b) for a, b in zip(grads, grads2))


def run_both(c, **kw):
    out, lse = fv_sdpa.packed_attention(c.q, c.k, c.v, c.batch, with_lse=True, **c.how)
    return out, lse, fv_sdpa.packed_attention_backward(c.dout, c.q, c.k, c.v, out, lse, c.batch, **c.how, **kw)


@pytest.mark.parametrize("heads,seqs,mask", [(HEADS[3], "tails", "causal"), (HEADS[3], "cross", "full"), (HEADS[4], "long", "window"), (HEADS[4], "short", "blocks")], ids=str)
def test_more_heads(heads, seqs, mask):
    announce(f"{heads} {seqs} {mask}")
    c = Case(SEQS[seqs], *heads, MASKS[mask], seed=7)
    out, lse, grads = run_both(c)
    c.check_forward(out, lse, "forward")
    c.check_backward(out, lse, grads, "backward")


@pytest.mark.parametrize("seqs", ["long", "short"])
@pytest.mark.parametrize("d", [64, 128])
def test_types(d, seqs):
    """f32 results, f32 gradients in (rounded first) and out, each against the same bounds with its own rounding."""
    c = Case(SEQS[seqs], 4, 2, d, MASKS["causal"], seed=3)
    announce(f"f32 result, d {d}, {seqs}")
    out, lse = fv_sdpa.packed_attention(c.q, c.k, c.v, c.batch, out_bf16=False, with_lse=True)
    assert out.dtype is torch.float32
    c.check_forward(out, lse, "f32 result", out_bf16=False)
    out16, lse16 = fv_sdpa.packed_attention(c.q, c.k, c.v, c.batch, with_lse=True)
    inside = slice(int(c.q0[0]), int(c.q0[-1]))
    assert torch.equal(out16[inside], out[inside].bfloat16()) and torch.equal(lse16[inside], lse[inside])
    announce("f32 gradients")
    g32 = c.dout.float() * (1 + 2.0 ** -10)
    rounded = g32.bfloat16()
    assert not torch.equal(rounded[inside], g32[inside])
    grads = fv_sdpa.packed_attention_backward(g32, c.q, c.k, c.v, out, lse, c.batch, grads_bf16=False)
    assert all(g.dtype is torch.float32 for g in grads)
    c.check_backward(out, lse, grads, "f32 gradients", bf16=False, dout=rounded.double().cpu().numpy())
    same = fv_sdpa.packed_attention_backward(rounded, c.q, c.k, c.v, out, lse, c.batch, grads_bf16=True)
    for a, b, at in zip(same, grads, (inside, slice(int(c.k0[0]), int(c.k0[-1])), slice(int(c.k0[0]), int(c.k0[-1])))):
        assert torch.equal(a[at], b[at].bfloat16())


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 3.0, 50.0])
def test_scales(scale):
    """Nearly even weights to one key a row (and the pass with the running maximum)."""
    announce(f"scale {scale}")
    c = Case(SEQS["long"], 4, 2, 64, MASKS["causal"], seed=12)
    c.scale = scale
    out, lse = fv_sdpa.packed_attention(c.q, c.k, c.v, c.batch, scale=scale, with_lse=True)
    c.check_forward(out, lse, f"scale {scale}")
    grads = fv_sdpa.packed_attention_backward(c.dout, c.q, c.k, c.v, out, lse, c.batch, scale=scale)
    c.check_backward(out, lse, grads, f"scale {scale} backward")


@pytest.mark.parametrize("causal,block,window,sink,seqs", [
    (True, 1, 0, 0, [(1, 1)] * 9), (False, 1, 0, 0, [(7, 1), (130, 1)]), (True, 1, 1, 0, [(200, 200), (3, 40)]), (True, 4, 1, 0, [(65, 65), (1, 129)]),
    (True, 1, 1, 0, [(700, 500), (40, 900)])])
def test_rows_that_see_one_key(causal, block, window, sink, seqs):
    """Their scores have no gradient: exact zeros, and the values' gradient is that of the results."""
    announce(f"{causal} {block} {window} {sink} {seqs}")
    c = Case(seqs, 4, 2, 128, (causal, block, window, sink), seed=5)
    out, lse, (dq, dk, dv) = run_both(c)
    c.check_forward(out, lse, "forward")
    c.check_backward(out, lse, (dq, dk, dv), "backward")
    for rows, keys, h, y, seen in c.heads_of():
        one = seen.sum(1) == 1
        assert one.any() and (dq[rows, h].float().cpu().numpy()[one] == 0).all()
        alone = ~seen[~one].any(0)          # keys that no other row sees
        assert (dk[keys, y].float().cpu().numpy()[alone] == 0).all()


def test_second_pass():
    """Scores that grow along the keys by far more than the first tile's offset takes: the pass with the running maximum; a value that
    is not finite reaches the rows that see it and no other."""
    for d in (64, 128):
        announce(f"growing scores, d {d}")
        c = Case([(300, 300), (64, 700)], 4, 2, d, MASKS["causal"], seed=1, fused=False)
        ramp = torch.linspace(0, 40, c.nk, device="cuda")[:, None, None].bfloat16()
        k = (c.k * ramp).contiguous()
        q = (c.q.abs() + 1) * 2
        k[..., ::2] = k[..., ::2].abs()
        k[..., 1::2] = k[..., 1::2].abs()
        c.q, c.k, c.v = q.contiguous(), k, c.v.contiguous()
        c.np[0], c.np[1] = c.q.double().cpu().numpy(), c.k.double().cpu().numpy()
        out, lse = fv_sdpa.packed_attention(c.q, c.k, c.v, c.batch, with_lse=True)
        c.check_forward(out, lse, "growing scores")
        announce(f"values that are not finite, d {d}")
        for value in (float("nan"), float("inf")):
            v = c.v.clone()
            at = int(c.k0[0]) + 200
            v[at, 0, 5] = value
            again = fv_sdpa.packed_attention(c.q, c.k, v, c.batch)
            before, behind = slice(int(c.q0[0]), int(c.q0[0]) + 200), slice(int(c.q0[0]) + 200, int(c.q0[1]))
            assert torch.equal(again[before], out[before]), "rows before it"
            assert torch.equal(again[int(c.q0[1]):int(c.q0[2])], out[int(c.q0[1]):int(c.q0[2])]), "the other sequence"
            assert not torch.isfinite(again[behind, :2, 5]).any() and torch.isfinite(again[behind, 2:]).all()
        announce(f"a key that is not a number, d {d}")
        k = c.k.clone()
        k[at, 0, 5] = float("nan")
        again = fv_sdpa.packed_attention(c.q, k, c.v, c.batch)
        # (either pass is within a half step of its weights and one of its result: 2^-8 + 2^-8 of the largest value)
        room = 4 * pu.BF16_HALF * c.v[int(c.k0[0]):int(c.k0[-1])].abs().max()
        inside = slice(int(c.q0[1]), int(c.q0[2]))
        assert ((again[before].float() - out[before].float()).abs() <= room).all() and torch.equal(again[inside], out[inside])
        assert again[behind, :2].isnan().all() and torch.equal(again[behind, 2:], out[behind, 2:])


def raw_backward(c, out, lse, dq, dk, dv, starts=None, nbytes=None):
    """fv_packed_attention_backward into given tensors."""
    lib = fv_sdpa.lib()
    b = starts if starts is not None else c.batch
    n = b.q_start.shape[0] - 1
    m = (c.block, c.window, c.sink)
    numbers = (c.heads, c.kvh, c.d, n, c.nq, c.nk, b.max_q, b.max_k, int(c.causal), *m)
    need = lib.fv_packed_attention_backward_workspace_bytes(1, *numbers)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    rc = lib.fv_packed_attention_backward(
        c.dout.data_ptr(), 1, c.q.data_ptr(), c.q.stride(0), c.k.data_ptr(), c.k.stride(0), c.v.data_ptr(), c.v.stride(0), out.data_ptr(), 1, lse.data_ptr(),
        dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), 1, c.heads, c.kvh, c.d, b.q_start.data_ptr(), b.k_start.data_ptr(), n, c.nq, c.nk, b.max_q, b.max_k,
        c.scale, int(c.causal), *m, work.data_ptr(), need if nbytes is None else nbytes, st)
    return rc, work


def test_rows_outside_are_left():
    c = Case(SEQS["long"], 4, 2, 128, MASKS["causal"], seed=2)
    out = torch.full((c.nq, 4, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    _, lse = fv_sdpa.packed_attention(c.q, c.k, c.v, c.batch, out=out, with_lse=True)
    grads = [torch.full_like(x, 7.0) for x in (c.dout, c.k.contiguous(), c.k.contiguous())]
    rc, _ = raw_backward(c, out, lse, *grads)
    assert rc == 0
    torch.cuda.synchronize()
    for x, a, b in ((out, c.q0[0], c.q0[-1]), (grads[0], c.q0[0], c.q0[-1]), (grads[1], c.k0[0], c.k0[-1]), (grads[2], c.k0[0], c.k0[-1])):
        assert (x[:a] == 7).all() and (x[b:] == 7).all() and torch.isfinite(x[a:b]).all()
    c.check_backward(out, lse, grads, "into given tensors")


def test_far_tokens():
    """Tokens 32 KB apart, the second sequence past 4 GB."""
    tokens, wide, d = 150_000, 16384, 128
    base = torch.zeros(tokens, wide, dtype=torch.bfloat16, device="cuda")
    c = Case([(190, 190), (260, 260)], 4, 2, d, MASKS["causal"], seed=4, fused=False, lead=0, trail=0)
    at = [0, tokens - 260]
    rows = torch.cat([torch.arange(at[0], at[0] + 190), torch.arange(at[1], at[1] + 260)]).cuda()
    for i, x in enumerate((c.q, c.k, c.v)):
        base.view(tokens, wide)[rows, i * 1024:i * 1024 + x.shape[1] * d] = x.reshape(len(rows), -1)
    q, k, v = (base[:, i * 1024:i * 1024 + h * d].unflatten(1, (h, d)) for i, h in enumerate((4, 2, 2)))
    batch = fv_sdpa.PackedSeqs(torch.tensor([tokens - 260, tokens], dtype=torch.int32, device="cuda"), 260)
    announce("past 4 GB, forward")
    out, lse = fv_sdpa.packed_attention(q, k, v, batch, with_lse=True)
    small, small_lse = fv_sdpa.packed_attention(c.q, c.k, c.v, c.batch, with_lse=True)
    torch.cuda.synchronize()
    assert torch.equal(out[tokens - 260:], small[190:]) and torch.equal(lse[tokens - 260:], small_lse[190:])
    announce("past 4 GB, backward")
    dout = torch.zeros(tokens, 4, d, dtype=torch.bfloat16, device="cuda")
    dout[tokens - 260:] = c.dout[190:]
    grads = fv_sdpa.packed_attention_backward(dout, q, k, v, out, lse, batch)
    want = fv_sdpa.packed_attention_backward(c.dout, c.q, c.k, c.v, small, small_lse, c.batch)
    torch.cuda.synchronize()
    for a, b in zip(grads, want):
        x, y = a[tokens - 260:].float(), b[190:].float()
        assert (x - y).abs().max() <= 2.0 ** -7 * y.abs().max()   # (cut elsewhere: other sums)


def test_the_same_bits_and_streams():
    c = Case(SEQS["long"], 6, 2, 64, MASKS["window"], seed=6)
    first = run_both(c)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for s in side:                     # two calls at once, each with its own workspace
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            results.append(run_both(c))
    torch.cuda.synchronize()
    ins, ks = slice(int(c.q0[0]), int(c.q0[-1])), slice(int(c.k0[0]), int(c.k0[-1]))
    for out, lse, grads in results:
        assert torch.equal(out[ins], first[0][ins]) and torch.equal(lse[ins], first[1][ins])
        for a, b, at in zip(grads, first[2], (ins, ks, ks)):
            assert torch.equal(a[at], b[at])


@pytest.mark.parametrize("most,batches", [
    (300, [[(300, 300), (1, 1), (77, 77), (0, 0)], [(10, 10), (300, 300), (129, 129), (64, 64)], [(0, 0), (0, 0), (5, 5), (33, 33)]]),
    (40, [[(40, 40), (1, 1), (7, 7), (0, 0)], [(3, 3), (2, 2), (40, 40), (5, 5)], [(0, 0), (0, 0), (5, 5), (33, 33)]])])
def test_a_captured_step_replays_with_other_lengths(most, batches):
    """Forward and backward captured once, replayed with other starts within the bounds, each replay against its own eager calls."""
    heads, kvh, d, n = 4, 2, 128, 4
    tokens = 520
    g = torch.Generator(device="cuda").manual_seed(11)
    q = torch.randn(tokens, heads, d, device="cuda", generator=g).bfloat16()
    k, v = (torch.randn(tokens, kvh, d, device="cuda", generator=g).bfloat16() for _ in range(2))
    dout = torch.randn(tokens, heads, d, device="cuda", generator=g).bfloat16()
    starts = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    batch = fv_sdpa.PackedSeqs(starts, most)

    def step():
        out, lse = fv_sdpa.packed_attention(q, k, v, batch, with_lse=True)
        return (out, *fv_sdpa.packed_attention_backward(dout, q, k, v, out, lse, batch))

    def lengths(b):
        starts.copy_(torch.tensor(np.concatenate([[0], np.cumsum([x for x, _ in b])]), dtype=torch.int32))
        return int(sum(x for x, _ in b))

    lengths(batches[0])
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for turn in range(2):
        for b in batches:
            m = lengths(b)
            graph.replay()
            torch.cuda.synchronize()
            want = step()
            torch.cuda.synchronize()
            for name, x, y in zip(("out", "dq", "dk", "dv"), held, want):
                assert torch.equal(x[:m], y[:m]), (turn, b, name)


def test_gradients_against_differences():
    """Along the gradients themselves and along them with random parts left out: the change of sum(out dout) in 64 bits by the gradients,
    within their bounds (which say more than nothing: less than the change itself)."""
    c = Case([(90, 90), (40, 120)], 4, 2, 64, MASKS["window"], seed=9, lead=0, trail=0)
    out, lse, grads = run_both(c, grads_bf16=False)
    torch.cuda.synchronize()
    q, k, v, g = c.np
    rng = np.random.Generator(np.random.PCG64(1))

    def loss(q, k, v):
        return sum((pu.attention(q[r, h], k[s, y], v[s, y], seen, c.scale, False)[0] * g[r, h]).sum() for r, s, h, y, seen in c.heads_of())

    got = [x.double().cpu().numpy() for x in grads]
    bound = [np.zeros_like(x) for x in got]
    for r, s, h, y, seen in c.heads_of():
        b = pu.gradients(q[r, h], k[s, y], v[s, y], g[r, h], out.double().cpu().numpy()[r, h], lse.double().cpu().numpy()[r, h], seen, c.scale, c.few())
        # the given result is rounded to bf16: dP - D is off by its half step's part
        off = (np.abs(g[r, h]) * np.abs(out.double().cpu().numpy()[r, h])).sum(1, keepdims=True) * pu.BF16_HALF
        p = np.where(seen, np.exp(np.where(seen, q[r, h] @ k[s, y].T, 0) * c.scale - lse.double().cpu().numpy()[r, h][:, None]), 0)
        bound[0][r, h] += b[3] + (p * off) @ np.abs(k[s, y]) * c.scale
        bound[1][s, y] += b[4] + (p * off).T @ np.abs(q[r, h]) * c.scale
        bound[2][s, y] += b[5]
    for turn in range(3):
        u = [x if turn == 0 else x * rng.integers(0, 2, x.shape) for x in got]
        e = 1e-5
        diff = (loss(*(x + e * y for x, y in zip((q, k, v), u))) - loss(*(x - e * y for x, y in zip((q, k, v), u)))) / (2 * e)
        along = sum((a * b).sum() for a, b in zip(got, u))
        room = sum((a * np.abs(b)).sum() for a, b in zip(bound, u))
        print(f"[packed] along a direction: {along:.6f}, by differences {diff:.6f}, room {room:.4f}", flush=True)
        # (the differences' own error: third derivatives times e^2, 1e-6 of the change and less)
        assert abs(along - diff) <= room + 1e-6 * abs(diff) and room < abs(diff)


def test_refusals():
    c = Case(SEQS["tails"], 4, 2, 128, MASKS["causal"])
    b = fv_sdpa.BlockCausal(1, 0, 0)
    f, back = fv_sdpa.packed_attention, fv_sdpa.packed_attention_backward
    out, lse = f(c.q, c.k, c.v, c.batch, with_lse=True)
    for call in (lambda: f(c.q.float(), c.k, c.v, c.batch), lambda: f(c.q, c.k[:, :1], c.v, c.batch), lambda: f(c.q, c.k[:-1], c.v, c.batch),
                 lambda: f(c.q, c.k, c.v, c.batch, mask=b, causal=False), lambda: f(c.q.cpu(), c.k, c.v, c.batch), lambda: f(c.q.transpose(0, 1), c.k, c.v, c.batch),
                 lambda: f(c.q[..., :64], c.k, c.v, c.batch), lambda: f(c.q, c.k, c.v, c.batch, out=out.float()), lambda: f(c.q[0], c.k, c.v, c.batch),
                 lambda: back(c.dout[:-1], c.q, c.k, c.v, out, lse, c.batch), lambda: back(c.dout.half(), c.q, c.k, c.v, out, lse, c.batch),
                 lambda: back(c.dout, c.q, c.k, c.v, out, lse.double(), c.batch), lambda: back(c.dout, c.q, c.k, c.v, out.transpose(0, 1), lse, c.batch),
                 lambda: fv_sdpa.PackedSeqs(c.batch.q_start.long(), 5), lambda: fv_sdpa.PackedSeqs(c.batch.q_start.cpu(), 5),
                 lambda: fv_sdpa.PackedSeqs(c.batch.q_start, -1), lambda: fv_sdpa.PackedSeqs(c.batch.q_start, 5, c.batch.k_start[:-1]),
                 lambda: fv_sdpa.PackedSeqs(c.batch.q_start[:0], 5)):
        with pytest.raises(ValueError):
            call()
    three = torch.zeros(c.nq, 3, 128, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(fv_sdpa.FvError, match="multiple of the key heads"):
        f(three, c.k, c.v, c.batch)
    odd = torch.zeros(c.nq, 4, 96, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(fv_sdpa.FvDeclined, match="head dim"):
        f(odd, odd[:, :2], odd[:, :2], c.batch)
    grads = [torch.zeros_like(c.dout) for _ in range(3)]
    assert raw_backward(c, out, lse, *grads, nbytes=100)[0] != 0 and "workspace too small" in fv_sdpa.lib().fv_sdpa_last_error().decode()
    twin = copy.deepcopy(c.batch)
    assert twin.q_start.data_ptr() != c.batch.q_start.data_ptr() and twin._args[0] == twin.q_start.data_ptr()


def test_empty_calls():
    e = lambda n, h: torch.zeros(n, h, 128, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    zeros = torch.zeros(3, dtype=torch.int32, device="cuda")
    batch = fv_sdpa.PackedSeqs(zeros, 0)
    out, lse = fv_sdpa.packed_attention(e(0, 4), e(0, 2), e(0, 2), batch, with_lse=True)
    grads = fv_sdpa.packed_attention_backward(e(0, 4), e(0, 4), e(0, 2), e(0, 2), out, lse, batch)
    assert out.shape == (0, 4, 128) and [g.shape[0] for g in grads] == [0, 0, 0]
    # rows without any key, keys without any row
    rows = fv_sdpa.PackedSeqs(torch.tensor([0, 5, 9], dtype=torch.int32, device="cuda"), 5, zeros, 0)
    out, lse = fv_sdpa.packed_attention(e(9, 4) + 1, e(0, 2), e(0, 2), rows, causal=False, with_lse=True)
    dq, dk, dv = fv_sdpa.packed_attention_backward(e(9, 4) + 1, e(9, 4) + 1, e(0, 2), e(0, 2), out, lse, rows, causal=False)
    torch.cuda.synchronize()
    assert (out == 0).all() and torch.isneginf(lse).all() and (dq == 0).all() and dk.shape[0] == 0
    keys = fv_sdpa.PackedSeqs(zeros, 0, torch.tensor([0, 5, 9], dtype=torch.int32, device="cuda"), 5)
    out, lse = fv_sdpa.packed_attention(e(0, 4), e(9, 2) + 1, e(9, 2) + 1, keys, causal=False, with_lse=True)
    dq, dk, dv = fv_sdpa.packed_attention_backward(e(0, 4), e(0, 4), e(9, 2) + 1, e(9, 2) + 1, out, lse, keys, causal=False)
    torch.cuda.synchronize()
    assert dq.shape[0] == 0 and (dk == 0).all() and (dv == 0).all()
