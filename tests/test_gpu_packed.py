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
            r = pu.gradients(q[rows, h], k[keys, y], v[keys, y], g[rows, h], o[rows, h], l[rows, h], seen, self.scale)
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
