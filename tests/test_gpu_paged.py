"""The paged KV cache on the device against plain numpy: what is stored bit for bit, attention against 64 bits."""
import numpy as np
import pytest

import paged_util as pu
from util import announce

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fv():
    import torch

    assert torch.cuda.is_available()
    import fv_sdpa

    fv_sdpa.lib()
    return fv_sdpa


class World:
    """A pool with a page table for sequences of the given lengths, and the batch of their last tokens. Host copies are
    kept by position: `held` is what every token of every sequence holds."""

    def __init__(self, fv, seed, lens, counts, kvh, d, page=16, four=False, spare=3, columns=None, max_q=None, max_len=None, fill="normal"):
        import torch

        self.fv, self.torch = fv, torch
        self.lens, self.counts, self.kvh, self.d, self.page, self.four = list(lens), list(counts), kvh, d, page, four
        rng = self.rng = np.random.Generator(np.random.PCG64(seed))
        need = [-(-n // page) for n in lens]
        self.pages = sum(need) + spare
        width = columns or max(max(need), 1)
        order = rng.permutation(self.pages)
        self.table = np.full((len(lens), width), -7, dtype=np.int32)     # entries that no call may follow
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        shape = (self.pages, kvh, page)
        if four:
            self.host = {n: rng.integers(0, 256, (*shape, d // 2), dtype=np.uint8) for n in "kv"}
            self.scales = {n: rng.integers(122, 129, (*shape, d // 32), dtype=np.uint8) for n in "kv"}
        else:
            self.host = {n: pu.bf16(rng.standard_normal((*shape, d))) for n in "kv"}
            self.scales = None
        if fill == "nan":      # whatever lies outside the sequences
            inside = np.zeros(shape[:1] + shape[2:], dtype=bool)
            for s, n in enumerate(lens):
                j = np.arange(n)
                inside[self.table[s, j // page], j % page] = True
            for n in "kv":
                for p, t in zip(*np.nonzero(~inside)):
                    if four:
                        self.scales[n][p, :, t] = 255
                    else:
                        self.host[n][p, :, t] = np.nan if (p + t) % 2 else np.inf
        self.push()
        self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.batch = fv.PagedBatch(self.dev(self.starts), self.dev(np.array(lens, dtype=np.int32)), self.dev(self.table),
                                   max(counts) if max_q is None else max_q, max(lens) if max_len is None else max_len)

    def dev(self, x):
        return self.torch.from_numpy(np.ascontiguousarray(x)).cuda()

    def push(self):
        if self.four:
            self.pool = self.fv.PagedKv(*(self.dev(self.host[n]) for n in "kv"), *(self.dev(self.scales[n]) for n in "kv"))
        else:
            self.pool = self.fv.PagedKv(*(self.dev(self.host[n]).to(self.torch.bfloat16) for n in "kv"))

    def pull(self):
        self.torch.cuda.synchronize()
        k, v = (t.float().cpu().numpy() if not self.four else t.cpu().numpy() for t in (self.pool.k, self.pool.v))
        s = (self.pool.k_scales.cpu().numpy(), self.pool.v_scales.cpu().numpy()) if self.four else (None, None)
        return {"k": k, "v": v}, {"k": s[0], "v": s[1]}

    def held(self, name, s):
        """f64 [len, kv_heads, d] of sequence s."""
        j = np.arange(self.lens[s])
        p, t = self.table[s, j // self.page], j % self.page
        ok = (p >= 0) & (p < self.pages)
        p = np.where(ok, p, 0)
        x = self.host[name][p, :, t]
        return pu.values4(x, self.scales[name][p, :, t]) if self.four else x.astype(np.float64)

    def usable(self, s):
        p = self.table[s, np.arange(self.lens[s]) // self.page]
        return (p >= 0) & (p < self.pages)

    def rows(self):
        return int(self.starts[-1])

    def queries(self, heads, std=1.0, extra=0):
        return pu.bf16(self.rng.standard_normal((self.rows() + extra, heads, self.d)) * std)

    def check(self, q, got, tag, block=1, window=0, sink=0, scale=None):
        """`got` against the definition in 64 bits, sequence by sequence."""
        scale = self.d ** -0.5 if scale is None else scale
        got16 = got.dtype == self.torch.bfloat16
        got = got.float().cpu().numpy()
        worst = 0.0
        for s, n in enumerate(self.counts):
            if n == 0:
                continue
            part = slice(self.starts[s], self.starts[s] + n)
            k, v = self.held("k", s), self.held("v", s)
            out, mag = pu.attention(q[part], k, v, self.lens[s] - n, scale, block, window, sink, self.usable(s))
            top = scale * 1.45 * float((np.abs(q[part]).max(initial=0) * np.nan_to_num(np.abs(k), posinf=0).max(initial=0))) * self.d
            bound = pu.attention_bound(out, mag, got16, top)
            x = got[part]
            nan = int((np.isnan(x) != np.isnan(out)).sum())
            assert nan == 0, f"{tag}: sequence {s}: {nan} of {x.size} values are NaN where the definition has none, or the reverse"
            off = np.nan_to_num(np.abs(x - out) - bound, nan=-1.0)
            worst = max(worst, float(np.nan_to_num(np.abs(x - out) / np.maximum(bound, 1e-300)).max()))
            fine = bool(off.max() <= 0)
            assert fine, f"{tag}: sequence {s}: off by {np.abs(x - out).max()} at {np.unravel_index(off.argmax(), off.shape)}"
        print(f"[paged] {tag}: worst {worst:.3f} of the bound", flush=True)


def tables(rows, d, halves):
    a = np.arange(rows)[:, None] * 10000.0 ** (-np.arange(0, d, 2) / d)[None, :]
    spread = (lambda t: np.concatenate([t, t], 1)) if halves else (lambda t: np.repeat(t, 2, 1))
    return tuple(spread(f(a)).astype(np.float32) for f in (np.cos, np.sin))


# ---- append and read -------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("d,page,halves,in16", [(128, 16, False, True), (64, 64, True, False), (128, 32, True, False), (64, 16, False, True)])
def test_append_stores_the_plain_values_bit_for_bit(fv, four, d, page, halves, in16):
    """Ragged sequences, some with no new token and one with no token at all; slices of a fused projection as inputs; slots
    that the call does not name keep their bits."""
    import torch

    announce(f"paged append four={four} d={d} page={page} halves={halves} in16={in16}")
    kvh, heads = 3, 6
    w = World(fv, 11 + d, [5, 0, 70, 33, 1, 17], [5, 0, 41, 0, 1, 2], kvh, d, page, four)
    n, extra = w.rows(), 4                       # rows behind the last sequence
    dtype = torch.bfloat16 if in16 else torch.float32
    fused = w.rng.standard_normal((n + extra, (heads + 2 * kvh) * d)).astype(np.float32)
    fused = pu.bf16(fused) if in16 else fused
    dev = w.dev(fused).to(dtype)
    q, k, v = (t.unflatten(1, (-1, d)) for t in dev.split([heads * d, kvh * d, kvh * d], 1))
    hq, hk, hv = (x.reshape(n + extra, -1, d) for x in np.split(fused, [heads * d, (heads + kvh) * d], 1))
    cos, sin = tables(80, d, halves)
    got_q = fv.paged_append(w.pool, w.batch, k, v, rope=(w.dev(cos), w.dev(sin)), halves=halves, q=q)
    got, got_s = w.pull()
    want_q = np.zeros((n, heads, d), dtype=np.float32)
    for s, c in enumerate(w.counts):
        part = slice(w.starts[s], w.starts[s] + c)
        pos = np.arange(w.lens[s] - c, w.lens[s])
        p, t = w.table[s, pos // page], pos % page
        want_q[part] = pu.bf16(pu.rotate(hq[part], cos, sin, pos, halves))
        for name, x in (("k", pu.rotate(hk[part], cos, sin, pos, halves)), ("v", hv[part])):
            if four:
                w.host[name][p, :, t], w.scales[name][p, :, t] = pu.quantize4(x)
            else:
                w.host[name][p, :, t] = pu.bf16(x)
    assert np.array_equal(got_q[:n].float().cpu().numpy(), want_q)
    for name in "kv":
        assert np.array_equal(got[name], w.host[name]), name
        if four:
            assert np.array_equal(got_s[name], w.scales[name]), name
    # and out again, as either type
    for out16 in (True, False):
        back = fv.paged_read(w.pool, w.batch, n, out_bf16=out16)
        for name, x in zip("kv", back):
            want = np.concatenate([w.held(name, s)[w.lens[s] - c:] for s, c in enumerate(w.counts)])
            assert np.array_equal(x.float().cpu().numpy().astype(np.float64), want), (name, out16)


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("in16", [False, True])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_append_in_every_form(fv, d, halves, in16, four):
    """Each kind of pages, inputs, pairs and head sizes: keys and queries turned, values as they are, bit for bit; with queries and
    without."""
    import torch

    announce(f"paged append: every form d={d} halves={halves} in16={in16} four={four}")
    kvh, heads = 5, 15
    for with_q in (True, False):
        w = World(fv, 500 + d, [40, 7, 100], [33, 7, 3], kvh, d, 32, four)
        n = w.rows()
        k, v, q = (w.rng.standard_normal((n, h, d)).astype(np.float32) * 3 for h in (kvh, kvh, heads))
        if in16:
            k, v, q = pu.bf16(k), pu.bf16(v), pu.bf16(q)
        cos, sin = tables(100, d, halves)
        pos = np.concatenate([np.arange(w.lens[s] - c, w.lens[s]) for s, c in enumerate(w.counts)])
        to = lambda x: w.dev(x).to(torch.bfloat16 if in16 else torch.float32)  # noqa: E731
        got_q = fv.paged_append(w.pool, w.batch, to(k), to(v), rope=(w.dev(cos), w.dev(sin)), halves=halves, q=to(q) if with_q else None)
        got, got_s = w.pull()
        if with_q:
            assert np.array_equal(got_q.float().cpu().numpy(), pu.bf16(pu.rotate(q, cos, sin, pos, halves)))
        else:
            assert got_q is None
        for name, x in (("k", pu.rotate(k, cos, sin, pos, halves)), ("v", v)):
            for s, c in enumerate(w.counts):
                part = slice(w.starts[s], w.starts[s] + c)
                p, t = w.table[s, pos[part] // 32], pos[part] % 32
                if four:
                    w.host[name][p, :, t], w.scales[name][p, :, t] = pu.quantize4(x[part])
                else:
                    w.host[name][p, :, t] = pu.bf16(x[part])
            assert np.array_equal(got[name], w.host[name]), name
            if four:
                assert np.array_equal(got_s[name], w.scales[name]), name


def test_append_without_tables_and_with_rows_of_its_own(fv):
    """No rotation; then a table row for each token (tokens of a frame that share an angle, a token twice)."""
    import torch

    announce("paged append: no rope, rope_at")
    d, kvh = 128, 2
    w = World(fv, 5, [40, 9], [7, 9], kvh, d, 16)
    n = w.rows()
    k, v = (w.rng.standard_normal((n, kvh, d)).astype(np.float32) for _ in range(2))
    assert fv.paged_append(w.pool, w.batch, w.dev(k), w.dev(v)) is None
    back = fv.paged_read(w.pool, w.batch, n)
    assert np.array_equal(back[0].float().cpu().numpy(), pu.bf16(k)) and np.array_equal(back[1].float().cpu().numpy(), pu.bf16(v))
    cos, sin = tables(6, d, False)
    rows = np.array([5, 5, 0, 3, 1, 1, 2, 4, 0, 0, 5, 3, 2, 2, 1, 4], dtype=np.int32)
    fv.paged_append(w.pool, w.batch, w.dev(k), w.dev(v), rope=(w.dev(cos), w.dev(sin)), rope_at=w.dev(rows))
    back = fv.paged_read(w.pool, w.batch, n)
    assert np.array_equal(back[0].float().cpu().numpy(), pu.bf16(pu.rotate(k, cos, sin, rows, False)))
    torch.cuda.synchronize()


def test_4_bit_blocks_of_every_kind(fv):
    """Zeros, borders between codes, one large value, the smallest and the largest numbers of f32, values that are not finite."""
    announce("paged append: 4-bit blocks")
    d, kvh = 64, 1
    border = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], dtype=np.float32)
    rows = [np.zeros(64), np.tile(border, 8), np.tile(-border, 8), np.tile(np.nextafter(border, np.float32(9)), 8),
            np.tile(np.nextafter(border, np.float32(0)), 8), np.tile(border, 8) * 2.0 ** -20, np.tile(border, 8) * 2.0 ** 100,
            np.r_[np.full(31, 1e-3), 1e3, np.full(32, -7.0)], np.full(64, 3.4e38), np.full(64, -1e-38), np.full(64, 1e-40),
            np.r_[np.full(31, 1.0), np.inf, np.full(32, 2.0)], np.r_[np.full(31, 1.0), np.nan, np.full(32, 2.0)],
            np.r_[np.full(32, 1.0), -np.inf, np.full(31, 2.0)], np.r_[np.full(32, 1.5), np.full(32, np.float32(1.5000001))],
            np.r_[np.full(32, 3.0), np.full(32, np.float32(3.0000002))]]
    x = np.stack(rows).astype(np.float32).reshape(-1, kvh, d)
    w = World(fv, 3, [len(rows)], [len(rows)], kvh, d, 16, four=True)
    fv.paged_append(w.pool, w.batch, w.dev(x), w.dev(x[::-1].copy()))
    got, scales = w.pull()
    for name, y in (("k", x), ("v", x[::-1])):
        codes, want_s = pu.quantize4(y)
        p, t = w.table[0, np.arange(len(rows)) // 16], np.arange(len(rows)) % 16
        assert np.array_equal(scales[name][p, :, t], want_s), name
        fine = np.repeat(want_s != 255, 16, -1)
        assert np.array_equal(np.where(fine, got[name][p, :, t], 0), np.where(fine, codes, 0)), name
        back = fv.paged_read(w.pool, w.batch, len(rows), out_bf16=False)[0 if name == "k" else 1].cpu().numpy()
        with np.errstate(over="ignore"):   # 3.4e38 is 3.997 x 2^126: code 4, which stands for 2^128, no number of f32 or bf16
            want = pu.values4(codes, want_s).astype(np.float32)
        assert np.array_equal(back, want, equal_nan=True), name


@pytest.mark.parametrize("d", [64, 128])
def test_every_4_bit_value_reads_as_what_it_stands_for(fv, d):
    """All codes under all 256 scales (f32 and bf16 hold every one of them, subnormal ones too, up to 2^128)."""
    announce(f"paged read: every 4-bit value d={d}")
    w = World(fv, 4, [256], [256], 1, d, 16, four=True)
    p, t = w.table[0, np.arange(256) // 16], np.arange(256) % 16
    for n, both in (("k", 0x10), ("v", 0x01)):
        w.host[n][p, 0, t] = (np.arange(d // 2) % 16 * both + 7 * (0x11 - both)).astype(np.uint8)
        w.scales[n][p, 0, t] = (np.arange(256)[:, None] + np.arange(d // 32)) % 256
    w.push()
    with np.errstate(over="ignore"):
        want = [w.held(n, 0).astype(np.float32) for n in "kv"]
    for out16 in (False, True):
        for x, y in zip(fv.paged_read(w.pool, w.batch, 256, out_bf16=out16), want):
            assert np.array_equal(x.float().cpu().numpy(), y, equal_nan=True), out16


def test_tokens_that_lie_nowhere_are_left_out(fv):
    """Page numbers outside the pool, table rows outside the tables, more rows than tokens: the others are as always, the
    pool's other slots keep their bits, queries without a place are zeros."""
    announce("paged append: pages and rows outside")
    import torch

    d, kvh, page, heads = 128, 2, 16, 4
    w = World(fv, 21, [40, 3, 20], [40, 5, 20], kvh, d, page)
    w.table[0, 1], w.table[2, 0] = w.pages, -1
    w.batch = fv.PagedBatch(w.dev(w.starts), w.dev(np.array(w.lens, dtype=np.int32)), w.dev(w.table), 40, 48)
    n = w.rows()
    k, v = (pu.bf16(w.rng.standard_normal((n, kvh, d))) for _ in range(2))
    q = w.queries(heads)
    cos, sin = tables(50, d, False)
    at = np.concatenate([np.arange(40), np.arange(5), np.arange(20)]).astype(np.int32)
    at[[2, 47]] = [50, -1]
    to = lambda x: w.dev(x).to(torch.bfloat16)  # noqa: E731
    got_q = fv.paged_append(w.pool, w.batch, to(k), to(v), rope=(w.dev(cos), w.dev(sin)), rope_at=w.dev(at), q=to(q))
    got, _ = w.pull()
    want_q = pu.bf16(pu.rotate(q, cos, sin, np.clip(at, 0, 49), False))
    turned = pu.bf16(pu.rotate(k, cos, sin, np.clip(at, 0, 49), False))
    lost_q = [2, 47, 40, 41]                     # rows outside the tables; two rows before the first token of sequence 1
    want_q[lost_q] = 0
    for s, c in enumerate(w.counts):
        for i in range(c):
            row, pos = w.starts[s] + i, w.lens[s] - c + i
            if row in lost_q or pos < 0 or not 0 <= w.table[s, pos // page] < w.pages:
                continue
            w.host["k"][w.table[s, pos // page], :, pos % page] = turned[row]
            w.host["v"][w.table[s, pos // page], :, pos % page] = v[row]
    assert np.array_equal(got_q.float().cpu().numpy(), want_q)
    assert np.array_equal(got["k"], w.host["k"]) and np.array_equal(got["v"], w.host["v"])
    back = fv.paged_read(w.pool, w.batch, n)[0].float().cpu().numpy()
    assert not back[16:32].any() and not back[40:42].any() and not back[45:61].any() and back[61:].any()


# ---- attention -------------------------------------------------------------------------------------------------------

MASKS = {"causal": (1, 0, 0), "window": (1, 37, 0), "sinks": (1, 37, 4), "blocks": (24, 0, 0), "block_window": (24, 2, 1), "one": (1, 1, 0)}


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("mask", sorted(MASKS))
@pytest.mark.parametrize("d,page,heads,kvh", [(128, 16, 8, 2), (64, 32, 6, 6), (128, 64, 5, 1), (64, 16, 12, 4)])
def test_single_tokens(fv, four, mask, d, page, heads, kvh):
    """One token a sequence, lengths from none to several steps and their neighbours; a row of a sequence without a token and
    a sequence without a row."""
    announce(f"paged tokens four={four} {mask} d={d} page={page} {heads}/{kvh}")
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 129, 500, 0, 77]
    w = World(fv, 100 + d + page, lens, [1] * 14 + [0], kvh, d, page, four, fill="nan")
    q = w.queries(heads)
    for out16 in (True, False):
        got = fv.paged_attention(w.dev(q).bfloat16(), w.pool, w.batch, fv.BlockCausal(*MASKS[mask]), out_bf16=out16)
        w.check(q, got, f"tokens {mask} four={four} d={d} out16={out16}", *MASKS[mask])
        assert not got[13].any()                 # no key: zeros


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("mask", sorted(MASKS))
@pytest.mark.parametrize("d,page,heads,kvh", [(128, 16, 8, 2), (64, 64, 3, 3), (128, 128, 7, 1)])
def test_ragged_rows(fv, four, mask, d, page, heads, kvh):
    """Drafts, prompts and continuations in one batch."""
    announce(f"paged ragged four={four} {mask} d={d} page={page} {heads}/{kvh}")
    lens, counts = [5, 300, 64, 1, 129, 200, 31], [5, 7, 64, 1, 33, 200, 0]
    w = World(fv, 200 + d, lens, counts, kvh, d, page, four, fill="nan")
    q = w.queries(heads, 2.0)
    for out16 in (True, False):
        got = fv.paged_attention(w.dev(q).bfloat16(), w.pool, w.batch, fv.BlockCausal(*MASKS[mask]), out_bf16=out16)
        w.check(q, got, f"ragged {mask} four={four} d={d} out16={out16}", *MASKS[mask])


def test_long_walks_are_split_and_joined(fv):
    """Few rows over a long axis, with and without the workspace for the shares; the same bits each time."""
    import torch

    announce("paged: split walks")
    for four, d in ((False, 128), (True, 128), (False, 64)):
        w = World(fv, 31, [9001, 300, 20000], [1, 1, 2], 2, d, 64, four, fill="nan")
        q = w.queries(4, 1.5)
        dq = w.dev(q).bfloat16()
        got = fv.paged_attention(dq, w.pool, w.batch, out_bf16=False)
        w.check(q, got, f"split four={four} d={d}")
        again = fv.paged_attention(dq, w.pool, w.batch, out_bf16=False)
        assert torch.equal(got, again)
        out = torch.full_like(got, 7.0)
        lib = fv.lib()
        assert lib.fv_paged_attention_workspace_bytes(4, 2, d, 3, 4, 2, 20000, 1, 0, 0) > 0
        rc = lib.fv_paged_attention(dq.data_ptr(), 4 * d, out.data_ptr(), 0, 4, *w.pool._args, *w.batch._args, 4, 2, 20000, d ** -0.5, 1, 0, 0,
                                    None, 0, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        w.check(q, out, f"unsplit four={four} d={d}")


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("d,page", [(128, 16), (128, 64), (64, 32)])
def test_many_rows_over_long_walks(fv, four, d, page):
    """More tiles than page numbers are looked up at once, walks split and whole, rows of one sequence and of several, a page
    that the pool does not have in the middle."""
    announce(f"paged: many rows, long walks four={four} d={d} page={page}")
    for lens, counts, mask in (([9000], [150], (1, 0, 0)), ([6000, 90, 5003], [40, 90, 3], (1, 0, 0)), ([7000, 5000], [64, 100], (1, 4500, 70)),
                               ([4680], [1560], (1560, 0, 0))):
        kvh, heads = (1, 2) if counts[0] > 1000 else (2, 4)
        w = World(fv, 61 + d + len(lens), lens, counts, kvh, d, page, four, fill="nan")
        w.table[0, 40 * 16 // page] = -3
        w.table[-1, 1] = w.pages + 5
        w.batch = fv.PagedBatch(w.dev(w.starts), w.dev(np.array(lens, dtype=np.int32)), w.dev(w.table), max(counts), max(lens))
        q = w.queries(heads, 1.5)
        for out16 in (True, False):
            got = fv.paged_attention(w.dev(q).bfloat16(), w.pool, w.batch, fv.BlockCausal(*mask), out_bf16=out16)
            w.check(q, got, f"long {lens} {mask} four={four} d={d} out16={out16}", *mask)


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("rows", ["tokens", "prompt"])
def test_scores_of_any_size(fv, four, rows):
    """Rows whose scores grow by hundreds after their first keys, whose first keys are hidden while all that they see is far below
    zero, and whose scores are all alike: no overflow, nothing vanishes."""
    announce(f"paged: scores of any size four={four} {rows}")
    d, kvh, heads, n = 128, 1, 4, 700
    for mask in ((1, 0, 0), (1, 90, 0), (1, 90, 3)):
        for grow in ("up", "down", "low", "flat"):
            counts = [1, 1] if rows == "tokens" else [300, 64]
            lens = [n, 130]
            w = World(fv, 71, lens, counts, kvh, d, 16, four)
            # keys along one direction: score = size(j) * |q| / sqrt(d)
            for s, length in enumerate(lens):
                j = np.arange(length)
                size = {"up": j / 8, "down": (length - j) / 8, "low": np.full(length, -40.0) + 0.5 * np.sin(j), "flat": np.full(length, 20.0)}[grow]
                k = np.zeros((length, kvh, d), dtype=np.float32)
                k[:, 0, :32] = size[:, None]
                p, t = w.table[s, j // 16], j % 16
                if four:
                    w.host["k"][p, :, t], w.scales["k"][p, :, t] = pu.quantize4(k)
                else:
                    w.host["k"][p, :, t] = pu.bf16(k)
            w.push()
            q = np.zeros((w.rows(), heads, d), dtype=np.float32)
            q[:, :, :32] = np.array([1.0, 2.0, 0.25, 4.0], dtype=np.float32)[None, :, None]
            got = fv.paged_attention(w.dev(q).bfloat16(), w.pool, w.batch, fv.BlockCausal(*mask), out_bf16=False)
            w.check(q, got, f"scores {rows} {mask} {grow} four={four}", *mask)


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("d,page", [(128, 16), (64, 64)])
def test_values_that_are_not_finite_reach_only_the_rows_that_see_them(fv, four, d, page):
    """NaN and infinities in keys and values at positions that some rows of a tile see and their neighbours do not."""
    announce(f"paged: NaN and infinities four={four} d={d}")
    for lens, counts, mask in (([70, 9], [5, 3], (1, 0, 0)), ([200, 150], [200, 90], (1, 0, 0)), ([300, 260], [120, 260], (1, 40, 3)),
                               ([40, 40], [12, 6], (1, 9, 2)), ([240, 96], [240, 48], (48, 1, 0))):
        kvh, heads = 2, 6
        for what in ("v", "k", "both"):
            w = World(fv, 81 + d, lens, counts, kvh, d, page, four)
            for s, n in enumerate(lens):
                for j in (n - counts[s] // 2, n - 3, n - counts[s] - 1 if counts[s] < n else n // 3, 1):
                    p, t = w.table[s, j // page], j % page
                    for name in ("kv" if what == "both" else what):
                        if four:
                            w.scales[name][p, 1, t, -1] = 255          # one head, its last 32 channels
                        else:
                            w.host[name][p, 1, t, 5] = np.nan if j % 2 or name == "k" else np.inf
            w.push()
            q = w.queries(heads)
            got = fv.paged_attention(w.dev(q).bfloat16(), w.pool, w.batch, fv.BlockCausal(*mask), out_bf16=False)
            got = got.cpu().numpy()
            for s, n in enumerate(counts):
                part = slice(w.starts[s], w.starts[s] + n)
                k, v = w.held("k", s), w.held("v", s)
                seen = pu.sees(np.arange(n) + w.lens[s] - n, np.arange(w.lens[s]), *mask)
                for h in range(heads):
                    kk, vv = k[:, h // 3], v[:, h // 3]
                    bad_k = ~np.isfinite(kk).all(1)
                    bad_row = (seen & bad_k[None, :]).any(1)
                    bad = bad_row[:, None] | ((seen[:, :, None] & ~np.isfinite(vv)[None, :, :]).any(1))
                    x = got[part, h]
                    assert (np.isfinite(x) == ~bad).all(), f"{lens} {mask} {what}: sequence {s} head {h}: {int((np.isfinite(x) != ~bad).sum())} values"
                fine = [w.held(name, s) for name in "kv"]
                clean = [np.nan_to_num(x, nan=0.0, posinf=0.0) for x in fine]
                out, mag = pu.attention(q[part], *clean, w.lens[s] - n, d ** -0.5, *mask)
                x = got[part]
                ok = np.isfinite(x)
                # rows that see nothing of the kind are as always (a row whose sum holds no such key, in every channel)
                whole = ok.all(-1)
                for h in range(heads):
                    some = (seen & (~np.isfinite(fine[0][:, h // 3]).all(1) | ~np.isfinite(fine[1][:, h // 3]).all(1))[None, :]).any(1)
                    whole[some, h] = False
                off = np.abs(x - out)[whole] - pu.attention_bound(out, mag, False, 60.0)[whole]
                assert off.size == 0 or off.max() <= 0


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("heads,kvh,d,rows,length,block", [(40, 40, 128, 1560, 3120, 1560), (32, 2, 64, 1500, 2000, 1500), (48, 16, 128, 500, 900, 1)])
def test_calls_of_more_than_a_round(fv, four, heads, kvh, d, rows, length, block):
    """More tiles than the chip holds at once: those of full rounds keep their walk, the rest are cut and joined. Against sums in 64
    bits (made on the device, head by head)."""
    import torch

    announce(f"paged: more than a round four={four} {heads}/{kvh} d={d}")
    w = World(fv, 91, [length], [rows], kvh, d, 64, four)
    q = w.queries(heads, 1.5)
    dq = w.dev(q).bfloat16()
    need = fv.lib().fv_paged_attention_workspace_bytes(heads, kvh, d, 1, rows, rows, length, block, 0, 0)
    got = fv.paged_attention(dq, w.pool, w.batch, fv.BlockCausal(block), out_bf16=False)
    k, v = (w.dev(w.held(n, 0)) for n in "kv")
    seen = w.dev(pu.sees(np.arange(rows) + length - rows, np.arange(length), block, 0, 0))
    for h in range(heads):
        s = (dq[:, h].double() @ k[:, h * kvh // heads].T) * d ** -0.5
        p = torch.softmax(s.masked_fill(~seen, -float("inf")), -1)
        out, mag = p @ v[:, h * kvh // heads], p @ v[:, h * kvh // heads].abs()
        # (the bound of attention_bound, with scores of up to 60)
        bound = (2.0 ** -8 + 2.0 * 130 * 2.0 ** -24 * 60 + 2.0 ** -12) * mag + 2.0 ** -24 * out.abs() + 1e-30
        off = float(((got[:, h].double() - out).abs() - bound).max())
        assert off <= 0, (h, off)
    print(f"[paged] {heads}/{kvh} d={d}: workspace {need} bytes", flush=True)


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("seqs,heads,kvh,d,window,long", [
    (2, 10, 2, 128, 0, (300,)), (64, 5, 1, 128, 0, (90, 700)), (65, 12, 12, 64, 50, (130,)), (200, 16, 1, 64, 0, (257, 64)),
    (33, 24, 3, 128, 0, (40,)), (4200, 5, 1, 64, 33, (1000, 128))])
def test_long_and_short_sequences_of_a_batch(fv, four, seqs, heads, kvh, d, window, long):
    """Sequences of no row, of one, of a few and of many, in any order, few of them long; the longest by itself says how much a
    sequence may have."""
    announce(f"paged: long and short four={four} {seqs} sequences {heads}/{kvh} d={d}")
    rng = np.random.Generator(np.random.PCG64(seqs))
    counts = rng.choice([0, 1, 1, 1, 2, 7], seqs)
    counts[rng.permutation(seqs)[:len(long)]] = long
    lens = counts + rng.integers(0, 90, seqs)
    if seqs in (33, 65):                         # (a walk that is cut)
        lens[counts.argmax()] += 9000
    w = World(fv, 700 + seqs, lens.tolist(), counts.tolist(), kvh, d, 16, four, fill="nan" if seqs < 1000 else "normal")
    q = w.queries(heads, 1.5)
    got = fv.paged_attention(w.dev(q).bfloat16(), w.pool, w.batch, fv.BlockCausal(1, window, 3 if window else 0), out_bf16=False)
    w.check(q, got, f"{seqs} sequences four={four}", 1, window, 3 if window else 0)
