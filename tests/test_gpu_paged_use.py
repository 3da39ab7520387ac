"""The paged KV cache as a program uses it: a clip block by block against the whole clip's block-causal attention, prompts in pieces,
captured serving steps replayed with other lengths, padded batches, shared pages, several streams, pools past 4 GB."""
import numpy as np
import pytest

import paged_util as pu
from test_gpu_paged import World, tables
from util import announce

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fv():
    import torch

    assert torch.cuda.is_available()
    import fv_sdpa

    fv_sdpa.lib()
    return fv_sdpa


def _gen(seed):
    import torch

    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(*x):
    import torch

    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("block,frames,window,sink", [(48, 9, 0, 0), (100, 7, 3, 1), (17, 12, 4, 0)])
def test_a_clip_block_by_block_is_the_block_causal_clip(fv, four, block, frames, window, sink):
    """Two clips in one pool, a block of each at a time: what the dense entry computes from the whole clips under the same mask on
    the keys and values that the cache holds (of 4 bits: read back from it)."""
    import torch

    announce(f"paged clip four={four} block={block} frames={frames} window={window} sink={sink}")
    d, heads, page, n = 128, 3, 16, block * frames
    g = _gen(1)
    q, k, v = (torch.randn((2, n, heads, d), generator=g, device="cuda").to(torch.bfloat16) for _ in range(3))
    rope = tuple(torch.from_numpy(t).cuda() for t in tables(n, d, False))
    columns = -(-n // page)
    pool = fv.PagedKv.new(2 * columns, page, heads, d, four_bits=four)
    table = torch.randperm(2 * columns, generator=g, device="cuda").to(torch.int32).view(2, columns)
    mask = fv.BlockCausal(block, window, sink)
    outs, turned = [], []
    for f in range(frames):
        part = slice(f * block, (f + 1) * block)
        batch = fv.PagedBatch(_i32(0, block, 2 * block), _i32((f + 1) * block, (f + 1) * block), table, block, (f + 1) * block)
        new = [x[:, part].reshape(2 * block, heads, d) for x in (k, v, q)]
        rq = fv.paged_append(pool, batch, new[0], new[1], rope=rope, q=new[2])
        turned.append(rq.view(2, block, heads, d))
        outs.append(fv.paged_attention(rq, pool, batch, mask).view(2, block, heads, d))
    got, rq = torch.cat(outs, 1), torch.cat(turned, 1)
    whole = fv.PagedBatch(_i32(0, n, 2 * n), _i32(n, n), table, n, n)
    hk, hv = (t.view(2, n, heads, d) for t in fv.paged_read(pool, whole, 2 * n))
    if not four:   # the rotation is the framework's own, bit for bit
        assert torch.equal(rq.transpose(1, 2).contiguous(), fv.rope_bhsd(q.transpose(1, 2).contiguous(), *rope))
        assert torch.equal(hk.transpose(1, 2).contiguous(), fv.rope_bhsd(k.transpose(1, 2).contiguous(), *rope))
        assert torch.equal(hv, v)
    flat = [t.transpose(1, 2).reshape(2 * heads, n, d).contiguous() for t in (rq, hk, hv)]
    want = fv.sdpa_block_causal_bf16(*flat, block, window, sink).view(2, heads, n, d).transpose(1, 2)
    mag = fv.sdpa_block_causal_bf16(flat[0], flat[1], flat[2].abs(), block, window, sink).view(2, heads, n, d).transpose(1, 2)
    # both round their probabilities to bf16 (2^-8 of each term), one rounds its result (2^-8); scores in f32 besides
    off = (got.float() - want).abs() - (2 * 2.0 ** -8 + 2.0 ** -10) * mag - 2.0 ** -8 * want.abs()
    assert float(off.max()) <= 0


@pytest.mark.parametrize("four", [False, True])
def test_a_prompt_in_pieces(fv, four):
    """Pieces of any size and the prompt at once agree with the definition, and leave the same cache."""
    announce(f"paged: prompt in pieces four={four}")
    n, d, kvh, heads = 333, 64, 2, 4
    w = World(fv, 9, [n], [n], kvh, d, 16, four)
    k, v, q = (pu.bf16(w.rng.standard_normal((n, h, d))) for h in (kvh, kvh, heads))
    to = lambda x: w.dev(x).bfloat16()  # noqa: E731
    rope = tuple(w.dev(t) for t in tables(n, d, True))
    rq = fv.paged_append(w.pool, w.batch, to(k), to(v), rope=rope, halves=True, q=to(q))
    once = fv.paged_attention(rq, w.pool, w.batch, fv.BlockCausal(1, 100, 5))
    cache = w.pull()
    w.host, w.scales = cache if four else (cache[0], None)
    w.check(rq.float().cpu().numpy(), once, f"at once four={four}", 1, 100, 5)
    for t in (w.pool.k, w.pool.v):
        t.zero_()
    at = 0
    for piece in (1, 64, 2, 129, 100, 37):
        end = at + piece
        batch = fv.PagedBatch(_i32(0, piece), _i32(end), w.batch.table, piece, end)
        part = fv.paged_append(w.pool, batch, to(k[at:end]), to(v[at:end]), rope=rope, halves=True, q=to(q[at:end]))
        got = fv.paged_attention(part, w.pool, batch, fv.BlockCausal(1, 100, 5))
        out, mag = pu.attention(part.float().cpu().numpy(), w.held("k", 0)[:end], w.held("v", 0)[:end], at, d ** -0.5, 1, 100, 5)
        off = np.abs(got.float().cpu().numpy() - out) - pu.attention_bound(out, mag, True, 60.0)
        fine = bool(off.max() <= 0)
        assert fine, (piece, off.max())
        at = end
    again = w.pull()
    inside = w.table[0, np.arange(n) // 16], np.arange(n) % 16
    for name in "kv":
        assert np.array_equal(again[0][name][inside[0], :, inside[1]], cache[0][name][inside[0], :, inside[1]])


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("long", [False, True])
def test_a_captured_step_is_replayed_with_other_lengths(fv, four, long):
    """append + attention of a padded batch in one graph: between the replays the program writes new tokens, lengths, counts and
    tables into the same arrays (and works and waits besides). Every replay equals the eager calls bit for bit; rows behind
    the last sequence keep what they held. `long`: walks in shares, whose workspace the graph owns."""
    import torch

    announce(f"paged graph four={four} long={long}")
    d, kvh, heads, page, seqs, rows = 128, 2, 8, 64, 5, 24
    max_len = 9000 if long else 500
    g = _gen(3)
    columns = -(-max_len // page)
    rng = np.random.Generator(np.random.PCG64(4))
    pools = [fv.PagedKv.new(seqs * columns + 2, page, kvh, d, four_bits=four) for _ in range(2)]
    for a, b in zip((pools[0].k, pools[0].v, pools[0].k_scales, pools[0].v_scales), (pools[1].k, pools[1].v, pools[1].k_scales, pools[1].v_scales)):
        if a is not None:
            if a.dtype == torch.uint8:
                a.copy_(torch.randint(120, 130, a.shape, generator=g, device="cuda", dtype=torch.uint8))
            else:
                a.copy_(torch.randn(a.shape, generator=g, device="cuda"))
            b.copy_(a)
    rope = tuple(torch.from_numpy(t).cuda() for t in tables(max_len, d, False))
    k, v = (torch.zeros((rows, kvh, d), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    q = torch.zeros((rows, heads, d), device="cuda", dtype=torch.bfloat16)
    start, lens = torch.zeros(seqs + 1, dtype=torch.int32, device="cuda"), torch.zeros(seqs, dtype=torch.int32, device="cuda")
    table = torch.zeros((seqs, columns), dtype=torch.int32, device="cuda")
    batch = fv.PagedBatch(start, lens, table, 8, max_len)
    mask = fv.BlockCausal(1, 0 if long else 200, 4)

    def fill(i):
        counts = rng.integers(0, 5, seqs)
        counts[i % seqs] = [0, 1, 8, 3][i % 4]
        n = np.maximum(rng.integers(1, max_len + 1, seqs), counts)
        order = rng.permutation(seqs * columns)
        start.copy_(torch.from_numpy(np.r_[0, np.cumsum(counts)].astype(np.int32)))
        lens.copy_(torch.from_numpy(n.astype(np.int32)))
        table.copy_(torch.from_numpy(order.reshape(seqs, columns).astype(np.int32)))
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        return int(counts.sum())

    def step(pool, out):
        rq = fv.paged_append(pool, batch, k, v, rope=rope, q=q)
        fv.paged_attention(rq, pool, batch, mask, out=out)

    out = torch.zeros((rows, heads, d), device="cuda", dtype=torch.bfloat16)
    want = torch.zeros_like(out)
    fill(0)
    step(pools[0], out)
    step(pools[1], want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(pools[0], out)
    for i in range(6):
        n = fill(i + 1)
        out.fill_(3.0)
        want.fill_(3.0)
        step(pools[1], want)
        if i % 2:
            torch.cuda.synchronize()
        graph.replay()
        junk = torch.randn((512, 512), device="cuda") @ torch.randn((512, 512), device="cuda")
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        assert (out[n:] == 3.0).all() and torch.isfinite(out.float()).all() and torch.isfinite(junk).all()
        assert torch.equal(pools[0].k, pools[1].k) and torch.equal(pools[0].v, pools[1].v)


def test_two_streams_at_once(fv):
    """Two batches on two streams in turn, each with its own workspace: the bits of one after the other."""
    import torch

    announce("paged: two streams")
    worlds = [World(fv, 300 + i, [7000, 900, 12000], [1, 3, 2], 2, 128, 64, four=bool(i)) for i in range(2)]
    qs = [w.dev(w.queries(8)).bfloat16() for w in worlds]
    want = [fv.paged_attention(q, w.pool, w.batch, out_bf16=False) for q, w in zip(qs, worlds)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in worlds]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(fv.paged_attention(qs[i], worlds[i].pool, worlds[i].batch, out_bf16=False))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_rows_outside_the_sequences_are_left(fv):
    """q_start that begins past the first row and ends before the last."""
    import torch

    announce("paged: rows outside")
    d, kvh, heads = 64, 2, 4
    w = World(fv, 13, [20, 90], [3, 70], kvh, d, 16)
    n, first, rows = w.rows(), 5, 90
    batch = fv.PagedBatch(w.dev(w.starts + first), w.batch.lens, w.batch.table, 70, 90)
    q, k, v = (pu.bf16(w.rng.standard_normal((rows, h, d))) for h in (heads, kvh, kvh))
    before = w.pull()[0]
    lib = fv.lib()
    dq, dk, dv = (w.dev(x).bfloat16() for x in (q, k, v))
    marked = [torch.full((rows, h, d), 9.0, device="cuda", dtype=torch.bfloat16) for h in (heads, kvh, kvh, heads)]
    st = torch.cuda.current_stream().cuda_stream
    assert lib.fv_paged_append(dk.data_ptr(), kvh * d, dv.data_ptr(), kvh * d, dq.data_ptr(), heads * d, marked[0].data_ptr(), 1, heads, None, None, 0,
                               None, 0, *w.pool._args, *batch._args, rows, st) == 0
    assert lib.fv_paged_read(marked[1].data_ptr(), marked[2].data_ptr(), 1, *w.pool._args, *batch._args, rows, st) == 0
    fv.paged_attention(dq, w.pool, batch, out=marked[3])
    torch.cuda.synchronize()
    part = slice(first, first + n)
    assert torch.equal(marked[0][part], dq[part]) and torch.equal(marked[1][part], dk[part]) and torch.equal(marked[2][part], dv[part])
    for t in marked:
        assert (t[:first] == 9.0).all() and (t[first + n:] == 9.0).all()
    for s, c in enumerate(w.counts):
        at = first + w.starts[s]
        pos = np.arange(w.lens[s] - c, w.lens[s])
        w.host["k"][w.table[s, pos // 16], :, pos % 16] = k[at:at + c]
        w.host["v"][w.table[s, pos // 16], :, pos % 16] = v[at:at + c]
    after = w.pull()[0]
    assert all(np.array_equal(after[x], w.host[x]) for x in "kv") and not np.array_equal(before["k"], after["k"])
    w.check(q[part], marked[3][part].contiguous(), "rows outside")


@pytest.mark.parametrize("heads,kvh", [(4, 4), (10, 2)])
def test_many_rows_before_the_first_sequence(fv, heads, kvh):
    """A batch of long and short sequences whose first row is far behind the tensors' first: pieces of rows that belong to nobody."""
    import torch

    announce(f"paged: rows before the first sequence {heads}/{kvh}")
    lens, counts, before = [700, 3, 50, 9000, 2, 1, 1, 1], [300, 1, 0, 130, 1, 1, 1, 1], 1000
    w = World(fv, 41, lens, counts, kvh, 64, 16)
    n, rows = w.rows(), before + w.rows() + 200
    q = w.queries(heads, 1.5)
    dq = torch.zeros((rows, heads, 64), device="cuda", dtype=torch.bfloat16)
    dq[before:before + n] = w.dev(q).bfloat16()
    batch = fv.PagedBatch(w.dev(w.starts + np.int32(before)), w.dev(np.array(lens, dtype=np.int32)), w.dev(w.table), max(counts), max(lens))
    out = torch.full((rows, heads, 64), 5.0, device="cuda", dtype=torch.float32)
    fv.paged_attention(dq, w.pool, batch, out_bf16=False, out=out)
    w.check(q, out[before:before + n], f"rows before {heads}/{kvh}")
    assert (out[:before] == 5.0).all() and (out[before + n:] == 5.0).all()


def test_sequences_may_share_pages(fv):
    """A prefix kept once: both sequences read it, each appends to pages of its own."""
    announce("paged: a shared prefix")
    w = World(fv, 17, [100, 75], [4, 11], 2, 128, 16)
    w.table[1, :4] = w.table[0, :4]
    w.batch = fv.PagedBatch(w.dev(w.starts), w.dev(np.array(w.lens, dtype=np.int32)), w.dev(w.table), 11, 100)
    q = w.queries(6)
    w.check(q, fv.paged_attention(w.dev(q).bfloat16(), w.pool, w.batch), "shared prefix")


def test_more_rows_than_tokens(fv):
    """Rows before a sequence's first token see nothing and are zeros, in both kernels; lengths past the bound are cut to it."""
    announce("paged: rows before the first token")
    for counts in ([5, 2], [130, 70]):
        w = World(fv, 19, [3, 40], counts, 2, 64, 16)
        q = w.queries(2)
        got = fv.paged_attention(w.dev(q).bfloat16(), w.pool, w.batch)
        w.check(q, got, f"few tokens {counts}")
        assert not got[:counts[0] - 3].any() and got[counts[0] - 3:counts[0]].any()
    w = World(fv, 23, [60, 40], [2, 2], 2, 64, 16, max_len=33)
    q = w.queries(2)
    got = fv.paged_attention(w.dev(q).bfloat16(), w.pool, w.batch)
    w.lens = [33, 33]
    w.check(q, got, "lengths cut to the bound")


def test_strided_queries_and_tables(fv):
    """Queries that are a slice of a fused projection, a table that is a slice of a wider one, one-row batches."""
    import torch

    announce("paged: strides")
    w = World(fv, 29, [50, 200, 31], [3, 40, 1], 2, 128, 32)
    q = w.queries(4)
    wide = torch.zeros((w.rows(), 10, 128), device="cuda", dtype=torch.bfloat16)
    wide[:, 3:7] = w.dev(q)
    tables_ = torch.full((3, 40), 1 << 20, device="cuda", dtype=torch.int32)
    tables_[:, 5:5 + w.table.shape[1]] = w.dev(w.table)
    batch = fv.PagedBatch(w.batch.q_start, w.batch.lens, tables_[:, 5:5 + w.table.shape[1]], 40, 200)
    got = fv.paged_attention(wide[:, 3:7], w.pool, batch)
    assert got.is_contiguous() and torch.equal(got, fv.paged_attention(w.dev(q).bfloat16(), w.pool, w.batch))
    w.check(q, got, "strides")
    one = fv.PagedBatch(_i32(0, 1), _i32(31), tables_[2:3, 5:6], 1, 31)
    last = fv.paged_attention(wide[-1:, 3:7], w.pool, one)
    assert torch.equal(last, got[-1:])


def test_refusals_in_python(fv):
    import torch

    announce("paged: refusals")
    w = World(fv, 37, [20], [2], 2, 64, 16)
    q = w.dev(w.queries(4)).bfloat16()
    with pytest.raises(ValueError):
        fv.PagedKv(w.pool.k, w.pool.v[:, :1])
    with pytest.raises(ValueError):
        fv.PagedKv(w.pool.k.float(), w.pool.v.float())
    with pytest.raises(ValueError):
        fv.PagedKv(w.pool.k.transpose(1, 2), w.pool.v.transpose(1, 2))
    with pytest.raises(ValueError):
        fv.PagedKv(w.pool.k.cpu(), w.pool.v.cpu())
    with pytest.raises(ValueError):
        fv.PagedBatch(w.batch.q_start.long(), w.batch.lens, w.batch.table, 2)
    with pytest.raises(ValueError):
        fv.PagedBatch(w.batch.q_start[:1], w.batch.lens, w.batch.table, 2)
    with pytest.raises(ValueError):
        fv.PagedBatch(w.batch.q_start, w.batch.lens, w.batch.table, -1)
    with pytest.raises(ValueError):
        fv.paged_attention(q.float(), w.pool, w.batch)
    with pytest.raises(ValueError):
        fv.paged_attention(q.transpose(1, 2).contiguous().transpose(1, 2), w.pool, w.batch)
    with pytest.raises(ValueError):
        fv.paged_attention(q, w.pool, w.batch, out=torch.empty_like(q).float())
    with pytest.raises(fv.FvError):
        fv.paged_attention(q[:, :3], w.pool, w.batch)             # 3 query heads over 2 key heads
    with pytest.raises(fv.FvError):
        fv.paged_attention(q[:, :2].expand(-1, -1, -1)[:1].expand(2, -1, -1), w.pool, w.batch)   # tokens that overlap
    with pytest.raises(fv.FvDeclined):
        fv.paged_attention(q, w.pool, w.batch, scale=0.0)
    with pytest.raises(fv.FvError):
        fv.paged_attention(q, w.pool, fv.PagedBatch(w.batch.q_start, w.batch.lens, w.batch.table, 2, 1000))
    with pytest.raises(ValueError):
        fv.paged_append(w.pool, w.batch, q[:, :2], q[:, :2].float())
    with pytest.raises(ValueError):
        fv.paged_append(w.pool, w.batch, q[:, :2], q[:, :2], rope=(q, q))
    with pytest.raises(ValueError):
        fv.paged_append(w.pool, w.batch, q[:, :2], q[:, :2], rope_at=w.batch.lens)
    # nothing to do
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    empty = fv.PagedBatch(_i32(0), none, none.view(0, 0), 0)
    assert fv.paged_attention(q[:0], w.pool, empty).shape == (0, 4, 64)
    assert fv.paged_append(w.pool, empty, q[:0, :2], q[:0, :2]) is None
    assert fv.paged_read(w.pool, empty, 0)[0].shape == (0, 2, 64)


@pytest.mark.parametrize("four", [False, True])
def test_pools_past_four_gigabytes(fv, four):
    """Pages whose rows lie past 2^32 bytes (bf16) and past 2^31 rows (4 bits; keys and values are one tensor there)."""
    import torch

    announce(f"paged: a large pool four={four}")
    d, kvh, page, heads = (64, 32, 64, 32) if four else (128, 8, 64, 16)
    pages = (1 << 31) // (kvh * page) + 100 if four else 40000
    free = torch.cuda.mem_get_info()[0]
    need = pages * kvh * page * (d // 2 + d // 32 if four else 4 * d)
    if need + (8 << 30) > free:
        pytest.skip("not enough memory free")
    shape = (pages, kvh, page)
    if four:
        codes = torch.empty((*shape, d // 2), dtype=torch.uint8, device="cuda")
        scales = torch.empty((*shape, d // 32), dtype=torch.uint8, device="cuda")
        pool = fv.PagedKv(codes, codes, scales, scales)
    else:
        pool = fv.PagedKv(*(torch.empty((*shape, d), dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    lens, counts = [200, 130], [200, 3]
    table = torch.tensor([[pages - 1, pages - 7, 0, pages // 2 + 1], [pages - 3, 2, pages - 2, 1]], dtype=torch.int32, device="cuda")
    batch = fv.PagedBatch(_i32(0, 200, 203), _i32(*lens), table, 200, 200)
    everything = fv.PagedBatch(_i32(0, 200, 330), _i32(*lens), table, 200, 200)
    rng = np.random.Generator(np.random.PCG64(5))
    x = pu.bf16(rng.standard_normal((330, kvh, d)))
    y = x if four else pu.bf16(rng.standard_normal((330, kvh, d)))
    dev = lambda t: torch.from_numpy(t).cuda().bfloat16()  # noqa: E731
    fv.paged_append(pool, everything, dev(x), dev(y))
    if four:
        x = y = pu.values4(*pu.quantize4(x)).astype(np.float32)
    for got, want in zip(fv.paged_read(pool, everything, 330), (x, y)):
        assert np.array_equal(got.float().cpu().numpy(), want)
    q = pu.bf16(rng.standard_normal((203, heads, d)))
    got = fv.paged_attention(dev(q), pool, batch).float().cpu().numpy()
    for part, rows, first in ((slice(0, 200), slice(0, 200), 0), (slice(200, 203), slice(200, 330), 127)):
        out, mag = pu.attention(q[part], x[rows], y[rows], first, d ** -0.5)
        off = np.abs(got[part] - out) - pu.attention_bound(out, mag, True, 60.0)
        fine = bool(off.max() <= 0)
        assert fine, off.max()
