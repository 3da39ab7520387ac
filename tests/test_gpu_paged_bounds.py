"""The paged KV cache at the borders of what a call describes."""
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


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("d,page,halves", [(128, 16, False), (64, 32, True)])
def test_tokens_past_the_table_are_not_stored(fv, four, d, page, halves):
    """Sequences of more tokens than their table has slots for: the new tokens that fit go to their places under their own
    angles, the others nowhere (the newest that fits keeps its slot), whose queries are turned like any; all read as zeros."""
    import torch

    announce(f"paged append: past the table four={four} d={d}")
    kvh, heads, columns = 2, 4, 2
    held = columns * page
    counts = [5, 3, 20, 2, 4]
    w = World(fv, 51, [held, held, 20, held, held], counts, kvh, d, page, four)
    lens = [held + 3, held + 8, 20, 2 ** 31 - 1, held]           # 3 tokens past it, all of them, none, all at the far end, none
    w.batch = fv.PagedBatch(w.batch.q_start, w.dev(np.array(lens, dtype=np.int32)), w.batch.table, 20)
    n = w.rows()
    k, v = (pu.bf16(w.rng.standard_normal((n, kvh, d))) for _ in range(2))
    q = w.queries(heads)
    rows = held + 20
    cos, sin = tables(rows, d, halves)
    to = lambda x: w.dev(x).to(torch.bfloat16)  # noqa: E731
    got_q = fv.paged_append(w.pool, w.batch, to(k), to(v), rope=(w.dev(cos), w.dev(sin)), halves=halves, q=to(q))
    pos = np.concatenate([np.arange(m - c, m, dtype=np.int64) for m, c in zip(lens, counts)])
    at = np.clip(pos, 0, rows - 1)
    want_q = pu.bf16(pu.rotate(q, cos, sin, at, halves))
    want_q[pos >= rows] = 0                                      # (no row of the tables)
    turned = pu.rotate(k, cos, sin, at, halves)
    fits = pos < held
    assert fits.sum() == 2 + 0 + 20 + 0 + 4
    want = {name: np.zeros((n, kvh, d)) for name in "kv"}
    for s, c in enumerate(counts):
        for i in range(w.starts[s], w.starts[s] + c):
            if not fits[i]:
                continue
            p, t = w.table[s, pos[i] // page], pos[i] % page
            for name, x in (("k", turned[i]), ("v", v[i])):
                if four:
                    w.host[name][p, :, t], w.scales[name][p, :, t] = pu.quantize4(x)
                    want[name][i] = pu.values4(w.host[name][p, :, t], w.scales[name][p, :, t])
                else:
                    want[name][i] = w.host[name][p, :, t] = pu.bf16(x)
    got, got_s = w.pull()
    assert np.array_equal(got_q.float().cpu().numpy(), want_q)
    for name in "kv":
        assert np.array_equal(got[name], w.host[name]), name
        assert not four or np.array_equal(got_s[name], w.scales[name]), name
    for x, name in zip(fv.paged_read(w.pool, w.batch, n, out_bf16=False), "kv"):
        assert np.array_equal(x.cpu().numpy().astype(np.float64), want[name]), name


def test_rope_tables_without_rows_are_refused(fv):
    """Every token's row lies outside them: storing the keys unturned is not what was asked."""
    import torch

    announce("paged append: empty rope tables")
    w = World(fv, 53, [20], [2], 2, 64, 16)
    x = torch.zeros((2, 2, 64), device="cuda", dtype=torch.bfloat16)
    none = torch.empty((0, 64), device="cuda")
    before = w.pull()[0]
    with pytest.raises(ValueError, match="rope"):
        fv.paged_append(w.pool, w.batch, x, x, rope=(none, none))
    with pytest.raises(ValueError, match="rope"):
        fv.paged_append(w.pool, w.batch, x, x, rope=(none, none), rope_at=torch.zeros(2, device="cuda", dtype=torch.int32))
    after = w.pull()[0]
    assert all(np.array_equal(before[n], after[n]) for n in "kv")


def test_drafts_over_bf16_pages_allocate_their_result_alone(fv):
    """64 sequences of 9 drafts, a bound of 131072 keys: no shares (over 4 bits there are, 380 MB)."""
    import torch

    announce("paged attention: memory of a call of drafts")
    seqs, rows, heads, kvh, d, page = 64, 9, 40, 8, 128, 64
    pool = fv.PagedKv.new(seqs, page, kvh, d)
    columns = 131072 // page
    table = torch.full((seqs, columns), -1, dtype=torch.int32, device="cuda")
    table[:, 0] = torch.arange(seqs, device="cuda")
    start = torch.arange(seqs + 1, device="cuda", dtype=torch.int32) * rows
    batch = fv.PagedBatch(start, torch.full((seqs,), 50, dtype=torch.int32, device="cuda"), table, rows)
    q = torch.zeros((seqs * rows, heads, d), device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = fv.paged_attention(q, pool, batch)
    torch.cuda.synchronize()
    assert not out.any()
    more = torch.cuda.max_memory_allocated() - before
    assert more <= out.numel() * 2 + (1 << 20), more


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("lens,counts,heads,mask", [([45, 20], [3, 2], 2, (1, 0, 0)), ([45, 200], [7, 9], 4, (1, 12, 2)), ([300], [150], 2, (1, 0, 0)),
                                                    ([260, 90], [140, 70], 4, (1, 40, 3)), ([240], [96], 4, (48, 0, 0))])
def test_a_value_that_is_not_finite_reaches_rows_whose_weight_for_it_vanishes(fv, four, lens, counts, heads, mask):
    """Its key scores 300 below the others, so that its weight is less than any f32; a row that sees it is not a number all the
    same (as where every row of the tile sees it), a row that does not is as always."""
    import torch

    d, kvh, page = 128, 2, 16
    announce(f"paged: a vanishing weight on NaN four={four} {lens} {mask}")
    for back in (1, 5, 20):                                      # the planted key, from the first new token back
        w = World(fv, 57, lens, counts, kvh, d, page, four)
        for s, n in enumerate(lens):
            j = np.arange(n)
            keys = np.zeros((n, kvh, d), dtype=np.float32)
            bad = [x for x in (n - counts[s] - back, n - counts[s] + counts[s] // 2) if x >= 0]
            keys[bad] = -6.0
            p, t = w.table[s, j // page], j % page
            if four:
                w.host["k"][p, :, t], w.scales["k"][p, :, t] = pu.quantize4(keys)
            else:
                w.host["k"][p, :, t] = keys
            for x in bad:
                if four:
                    w.scales["v"][w.table[s, x // page], 1, x % page, -1] = 255
                else:
                    w.host["v"][w.table[s, x // page], 1, x % page, 5] = np.nan
        w.push()
        q = np.full((w.rows(), heads, d), 4.5, dtype=np.float32)   # -6 x 4.5 x 128 / sqrt(128) = -305
        got = fv.paged_attention(w.dev(q).bfloat16(), w.pool, w.batch, fv.BlockCausal(*mask), out_bf16=False).cpu().numpy()
        some = False
        for s, n in enumerate(counts):
            part = slice(w.starts[s], w.starts[s] + n)
            k, v = w.held("k", s), w.held("v", s)
            seen = pu.sees(np.arange(n) + lens[s] - n, np.arange(lens[s]), *mask)
            finite = np.stack([~(seen[:, :, None] & ~np.isfinite(v[:, h * kvh // heads])[None]).any(1) for h in range(heads)], 1)
            x = got[part]
            wrong = int((np.isfinite(x) != finite).sum())
            assert wrong == 0, f"back={back}: sequence {s}: {wrong} of {x.size} values are numbers where they are none, or the reverse"
            out, mag = pu.attention(q[part], k, np.nan_to_num(v, nan=0.0), lens[s] - n, d ** -0.5, *mask)
            off = np.where(finite, np.abs(x - out) - pu.attention_bound(out, mag, False, 1.45 * 306), -1.0)
            assert off.max() <= 0, (back, s, off.max())
            some |= bool((~finite).any() and finite[:, -1].any())
        assert some or back > 1


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("counts", [[1, 1, 2], [90, 1, 150]])
def test_entries_that_no_row_reaches_may_hold_anything(fv, four, page, counts):
    """Pages that lie wholly outside a window and its sinks, or behind the last token: numbers outside the pool, and of a page of
    NaN that is another's (a window's pages given away)."""
    announce(f"paged: entries out of reach four={four} page={page} {counts}")
    lens, mask = [1003, 37, 777], (1, 70, 5)
    w = World(fv, 61, lens, counts, 2, 128, page, four, columns=-(-1003 // page) + 2)
    other = next(p for p in range(w.pages) if not (w.table == p).any())   # (a spare page, no sequence's)
    for name in "kv":
        if four:
            w.scales[name][other] = 255
        else:
            w.host[name][other] = np.nan
    w.push()
    reached = np.zeros(w.table.shape, dtype=bool)
    for s, (n, c) in enumerate(zip(lens, counts)):
        seen = pu.sees(np.arange(c) + n - c, np.arange(n), *mask).any(0)
        reached[s, np.unique(np.nonzero(seen)[0] // page)] = True
    assert (~reached).sum() > 5
    q = w.queries(4)
    for stale in (other, -1, w.pages, 2 ** 31 - 1, -2 ** 31):
        w.batch = fv.PagedBatch(w.batch.q_start, w.batch.lens, w.dev(np.where(reached, w.table, np.int32(stale))), max(counts), max(lens))
        got = fv.paged_attention(w.dev(q).bfloat16(), w.pool, w.batch, fv.BlockCausal(*mask), out_bf16=False)
        w.check(q, got, f"stale {stale} page={page} {counts}", *mask)


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("lens,counts,first,rows", [([40, 50], [10, 20], 0, 22), ([40, 50], [3, 2], -2, 20), ([300, 260], [150, 160], -7, 200)])
def test_rows_that_the_tensors_do_not_have(fv, four, lens, counts, first, rows):
    """q_start from before the tensors' first row, or to behind their last: the rows that are there are the tokens that q_start says."""
    import torch

    announce(f"paged: rows past the tensors four={four} {counts} {first} {rows}")
    kvh, heads, d, page = 2, 4, 64, 16
    w = World(fv, 67, lens, counts, kvh, d, page, four)
    starts = w.starts + np.int32(first)
    batch = fv.PagedBatch(w.dev(starts), w.batch.lens, w.batch.table, max(counts), max(lens))
    k, v, q = (pu.bf16(w.rng.standard_normal((rows, h, d))) for h in (kvh, kvh, heads))
    cos, sin = tables(max(lens), d, False)
    to = lambda x: w.dev(x).to(torch.bfloat16)  # noqa: E731
    rq = fv.paged_append(w.pool, batch, to(k), to(v), rope=(w.dev(cos), w.dev(sin)), q=to(q))
    there = []
    for s, (n, c) in enumerate(zip(lens, counts)):
        t = np.arange(max(starts[s], 0), min(starts[s] + c, rows))
        pos = n - c + t - starts[s]
        there.append((t, pos))
        p, slot = w.table[s, pos // page], pos % page
        for name, x in (("k", pu.rotate(k[t], cos, sin, pos, False)), ("v", v[t])):
            if four:
                w.host[name][p, :, slot], w.scales[name][p, :, slot] = pu.quantize4(x)
            else:
                w.host[name][p, :, slot] = pu.bf16(x)
    got, _ = w.pull()
    fine = all(np.array_equal(got[name], w.host[name]) for name in "kv")
    assert fine
    back = fv.paged_read(w.pool, batch, rows, out_bf16=False)
    out = fv.paged_attention(rq, w.pool, batch, out_bf16=False).cpu().numpy()
    for s, (t, pos) in enumerate(there):
        turned = pu.bf16(pu.rotate(q[t], cos, sin, pos, False))
        fine = np.array_equal(rq[t].float().cpu().numpy(), turned)
        assert fine, s
        for x, name in zip(back, "kv"):
            fine = np.array_equal(x[t].cpu().numpy().astype(np.float64), w.held(name, s)[pos])
            assert fine, (s, name)
        want, mag = pu.attention(turned, w.held("k", s), w.held("v", s), pos[0], d ** -0.5)
        off = float((np.abs(out[t] - want) - pu.attention_bound(want, mag, False, 60.0)).max())
        assert off <= 0, (s, off)


@pytest.mark.parametrize("lens,counts,heads,mask", [([70, 9], [5, 3], 6, (1, 0, 0)), ([9000, 300], [2, 1], 4, (1, 0, 0)), ([200, 150], [200, 90], 2, (1, 0, 0)),
                                                    ([300, 260], [120, 260], 4, (1, 40, 3)), ([9000], [70], 4, (1, 0, 0))])
def test_infinite_keys_and_queries_that_are_not_numbers(fv, lens, counts, heads, mask):
    """A key of infinite entries scores infinity (the row is not a number) or minus infinity (its weight is zero) for a row that
    sees it, by the sign of the query there; a query that is not a number is its own row's alone."""
    d, kvh, page = 128, 2, 32
    announce(f"paged: infinite keys {lens} {mask}")
    w = World(fv, 71, lens, counts, kvh, d, page)
    for s, n in enumerate(lens):
        for j, x in ((n - counts[s] // 2 - 1, np.inf), (n - 2, -np.inf), (n // 2, np.inf), (3, -np.inf)):
            w.host["k"][w.table[s, j // page], 1, j % page, 7] = x
    w.push()
    q = w.queries(heads)
    q[:, heads // 2:, 7] = np.where(w.rng.random((w.rows(), heads - heads // 2)) < 0.5, 2.0, -2.0)
    lost = [0, w.rows() - 2]
    q[lost[0], 0, 3] = np.nan
    q[lost[1], heads - 1, 100] = np.inf
    got = fv.paged_attention(w.dev(q).bfloat16(), w.pool, w.batch, fv.BlockCausal(*mask), out_bf16=False).cpu().numpy()
    nan = number = 0
    for s, n in enumerate(counts):
        part = slice(w.starts[s], w.starts[s] + n)
        seen = pu.sees(np.arange(n) + lens[s] - n, np.arange(lens[s]), *mask)
        k = w.held("k", s)
        for h in range(heads):
            kk = k[:, h * kvh // heads]
            with np.errstate(invalid="ignore"):
                scores = q[part, h].astype(np.float64) @ kk.T * d ** -0.5
            scores[~seen] = -np.inf
            bad = ~(scores < np.inf).all(1)
            x = got[part, h]
            wrong = int((np.isnan(x).all(1) != bad).sum() + (np.isfinite(x).all(1) == bad).sum())
            assert wrong == 0, (s, h, wrong)
            some = ~bad & np.isfinite(scores).any(1)
            p = np.exp(scores[some] - scores[some].max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            v = w.held("v", s)[:, h * kvh // heads]
            out, mag = p @ v, p @ np.abs(v)
            off = np.abs(x[some] - out) - pu.attention_bound(out, mag, False, 1.45 * 40)
            assert off.size == 0 or off.max() <= 0, (s, h, off.max())
            nan, number = nan + int(bad.sum()), number + int(some.sum())
    assert nan > 2 and number > 2


@pytest.mark.parametrize("four", [False, True])
def test_copies_of_the_handles_are_of_their_own_tensors(fv, four):
    """A deep copy of a pool is another pool, of a batch another batch; a shallow one has the same tensors."""
    import copy

    import torch

    announce(f"paged: copies four={four}")
    w = World(fv, 73, [20, 9], [2, 1], 2, 64, 16, four)
    before = [t.clone() for t in (w.pool.k, w.pool.v)]
    other, batch = copy.deepcopy(w.pool), copy.deepcopy(w.batch)
    assert other.k.data_ptr() != w.pool.k.data_ptr() and other.four_bits == four
    x = torch.full((3, 2, 64), 3.0, device="cuda", dtype=torch.bfloat16)
    batch.lens.fill_(1)                                          # (the copy's: the first token of a sequence, two rows of which one is it)
    fv.paged_append(other, batch, x, x)
    assert torch.equal(w.pool.k, before[0]) and torch.equal(w.pool.v, before[1])
    back = fv.paged_read(other, batch, 3)[0]
    assert not back[0].any() and (back[1:] == 3.0).all()
    assert w.batch.lens.tolist() == [20, 9] and (batch.max_q, batch.max_len) == (w.batch.max_q, w.batch.max_len)
    same = copy.copy(w.pool)
    fv.paged_append(same, copy.copy(w.batch), x, x)
    assert (fv.paged_read(w.pool, w.batch, 3)[0] == 3.0).all()
