"""The paged KV cache's entries refuse what they cannot take, on the host, before anything is launched. No GPU: the pointers
are numbers that nothing follows."""
import ctypes as C

import pytest

import util  # noqa: F401  (puts the package on the path)
from fv_sdpa import _lib

P = 1 << 20          # an aligned address
INVALID, DECLINED = -1, 1


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


BASE = dict(pages=10, page_tokens=16, kv_heads=2, d=128, table_stride=8, table_pages=8, seqs=3, tokens=5)
APPEND = dict(k=P, k_stride=256, v=P, v_stride=256, q=None, q_stride=0, q_out=None, in_is_bf16=1, heads=0, cos_t=P, sin_t=P, rope_rows=64,
              rope_at=None, halves=0)
POOL = dict(k_pages=P, v_pages=P, k_scales=None, v_scales=None)
SEQS = dict(q_start=P, lens=P, table=P)
ATTEND = dict(q=P, q_stride=512, out=P, out_is_bf16=1, heads=4)
MASK = dict(max_q=2, max_len=100, scale=0.1, block_tokens=1, window=0, sink=0, workspace=None, workspace_bytes=0)
READ = dict(k_out=P, v_out=P, out_is_bf16=1)
ORDER = {
    "fv_paged_append": [*APPEND, *POOL, "pages", "page_tokens", "kv_heads", "d", *SEQS, "table_stride", "table_pages", "seqs", "tokens"],
    "fv_paged_read": [*READ, *POOL, "pages", "page_tokens", "kv_heads", "d", *SEQS, "table_stride", "table_pages", "seqs", "tokens"],
    "fv_paged_attention": [*ATTEND, *POOL, "pages", "page_tokens", "kv_heads", "d", *SEQS, "table_stride", "table_pages", "seqs", "tokens", *MASK],
}
OWN = {"fv_paged_append": APPEND, "fv_paged_read": READ, "fv_paged_attention": {**ATTEND, **MASK}}


def call(lib, name, **change):
    args = {**BASE, **POOL, **SEQS, **OWN[name], **change}
    assert set(change) <= set(ORDER[name]), change
    rc = getattr(lib, name)(*[args[n] for n in ORDER[name]], None)
    return rc, lib.fv_sdpa_last_error().decode()


ALL = sorted(ORDER)


@pytest.mark.parametrize("name", ALL)
@pytest.mark.parametrize("change,rc,text", [
    (dict(k_pages=None), INVALID, "null operand"), (dict(v_pages=None), INVALID, "null operand"), (dict(q_start=None), INVALID, "null operand"),
    (dict(lens=None), INVALID, "null operand"), (dict(table=None), INVALID, "null operand"),
    (dict(k_scales=P), INVALID, "scales of keys and values go together"), (dict(v_scales=P), INVALID, "scales of keys and values go together"),
    (dict(d=96), DECLINED, "head dim"), (dict(d=0), DECLINED, "head dim"), (dict(d=256), DECLINED, "head dim"),
    (dict(page_tokens=8), DECLINED, "power of two"), (dict(page_tokens=48), DECLINED, "power of two"), (dict(page_tokens=1 << 17), DECLINED, "power of two"),
    (dict(page_tokens=0), DECLINED, "power of two"),
    (dict(pages=0), INVALID, "empty pool"), (dict(kv_heads=0), INVALID, "empty pool"), (dict(pages=1 << 31), DECLINED, "too large"),
    (dict(pages=1 << 28), DECLINED, "too large"),
    (dict(k_pages=P + 8), INVALID, "16-byte aligned"), (dict(k_scales=P, v_scales=P + 4), INVALID, "16-byte aligned"),
    (dict(table_pages=9), INVALID, "shorter than their pages"), (dict(table_pages=1 << 28, table_stride=1 << 28), DECLINED, "too wide"),
    (dict(tokens=1 << 27), DECLINED, "too many"), (dict(seqs=1 << 25), DECLINED, "too many"),
])
def test_pool_and_batch(lib, name, change, rc, text):
    got, said = call(lib, name, **change)
    assert got == rc and text in said, (got, said)


@pytest.mark.parametrize("change,rc,text", [
    (dict(k=None), INVALID, "null operand"), (dict(v=None), INVALID, "null operand"), (dict(q=P), INVALID, "without a place"),
    (dict(q_out=P), INVALID, "without a place"), (dict(sin_t=None), INVALID, "one rope table"), (dict(cos_t=None), INVALID, "one rope table"),
    (dict(q=P, q_out=P, heads=0, q_stride=512), INVALID, "without heads"), (dict(k_stride=248), INVALID, "overlap"), (dict(v_stride=0), INVALID, "overlap"),
    (dict(q=P, q_out=P, heads=4, q_stride=504), INVALID, "overlap"), (dict(k_stride=260), DECLINED, "multiples of 8"),
    (dict(q=P, q_out=P, heads=4, q_stride=514), DECLINED, "multiples of 8"), (dict(v_stride=1 << 31), DECLINED, "multiples of 8"),
    (dict(k=P + 2), INVALID, "16-byte aligned"), (dict(cos_t=P + 4), INVALID, "16-byte aligned"), (dict(rope_rows=1 << 31), DECLINED, "too long"),
    (dict(q=P, q_out=P, heads=1 << 16, q_stride=1 << 24), DECLINED, "too many heads"),
    (dict(tokens=1 << 24), DECLINED, "too large for one launch"),
])
def test_append(lib, change, rc, text):
    got, said = call(lib, "fv_paged_append", **change)
    assert got == rc and text in said, (got, said)


@pytest.mark.parametrize("change,rc,text", [
    (dict(q=None), INVALID, "null operand"), (dict(out=None), INVALID, "null operand"), (dict(heads=0), INVALID, "multiple of the key heads"),
    (dict(heads=3), INVALID, "multiple of the key heads"), (dict(q_stride=504), INVALID, "overlap"), (dict(q_stride=516), DECLINED, "multiple of 8"),
    (dict(q=P + 8), INVALID, "16-byte aligned"), (dict(out=P + 2), INVALID, "16-byte aligned"), (dict(scale=0.0), DECLINED, "scale"),
    (dict(scale=-1.0), DECLINED, "scale"), (dict(scale=float("inf")), DECLINED, "scale"), (dict(scale=float("nan")), DECLINED, "scale"),
    (dict(block_tokens=0), INVALID, "block_tokens"), (dict(window=1 << 31), DECLINED, "mask too large"), (dict(sink=1 << 31), DECLINED, "mask too large"),
    (dict(block_tokens=1 << 31), DECLINED, "mask too large"), (dict(max_len=129), INVALID, "past the table"),
    (dict(heads=1 << 16, q_stride=1 << 24), DECLINED, "too many heads"),
])
def test_attention(lib, change, rc, text):
    got, said = call(lib, "fv_paged_attention", **change)
    assert got == rc and text in said, (got, said)


@pytest.mark.parametrize("change,rc,text", [(dict(k_out=None), INVALID, "null operand"), (dict(v_out=P + 8), INVALID, "16-byte aligned"),
                                            (dict(tokens=1 << 24, kv_heads=64), DECLINED, "too large for one launch")])
def test_read(lib, change, rc, text):
    got, said = call(lib, "fv_paged_read", **change)
    assert got == rc and text in said, (got, said)


@pytest.mark.parametrize("name", ALL)
def test_nothing_to_do(lib, name):
    """No rows or no sequences: nothing is looked at, not even the addresses (empty arrays have none)."""
    none = dict(q_start=None, lens=None, table=None)
    assert call(lib, name, tokens=0, **none)[0] == 0
    assert call(lib, name, seqs=0, **none)[0] == 0
    if name == "fv_paged_attention":
        assert call(lib, name, max_q=0)[0] == 0


def test_a_workspace_that_is_not_aligned_is_refused(lib):
    size = lib.fv_paged_attention_workspace_bytes(4, 2, 128, 1, 1, 1, 100000, 1, 0, 0)
    assert size > 0
    wide = dict(table_stride=6250, table_pages=6250, seqs=1, tokens=1, max_q=1, max_len=100000)
    got, said = call(lib, "fv_paged_attention", workspace=P + 16, workspace_bytes=size, **wide)
    assert got == INVALID and "256-byte aligned" in said


def test_workspace_bytes(lib):
    """None for short or empty calls and for numbers that no call takes; more shares, more bytes."""
    need = lib.fv_paged_attention_workspace_bytes
    assert need(4, 2, 128, 3, 5, 2, 100, 1, 0, 0) == 0
    assert need(3, 2, 128, 3, 5, 2, 1 << 20, 1, 0, 0) == 0
    assert need(4, 0, 128, 3, 5, 2, 1 << 20, 1, 0, 0) == 0
    assert need(4, 2, 128, 0, 5, 2, 1 << 20, 1, 0, 0) == 0
    assert need(4, 2, 128, 3, 0, 2, 1 << 20, 1, 0, 0) == 0
    assert need(4, 2, 128, 3, 5, 0, 1 << 20, 1, 0, 0) == 0
    assert need(4, 2, 128, 3, 5, 2, 1 << 20, 0, 0, 0) == 0
    long, longer = need(4, 2, 128, 1, 1, 1, 100000, 1, 0, 0), need(4, 2, 128, 1, 1, 1, 1 << 20, 1, 0, 0)
    assert 0 < long < longer and need(4, 2, 128, 1, 1, 1, 1 << 20, 1, 512, 4) == 0


def test_signatures_name_every_argument():
    assert len(_lib.SIGNATURES["fv_paged_append"][1]) == len(ORDER["fv_paged_append"]) + 1
    assert len(_lib.SIGNATURES["fv_paged_attention"][1]) == len(ORDER["fv_paged_attention"]) + 1
    assert all(t in (C.c_void_p, C.c_size_t, C.c_int, C.c_float) for t in _lib.SIGNATURES["fv_paged_attention"][1])


def test_workspace_of_long_and_short_sequences(lib):
    """256 single tokens on up to 131072 keys (32 shares of their 16 rows a key head at most) beside a longer one: the shares take no more
    than that and a gigabyte for the longer one, whose length does not count for the others."""
    few = 32 * 256 * 8 * 16 * (128 * 4 + 4)
    for longest in (1, 4, 100, 2048, 8192):
        need = lib.fv_paged_attention_workspace_bytes(40, 8, 128, 256, 255 + longest, longest, 131072, 1, 0, 0)
        assert 0 < need <= few + (1 << 30) * 129 // 128 + 1024, longest
