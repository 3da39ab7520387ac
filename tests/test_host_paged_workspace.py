"""The workspace of attention over pages: of the call's own kind of pages, and limited. Host arithmetic, no GPU."""
import itertools

import pytest

import util  # noqa: F401  (puts the package on the path)
from fv_sdpa import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


@pytest.mark.parametrize("seqs,rows", [(64, 9), (256, 12)])
def test_drafts_over_bf16_pages_need_none(lib, seqs, rows):
    """40 / 8 heads, up to 131072 keys: over bf16 pages they are the tiles', whose walks fill the chip uncut; over 4 bits the
    few rows' kernel cuts its long walks."""
    numbers = (40, 8, 128, seqs, seqs * rows, rows, 131072, 1, 0, 0)
    bf16, four = (lib.fv_paged_attention_workspace_bytes_for(kind, *numbers) for kind in (0, 1))
    assert bf16 == 0 and four > 0


def test_either_kind(lib):
    """The entry without a kind is enough for both, and no more."""
    for seqs, rows, longest, heads, window in itertools.product((1, 7, 64, 300), (1, 5, 20, 1000), (100, 5000, 131072), ((12, 12), (40, 8), (16, 1)), (0, 4096)):
        numbers = (*heads, 128, seqs, seqs * rows, rows, longest, 1, window, 4)
        bf16, four = (lib.fv_paged_attention_workspace_bytes_for(kind, *numbers) for kind in (0, 1))
        assert lib.fv_paged_attention_workspace_bytes(*numbers) == max(bf16, four), numbers


def test_nothing_for_numbers_that_no_call_takes(lib):
    """Numbers among them whose products pass 64 bits."""
    base = {"heads": 4, "kv_heads": 2, "d": 128, "seqs": 3, "tokens": 5, "max_q": 2, "max_len": 1 << 20, "block": 1, "window": 0, "sink": 0}
    far = [{name: n} for name in ("heads", "seqs", "tokens", "max_len", "block", "window", "sink") for n in (1 << 31, 1 << 61, (1 << 64) - 2)]
    for kind in (0, 1):
        assert lib.fv_paged_attention_workspace_bytes_for(kind, *base.values()) > 0
        for bad in (dict(heads=3), dict(kv_heads=0), dict(seqs=0), dict(tokens=0), dict(max_q=0), dict(block=0), dict(d=0), dict(d=96), *far):
            assert lib.fv_paged_attention_workspace_bytes_for(kind, *{**base, **bad}.values()) == 0, bad
            assert lib.fv_paged_attention_workspace_bytes(*{**base, **bad}.values()) == 0, bad
        every = lib.fv_paged_attention_workspace_bytes_for(kind, *{**base, "max_q": (1 << 64) - 1}.values())   # (cut to the rows)
        assert every == lib.fv_paged_attention_workspace_bytes_for(kind, *{**base, "max_q": 5}.values())


def test_shares_are_limited(lib):
    """Whatever the bounds: a gigabyte of shares for each of the two kernels, a sum beside every row of them (1 / d of that), and
    what rounding to 256 bytes adds."""
    worst = 0
    for kind, d, (heads, kvh) in itertools.product((0, 1), (64, 128), ((40, 8), (64, 8), (12, 12), (16, 1), (32, 2))):
        for seqs, rows, most in itertools.product((1, 16, 256, 1024, 20000), (1, 2, 12, 60), (None, 700, 8192)):
            for longest, window in itertools.product((4096, 131072, 1 << 20, (1 << 31) - 64), (0, 100000)):
                tokens, max_q = (seqs * rows, rows) if most is None else (seqs - 1 + most, most)
                worst = max(worst, lib.fv_paged_attention_workspace_bytes_for(kind, heads, kvh, d, seqs, tokens, max_q, longest, 1, window, 4))
    assert worst <= 2 * ((1 << 30) * 65 // 64 + 512), worst
    # (9.7 GB for 19 MB of results without the limit; these are cut as far as it lets them)
    drafts = lib.fv_paged_attention_workspace_bytes_for(1, 32, 8, 128, 256, 256 * 9, 9, 1 << 20, 1, 0, 0)
    assert (1 << 29) < drafts <= (1 << 30) * 129 // 128 + 512


def test_the_largest_numbers(lib):
    """Each bound of a call at its largest, all at once too: a gigabyte a kernel, or none."""
    most = {"heads": 65534, "kv_heads": 32767, "d": 128, "seqs": 1 << 24, "tokens": 1 << 26, "max_q": 1 << 26, "max_len": (1 << 31) - 1,
            "block": (1 << 30) - 1, "window": (1 << 30) - 1, "sink": (1 << 30) - 1}
    base = {"heads": 40, "kv_heads": 8, "d": 128, "seqs": 64, "tokens": 300, "max_q": 100, "max_len": 1 << 20, "block": 1, "window": 0, "sink": 0}
    some = [dict(base, **{n: most[n]}) for n in most if n not in ("heads", "kv_heads")] + [dict(base, heads=65535, kv_heads=1), dict(base, heads=65535, kv_heads=65535)]
    for kind in (0, 1):
        for numbers in (*some, most, dict(most, block=1), dict(most, window=0), dict(most, window=0, heads=65535, kv_heads=1), dict(most, max_q=1)):
            need = lib.fv_paged_attention_workspace_bytes_for(kind, *numbers.values())
            assert need <= 2 * ((1 << 30) * 129 // 128 + 512), numbers
