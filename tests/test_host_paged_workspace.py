"""The workspace of attention over pages: of the call's own kind of pages. Host arithmetic, no GPU."""
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
    need = lib.fv_paged_attention_workspace_bytes_for
    for kind in (0, 1):
        for bad in (dict(heads=3), dict(kv_heads=0), dict(seqs=0), dict(tokens=0), dict(max_q=0), dict(block=0)):
            n = {"heads": 4, "kv_heads": 2, "d": 128, "seqs": 3, "tokens": 5, "max_q": 2, "max_len": 1 << 20, "block": 1, "window": 0, "sink": 0, **bad}
            assert need(kind, *n.values()) == 0, bad
