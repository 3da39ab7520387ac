"""Rotary positions over as many heads as a call takes: their pieces are a launch's second dimension, which is below 2^16."""
import numpy as np
import pytest

import packed_util as pu
from test_gpu_rope_tokens import check
from util import announce

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

if torch.cuda.is_available():
    import fv_sdpa


@pytest.mark.parametrize("heads", [(65535, 65535), (65535, 1), (65535, 0)], ids=str)
def test_most_heads(heads):
    announce(f"heads {heads}")
    rope = fv_sdpa.Rope(16)
    gen = torch.Generator(device="cuda").manual_seed(5)
    q, k = (torch.randn(2, h, 16, device="cuda", generator=gen).bfloat16() for h in heads)
    positions = torch.tensor([3, 70001], dtype=torch.int32, device="cuda")
    for n in (1, 2):
        y = fv_sdpa.rope_tokens(rope, positions[:n], q[:n], k[:n] if heads[1] else None)
        for x, got in zip((q, k), y if heads[1] else (y,)):
            check(rope, x[:n], got, positions[:n], np.asarray(pu.frequencies(8)), False, True, f"{n} tokens, heads {heads}")
