"""The framework's q/k norm before the paged cache: its head planes merged back to tokens, stored as they are."""
import numpy as np
import pytest

from test_gpu_paged import tables
from util import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("in16", [False, True])
def test_norm_then_append(in16):
    """qk_norm_rope_bhsd (norm and rotation) -> merge_heads -> paged_append without tables, the values a slice of the projection:
    the pages hold what an sdpa call on the producers' tensors is given."""
    import torch

    import fv_sdpa as fv

    announce(f"paged: norm, merge, append in16={in16}")
    heads, d, page, n = 6, 128, 32, 70
    g = torch.Generator(device="cuda").manual_seed(5)
    proj = torch.randn((2, n, 3 * heads * d), generator=g, device="cuda").to(torch.bfloat16 if in16 else torch.float32)
    weight = 1 + 0.1 * torch.randn(heads * d, generator=g, device="cuda")
    cos, sin = (torch.from_numpy(t).cuda() for t in tables(n, d, False))
    q, k = (fv.qk_norm_rope_bhsd(proj, c * heads * d, heads, weight.to(proj.dtype), rope=(cos, sin)) for c in (0, 1))
    tokens = [fv.merge_heads(x).view(2 * n, heads, d) for x in (q, k)]
    v = proj[:, :, 2 * heads * d:].unflatten(2, (heads, d))
    i32 = {"dtype": torch.int32, "device": "cuda"}
    pool, table = fv.PagedKv.new(2 * 3, page, heads, d), torch.arange(6, **i32).view(2, 3)
    batch = fv.PagedBatch(torch.tensor([0, n, 2 * n], **i32), torch.tensor([n, n], **i32), table, n, n)
    assert fv.paged_append(pool, batch, tokens[1], v.reshape(2 * n, heads, d)) is None
    first = fv.PagedBatch(torch.tensor([0, n], **i32), torch.tensor([n], **i32), table[:1], n, n)
    fv.paged_append(pool, first, tokens[1][:n], v[0])             # (tokens of the projection, as they lie)
    back = fv.paged_read(pool, batch, 2 * n)
    planes = [x.bfloat16().transpose(1, 2).reshape(2 * n, heads, d) for x in (k, fv.split_heads_bhsd(proj, 2 * heads * d, heads, d))]
    assert torch.equal(back[0], planes[0]) and torch.equal(back[1], planes[1])
    got = fv.paged_attention(tokens[0].bfloat16(), pool, batch, fv.BlockCausal(14)).view(2, n, heads, d).transpose(1, 2)
    flat = [x.bfloat16().reshape(2 * heads, n, d).contiguous() for x in (q, k, fv.split_heads_bhsd(proj, 2 * heads * d, heads, d))]
    want = fv.sdpa_block_causal_bf16(*flat, 14).view(2, heads, n, d)
    mag = fv.sdpa_block_causal_bf16(flat[0], flat[1], flat[2].abs(), 14).view(2, heads, n, d)
    # both round their probabilities to bf16 (2^-8 of each term), one rounds its result (2^-8); scores in f32 besides
    off = (got.float() - want).abs() - (2 * 2.0 ** -8 + 2.0 ** -10) * mag - 2.0 ** -8 * want.abs()
    worst = float(off.max())
    assert worst <= 0 and np.isfinite(worst)
