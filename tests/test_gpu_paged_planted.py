"""Attention over pages loses no key and counts none twice: results that every key has a part in, or that one key decides, at the borders of
shares, steps, tiles, pages, windows and sinks, in both kernels, with walks in shares and whole."""
import numpy as np
import pytest

import paged_planted as pp
import paged_util as pu
from test_gpu_paged import World
from util import announce

pytestmark = pytest.mark.gpu

# lens, counts, heads, key heads, d, page, mask
CASES = {
    "tokens": ([9001, 300, 20000], [1, 1, 2], 8, 1, 128, 64, (1, 0, 0)),
    "tokens_pages_of_16": ([9007, 33], [1, 1], 12, 4, 128, 16, (1, 0, 0)),
    "tokens_64": ([12345, 4000], [2, 1], 6, 2, 64, 32, (1, 0, 0)),
    "tokens_window": ([9001, 7000], [1, 2], 8, 2, 128, 64, (1, 4500, 70)),
    "tokens_blocks": ([8000, 3001], [1, 3], 4, 1, 128, 128, (100, 40, 2)),
    "drafts": ([9001, 5000], [9, 3], 8, 2, 128, 64, (1, 0, 0)),
    "drafts_64": ([6011, 2000], [5, 12], 10, 2, 64, 16, (1, 3000, 5)),
    "rows": ([9000], [150], 4, 2, 128, 64, (1, 0, 0)),
    "rows_window": ([7000, 5000], [64, 100], 4, 2, 128, 16, (1, 4500, 70)),
    "rows_64": ([8111], [100], 6, 3, 64, 32, (1, 0, 0)),
    "frame": ([4680], [1560], 2, 1, 128, 64, (1560, 0, 0)),
    "prompt": ([2500, 700], [2500, 700], 2, 2, 128, 64, (1, 900, 30)),
    "mixed": ([9000, 4000, 500, 777, 12000, 31, 64, 2000], [200, 1, 1, 1, 2, 1, 1, 1], 8, 2, 128, 64, (1, 0, 0)),
}


@pytest.fixture(scope="module")
def fv():
    import torch

    assert torch.cuda.is_available()
    import fv_sdpa

    fv_sdpa.lib()
    return fv_sdpa


def world(fv, case, four, seed):
    lens, counts, heads, kvh, d, page, mask = CASES[case]
    return World(fv, seed, lens, counts, kvh, d, page, four, fill="nan")


def store(w, name, s, x):
    """x [len, kv_heads, d] into the host copy of sequence s's pages."""
    j = np.arange(w.lens[s])
    p, t = w.table[s, j // w.page], j % w.page
    if w.four:
        w.host[name][p, :, t], w.scales[name][p, :, t] = pu.quantize4(x)
    else:
        w.host[name][p, :, t] = pu.bf16(x)


def attend(fv, w, q, case, split):
    """f32 results with the workspace that the entry asks for, or (walks whole) with none."""
    import torch

    lens, counts, heads, kvh, d, page, mask = CASES[case]
    block, window, sink = mask
    rows, max_q, max_len = w.rows(), max(counts), max(lens)
    need = fv.lib().fv_paged_attention_workspace_bytes_for(w.four, heads, kvh, d, len(lens), rows, max_q, max_len, block, window, sink)
    assert need > 0, case   # (some walk is cut)
    if split:
        return fv.paged_attention(q, w.pool, w.batch, fv.BlockCausal(*mask), out_bf16=False)
    out = torch.full((rows, heads, d), float("nan"), device="cuda")
    rc = fv.lib().fv_paged_attention(q.data_ptr(), heads * d, out.data_ptr(), 0, heads, *w.pool._args, *w.batch._args, rows, max_q, max_len, d ** -0.5,
                                     block, window, sink, None, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    return out


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("case", sorted(CASES))
def test_every_key_counts_once(fv, case, four):
    import torch

    announce(f"paged: every key once {case} four={four}")
    lens, counts, heads, kvh, d, page, mask = CASES[case]
    for way in (0, 1):
        w = world(fv, case, four, 901)
        for s, n in enumerate(lens):
            store(w, "v", s, pp.marks(n, kvh, d, way))
        w.push()
        q = torch.zeros((w.rows(), heads, d), device="cuda", dtype=torch.bfloat16)
        want = np.concatenate([pp.mark_shares(n, c, d, way, mask) for n, c in zip(lens, counts)])[:, None]
        for split in (True, False):
            got = attend(fv, w, q, case, split).cpu().numpy().astype(np.float64)
            off = np.abs(got - want) - pp.MARK_TOLERANCE * want
            worst = float(off.max())
            assert worst <= 0, f"way {way}, split {split}: off by {worst} past the tolerance at {np.unravel_index(off.argmax(), off.shape)}"


def definition(q, k, v, seen, scale):
    """f64 on the device, head by head: (out, weights' sum of |v|)."""
    import torch

    out, mag = torch.empty_like(q), torch.empty_like(q)
    for h in range(q.shape[1]):
        kv = h * k.shape[1] // q.shape[1]
        s = (q[:, h] @ k[:, kv].T) * scale
        p = torch.softmax(s.masked_fill(~seen, -float("inf")), -1)
        out[:, h], mag[:, h] = p @ v[:, kv], p @ v[:, kv].abs()
    return out, mag


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("case", sorted(CASES))
def test_planted_keys_decide_their_rows(fv, case, four):
    import torch

    announce(f"paged: planted keys {case} four={four}")
    lens, counts, heads, kvh, d, page, mask = CASES[case]
    w = world(fv, case, four, 903)
    targets, held = [], []
    for s, n in enumerate(lens):
        keys = pu.bf16(w.rng.standard_normal((n, kvh, d)))
        targets.append(pp.plant(w.rng, keys, pp.borders(n, n - counts[s], mask)))
        store(w, "k", s, keys)
        held.append([w.dev(w.held(name, s)) for name in "kv"])
    w.push()
    seen = [w.dev(pu.sees(np.arange(c) + n - c, np.arange(n), *mask)) for n, c in zip(lens, counts)]
    calls = max(-(-len(t) // (c * heads)) for t, c in zip(targets, counts))
    worst = 0.0
    for call in range(calls):
        q = np.empty((w.rows(), heads, d), dtype=np.float32)
        for s, (t, c) in enumerate(zip(targets, counts)):       # (each row another target)
            q[w.starts[s]:w.starts[s] + c] = t[(np.arange(c * heads) + call * c * heads) % len(t)].reshape(c, heads, d)
        dq = w.dev(q).bfloat16()
        got = [attend(fv, w, dq, case, split).double() for split in (True, False)]
        for s, c in enumerate(counts):
            part = slice(int(w.starts[s]), int(w.starts[s]) + c)
            out, mag = definition(dq[part].double(), *held[s], seen[s], d ** -0.5)
            top = d ** -0.5 * 1.45 * 4 * float(held[s][0].abs().max()) * d
            # (as attention_bound)
            bound = (2.0 ** -8 + 2.0 * 130 * 2.0 ** -24 * top + 2.0 ** -12) * mag + 2.0 ** -24 * out.abs() + 1e-30
            for split, x in zip((True, False), got):
                off = float(((x[part] - out).abs() / bound).max())
                worst = max(worst, off)
                assert off <= 1, f"call {call}, sequence {s}, split {split}: {off} of the bound"
    print(f"[paged] planted {case} four={four}: {calls} calls, worst {worst:.3f} of the bound", flush=True)
