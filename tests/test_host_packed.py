"""The entries for packed sequences and rotary positions refuse what they cannot take, on the host, before anything is launched, and say how much
workspace they want. No GPU: the pointers are numbers that nothing follows."""
import ctypes as C

import numpy as np
import pytest

import util  # noqa: F401  (puts the package on the path)
import packed_util as pu
from fv_sdpa import _lib

P = 1 << 20          # an aligned address
INVALID, DECLINED = -1, 1


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


SIZES = dict(heads=4, kv_heads=2, d=128, q_start=P, k_start=P, seqs=3, q_tokens=50, k_tokens=60, max_q=20, max_k=30, scale=0.1, causal=1, block_tokens=1,
             window=0, sink=0, workspace=None, workspace_bytes=0)
QKV = dict(q=P, q_stride=512, k=P, k_stride=256, v=P, v_stride=256)
ORDER = {
    "fv_packed_attention": [*QKV, "out", "out_is_bf16", "lse", *SIZES],
    "fv_packed_attention_backward": ["dout", "dout_is_bf16", *QKV, "out", "out_is_bf16", "lse", "dq", "dk", "dv", "grads_are_bf16", *SIZES],
    "fv_rope_tokens": ["q", "q_stride", "q_out", "q_out_stride", "heads", "k", "k_stride", "k_out", "k_out_stride", "kv_heads", "d", "in_is_bf16", "out_is_bf16",
                       "freq", "pair_axis", "pairs", "positions", "axes", "tokens", "amplitude", "halves", "inverse"],
}
OWN = {
    "fv_packed_attention": {**SIZES, **QKV, "out": P, "out_is_bf16": 1, "lse": None},
    "fv_packed_attention_backward": {**SIZES, **QKV, "dout": P, "dout_is_bf16": 1, "out": P, "out_is_bf16": 1, "lse": P, "dq": P, "dk": P, "dv": P, "grads_are_bf16": 1},
    "fv_rope_tokens": dict(q=P, q_stride=512, q_out=2 * P, q_out_stride=512, heads=4, k=P, k_stride=256, k_out=2 * P, k_out_stride=256, kv_heads=2, d=128, in_is_bf16=1,
                           out_is_bf16=1, freq=P, pair_axis=None, pairs=64, positions=P, axes=1, tokens=10, amplitude=1.0, halves=0, inverse=0),
}


def call(lib, name, **change):
    args = {**OWN[name], **change}
    assert set(change) <= set(ORDER[name]), change
    rc = getattr(lib, name)(*[args[n] for n in ORDER[name]], None)
    return rc, lib.fv_sdpa_last_error().decode()


BOTH = ["fv_packed_attention", "fv_packed_attention_backward"]


@pytest.mark.parametrize("name", BOTH)
@pytest.mark.parametrize("change,rc,text", [
    (dict(q=None), INVALID, "null operand"), (dict(k=None), INVALID, "null operand"), (dict(v=None), INVALID, "null operand"), (dict(out=None), INVALID, "null operand"),
    (dict(q_start=None), INVALID, "null operand"), (dict(k_start=None), INVALID, "null operand"),
    (dict(heads=3), INVALID, "multiple of the key heads"), (dict(heads=0), INVALID, "multiple of the key heads"), (dict(kv_heads=0), INVALID, "multiple of the key heads"),
    (dict(d=96), DECLINED, "head dim"), (dict(d=0), DECLINED, "head dim"), (dict(d=256), DECLINED, "head dim"),
    (dict(heads=65536, q_stride=65536 * 128), DECLINED, "too many heads"), (dict(seqs=1 << 25), DECLINED, "too many"), (dict(q_tokens=1 << 27), DECLINED, "too many"),
    (dict(k_tokens=1 << 27), DECLINED, "too many"), (dict(q_tokens=1 << 26, heads=64, q_stride=64 * 128), DECLINED, "too many"),
    (dict(scale=0.0), DECLINED, "scale"), (dict(scale=-1.0), DECLINED, "scale"), (dict(scale=float("nan")), DECLINED, "scale"), (dict(scale=float("inf")), DECLINED, "scale"), (dict(scale=1e-31), DECLINED, "scale"), (dict(scale=1e31), DECLINED, "scale"),
    (dict(block_tokens=0), INVALID, "block_tokens"), (dict(window=1 << 31), DECLINED, "mask too large"), (dict(sink=1 << 31), DECLINED, "mask too large"),
    (dict(q=P + 8), INVALID, "16-byte aligned"), (dict(v=P + 2), INVALID, "16-byte aligned"), (dict(out=P + 4), INVALID, "16-byte aligned"),
    (dict(q_stride=504), INVALID, "tokens overlap"), (dict(k_stride=0), INVALID, "tokens overlap"), (dict(v_stride=260), DECLINED, "multiples of 8"),
    (dict(k_stride=(1 << 24) + 8), DECLINED, "2^24"), (dict(workspace=P + 16), INVALID, "256-byte aligned"),
])
def test_operands(lib, name, change, rc, text):
    got, said = call(lib, name, **change)
    assert got == rc and text in said, (got, said)


@pytest.mark.parametrize("change,text", [
    (dict(dout=None), "null operand"), (dict(lse=None), "null operand"), (dict(dq=None), "null operand"), (dict(dk=None), "null operand"), (dict(dv=None), "null operand"),
    (dict(dq=P + 8), "16-byte aligned"), (dict(), "workspace too small"), (dict(workspace=P, workspace_bytes=1000), "workspace too small")])
def test_backward_operands(lib, change, text):
    got, said = call(lib, "fv_packed_attention_backward", **change)
    assert got == INVALID and text in said, (got, said)


def test_empty_calls_follow_no_address(lib):
    for name in BOTH:
        for change in (dict(seqs=0), dict(q_tokens=0, k_tokens=0)):
            none = {n: None for n in ("q", "k", "v", "out", "q_start", "k_start")}
            assert call(lib, name, **none, **change)[0] == 0
    assert call(lib, "fv_packed_attention", q=None, max_q=0)[0] == 0
    assert call(lib, "fv_rope_tokens", q=None, freq=None, tokens=0)[0] == 0


def test_workspaces(lib):
    f, b = lib.fv_packed_attention_workspace_bytes, lib.fv_packed_attention_backward_workspace_bytes
    one = (8, 1, 128, 1, 1, 100_000, 1, 100_000, 1, 1, 0, 0)     # one token on many keys: its walk is cut
    assert f(*one) > 0 and f(*one) % 256 == 0
    assert f(32, 32, 128, 64, 64 * 512, 64 * 512, 512, 512, 1, 1, 0, 0) == 0     # walks enough for all units
    # numbers that no call takes: 0, without overflow
    for change in ({2: 96}, {0: 3}, {1: 0}, {3: 1 << 30}, {4: 1 << 40}, {5: 1 << 40}, {9: 0}, {10: 1 << 40}):
        numbers = [change.get(i, x) for i, x in enumerate(one)]
        if 0 in change:
            numbers[1] = 2
        assert f(*numbers) == 0 and b(1, *numbers) == 0, change
    # statistics of every row at least; a gradient in f32 is kept as bf16
    train = (32, 8, 128, 5, 20_000, 20_000, 6000, 6000, 1, 1, 0, 0)
    rows = 20_000 * 32
    assert b(1, *train) >= rows * 8 and rows * 256 <= b(0, *train) - b(1, *train) < rows * 256 + 512
    # what the cut walks leave is bounded by the units, not by the batch: 1 GB is far above it
    for tokens in (1000, 100_000, 5_000_000):
        n = (40, 8, 128, 7, tokens, tokens, tokens, tokens, 1, 1, 1024, 4)
        assert b(1, *n) < tokens * 40 * 8 + (1 << 29) + tokens * 8, tokens


@pytest.mark.parametrize("change,rc,text", [
    (dict(q=None), INVALID, "null operand"), (dict(q_out=None), INVALID, "null operand"), (dict(freq=None), INVALID, "null operand"), (dict(positions=None), INVALID, "null operand"),
    (dict(k=None), INVALID, "or the reverse"), (dict(k_out=None), INVALID, "or the reverse"), (dict(heads=0), INVALID, "no heads"), (dict(kv_heads=0), INVALID, "no heads"),
    (dict(d=100), DECLINED, "head dim"), (dict(d=0), DECLINED, "head dim"), (dict(d=8192), DECLINED, "head dim"), (dict(pairs=12), DECLINED, "pairs"), (dict(pairs=0), DECLINED, "pairs"),
    (dict(pairs=72), INVALID, "more pairs"), (dict(axes=0), INVALID, "axes"), (dict(axes=5), INVALID, "axes"), (dict(heads=70000, q_stride=70000 * 128, q_out_stride=70000 * 128), DECLINED, "heads"),
    (dict(tokens=1 << 27), DECLINED, "too many tokens"), (dict(tokens=1 << 26, d=4096, pairs=8, heads=1, q_stride=4096, q_out_stride=4096, kv_heads=1, k_stride=4096, k_out_stride=4096), DECLINED, "too many tokens"),
    (dict(amplitude=0.0), INVALID, "amplitude"), (dict(amplitude=float("nan")), INVALID, "amplitude"), (dict(q=P + 8), INVALID, "16-byte aligned"), (dict(k_out=P + 4), INVALID, "16-byte aligned"),
    (dict(q_stride=504), INVALID, "tokens overlap"), (dict(k_out_stride=100), INVALID, "tokens overlap"), (dict(k_stride=260), DECLINED, "multiples of 8"),
    (dict(q_out=P, out_is_bf16=0), INVALID, "in place"), (dict(q_out=P, q_out_stride=520), INVALID, "in place"), (dict(k_out=P, k_out_stride=264), INVALID, "in place"),
])
def test_rope_operands(lib, change, rc, text):
    got, said = call(lib, "fv_rope_tokens", **change)
    assert got == rc and text in said, (got, said)


def test_rope_frequencies(lib):
    out = (C.c_uint64 * 64)()
    ok = dict(pairs=64, base=10000.0, scaling=0, factor=1.0, original=1.0, low=0.0, high=1.0)

    def freq(**change):
        return lib.fv_rope_frequencies(*{**ok, **change}.values(), out), lib.fv_sdpa_last_error().decode()

    for change, text in ((dict(pairs=0), "pairs"), (dict(pairs=1 << 20), "pairs"), (dict(base=0.5), "base"), (dict(base=float("nan")), "base"), (dict(base=float("inf")), "base"),
                         (dict(scaling=4), "scaling"), (dict(scaling=-1), "scaling"), (dict(scaling=1, factor=0.5), "factor"), (dict(scaling=1, factor=float("nan")), "factor"),
                         (dict(scaling=2, pairs=1, factor=2.0), "two pairs"), (dict(scaling=3, factor=2.0, original=0.0), "original"), (dict(scaling=3, factor=2.0, low=2.0), "original")):
        rc, said = freq(**change)
        assert rc == INVALID and text in said, (change, rc, said)
    assert lib.fv_rope_frequencies(64, 10000.0, 0, 1.0, 1.0, 0.0, 1.0, None) == INVALID
    for scaling, numbers in ((None, (0, 1.0, 1.0, 0.0, 1.0)), (("linear", 3.0), (1, 3.0, 1.0, 0.0, 1.0)), (("base", 8.0), (2, 8.0, 1.0, 0.0, 1.0)),
                             (("parts", 8.0, 8192, 1.0, 32.0), (3, 8.0, 8192.0, 1.0, 32.0))):
        assert lib.fv_rope_frequencies(64, 10000.0, *numbers, out) == 0
        turns = pu.frequencies(64, 10000.0, scaling) / pu.TURN
        # half a unit of 2^-64 turns and a few roundings of 2^-64 of extended precision
        assert all(abs(np.longdouble(int(x)) / np.longdouble(2) ** 64 - t) <= np.longdouble(2) ** -65 + 16 * np.longdouble(2) ** -64 * t for x, t in zip(out, turns))


def test_the_plain_forms_agree_with_differences():
    """packed_util.gradients, which the kernels are compared with, against differences of packed_util.attention in 64 bits."""
    rng = np.random.Generator(np.random.PCG64(0))
    q, k, v, g = (rng.standard_normal((n, 8)) for n in (7, 9, 9, 7))
    for mask in ((False,), (True,), (True, 1, 3, 1), (True, 2, 2, 0)):
        seen = pu.visible(7, 9, *mask)
        out, lse = pu.attention(q, k, v, seen, 0.3, False)[:2]
        grads = pu.gradients(q, k, v, g, out, lse, seen, 0.3)[:3]
        for i, x in enumerate((q, k, v)):
            for _ in range(5):
                u = rng.standard_normal(x.shape)
                ops = [[q, k, v], [q, k, v]]
                for sign, o in zip((1, -1), ops):
                    o[i] = x + sign * 1e-6 * u
                diff = sum(sign * (pu.attention(*o, seen, 0.3, False)[0] * g).sum() for sign, o in zip((1, -1), ops)) / 2e-6
                assert abs(diff - (grads[i] * u).sum()) < 1e-7 * (1 + np.abs(grads[i] * u).sum())
