"""Training on packed sequences (include/fv_sdpa_hip.h, `fv_packed_*`, `fv_rope_*`; no counterpart in the reference): sequences of different
lengths one behind the other, attention with shared key heads inside each of them, its gradients, and rotary positions without tables. They
record no graph: a caller's autograd function calls them. Elsewhere, of tensors that autograd watches, the results are such that a gradient
asked for through them is an error (not silently left out), and a rotation in place is refused.
"""
import ctypes as C
import math
from operator import attrgetter

import torch
from torch.autograd.graph import increment_version

from . import _lib

__all__ = ["Rope", "rope_tokens", "PackedSeqs", "packed_attention", "packed_attention_backward"]

_BF16, _F32, _U8, _I32, _I64 = torch.bfloat16, torch.float32, torch.uint8, torch.int32, torch.int64
_SCALINGS = {"linear": 1, "base": 2, "parts": 3}


def _tokens(t, name, heads, d, device, dtypes=(_BF16,)):
    """(heads, elements between the tokens) of t [tokens, heads, d], whose heads are contiguous."""
    shape = t.shape
    if len(shape) != 3 or t.dtype not in dtypes or t.get_device() != device:
        raise ValueError(f"{name}: want a [tokens, heads, d] tensor of {' or '.join(str(x) for x in dtypes)} on cuda:{device}")
    n, h, dd = shape
    if (heads and h != heads) or dd != d:
        raise ValueError(f"{name}: want [tokens, {heads or 'heads'}, {d}], got {tuple(shape)}")
    if t.is_contiguous():
        return h, h * d
    a, b, c = t.stride()
    if c != 1 or (h > 1 and b != d):
        raise ValueError(f"{name}: the heads of a token must be contiguous")
    return h, a if n > 1 else h * d


def _like(t, dtype):
    """An uninitialised contiguous [tokens, heads, d] beside a checked t (empty_like, where it serves, is the shorter call; it lays slices out densely)."""
    return torch.empty_like(t) if t.dtype is dtype else torch.empty(t.shape, device=t.device, dtype=dtype)


def _on(device, name):
    if device < 0:
        raise ValueError(f"{name}: want CUDA tensors")
    if torch._C._cuda_getDevice() != device:
        raise ValueError(f"{name}: the tensors are on cuda:{device}, which is not the current device")


def _watched(a, b=None, c=None):
    """Whether autograd would record a call on these tensors."""
    return (a.requires_grad or (b is not None and b.requires_grad) or (c is not None and c.requires_grad)) and torch.is_grad_enabled()


class _NoGraph(torch.autograd.Function):
    """The results of call() (which runs with autograd off) for tensors that autograd watches: their backward says what is missing."""

    @staticmethod
    def forward(ctx, name, call, *watched):
        ctx.name = name
        return call()

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.name} records no graph: its gradient goes through an autograd function of the caller's (or call it under torch.no_grad())")


class Rope:
    """The frequencies of a rotation: the first `rot` channels of a head (default: all d) in pairs (2i, 2i + 1), or with `halves` (i, i +
    rot / 2), pair i of n = rot / 2 turned by base^(-i / n) a position. scaling, for longer contexts: None, ("linear", factor), ("base",
    factor) or ("parts", factor, original, low, high), as fv_rope_frequencies. axes: pairs of each position axis, first axis first (a
    video's frame, row and column; each a rotation of its own base^(-i / n)); None: one axis. amplitude: a factor on what is turned."""

    __slots__ = ("_d", "_rot", "_halves", "_axes", "_amplitude", "_turns", "_freq", "_pair_axis", "_device")
    d, rot, halves, axes, amplitude = (property(attrgetter(n)) for n in __slots__[:5])

    def __init__(self, d, base=10000.0, rot=None, halves=False, scaling=None, axes=None, amplitude=1.0, device=None):
        rot = d if rot is None else rot
        axes = (rot // 2,) if axes is None else tuple(axes)
        if rot % 2 or sum(axes) != rot // 2 or min(axes) < 1:
            raise ValueError(f"Rope: the pairs of the axes {axes} are not the {rot // 2} of {rot} channels")
        if rot > d or rot % 16 or d % 8 or len(axes) > 4:
            raise ValueError("Rope: want rot a multiple of 16 within d, d of 8, and four axes at most")
        kind, factor, original, low, high = 0, 1.0, 1.0, 0.0, 1.0
        if scaling is not None:
            if scaling[0] not in _SCALINGS or len(scaling) != (5 if scaling[0] == "parts" else 2):
                raise ValueError(f"Rope: scaling {scaling}: want (\"linear\" or \"base\", factor) or (\"parts\", factor, original, low, high)")
            kind, factor = _SCALINGS[scaling[0]], scaling[1]
            if kind == 3:
                original, low, high = scaling[2:]
        turns = []
        for n in axes:
            out = (C.c_uint64 * n)()
            _lib.check(_lib.lib().fv_rope_frequencies(n, base, kind, factor, original, low, high, out))
            turns += list(out)
        self._d, self._rot, self._halves, self._axes, self._amplitude, self._turns = d, rot, bool(halves), axes, float(amplitude), tuple(turns)
        device = torch.device("cuda" if device is None else device)
        self._freq = torch.tensor(turns, dtype=_I64, device=device)   # (below 2^62)
        self._pair_axis = torch.tensor([a for a, n in enumerate(axes) for _ in range(n)], dtype=_I32, device=device) if len(axes) > 1 else None
        self._device = self._freq.get_device()

    @property
    def turns(self):
        """Turns a position of each pair, in units of 2^-64."""
        return self._turns


def rope_tokens(rope, positions, q, k=None, inverse=False, out_bf16=None, in_place=False):
    """q [tokens, heads, d] (and k [tokens, kv_heads, d]), f32 or bf16, turned by the angles of positions, int32 [tokens] or [tokens, axes].
    inverse: turned back, which is the gradients' way. Returns contiguous tensors of the inputs' type (out_bf16: another one), or with
    in_place the inputs themselves; with k both."""
    if _watched(q, k):
        if in_place:
            raise ValueError("rope_tokens: autograd watches q or k and would not see them turned in place")
        return _NoGraph.apply("rope_tokens", lambda: rope_tokens(rope, positions, q, k, inverse, out_bf16), q, *(() if k is None else (k,)))
    dev, d = rope._device, rope._d
    _on(dev, "rope_tokens")
    dtypes = (q.dtype,) if q.dtype is _BF16 or q.dtype is _F32 else (_F32, _BF16)
    heads, qs = _tokens(q, "q", 0, d, dev, dtypes)
    tokens, kvh, ks = q.shape[0], 0, 0
    if k is not None:
        kvh, ks = _tokens(k, "k", 0, d, dev, dtypes)
        if k.shape[0] != tokens:
            raise ValueError("rope_tokens: q and k differ in tokens")
    axes = len(rope._axes)
    want = (tokens,) if positions.dim() == 1 and axes == 1 else (tokens, axes)
    if positions.dtype is not _I32 or positions.shape != want or not positions.is_contiguous() or positions.get_device() != dev:
        raise ValueError(f"rope_tokens: positions must be contiguous int32 {list(want)} on the frequencies' device")
    is16 = q.dtype is _BF16
    out16 = is16 if out_bf16 is None else bool(out_bf16)
    if in_place:
        if out16 != is16:
            raise ValueError("rope_tokens: in place keeps the type")
        q_out, k_out, qos, kos = q, k, qs, ks
    else:
        dtype = _BF16 if out16 else _F32
        q_out, qos = _like(q, dtype), heads * d
        k_out, kos = (_like(k, dtype), kvh * d) if k is not None else (None, 0)
    _lib.check(_lib.lib().fv_rope_tokens(
        q.data_ptr(), qs, q_out.data_ptr(), qos, heads, k.data_ptr() if k is not None else None, ks, k_out.data_ptr() if k is not None else None, kos, kvh, d,
        1 if is16 else 0, 1 if out16 else 0, rope._freq.data_ptr(), rope._pair_axis.data_ptr() if rope._pair_axis is not None else None, rope._rot // 2,
        positions.data_ptr(), axes, tokens, rope._amplitude, 1 if rope._halves else 0, 1 if inverse else 0, _lib.stream()))
    if in_place:   # (written by their addresses: tensors saved for a gradient are known to be others now)
        increment_version(q if k is None else (q, k))
    return q_out if k is None else (q_out, k_out)


class PackedSeqs:
    """The sequences of a call: int32 CUDA tensors q_start [n + 1] and k_start [n + 1] (None: q_start), the first row and key of each and the end
    of the last; max_q and max_k (None: max_q) bound the rows and keys of a sequence (host numbers: the launches are sized by
    them; of a longer sequence the first rows and keys, at the positions that they have in the whole, are taken).
    The tensors' addresses are taken here: other numbers go into them, other tensors are another PackedSeqs."""

    __slots__ = ("_q_start", "_k_start", "max_q", "max_k", "_args", "_device")
    q_start, k_start = (property(attrgetter(n)) for n in __slots__[:2])

    def __init__(self, q_start, max_q, k_start=None, max_k=None):
        dev = q_start.get_device()
        k_start = q_start if k_start is None else k_start
        for t in (q_start, k_start):
            if t.dtype is not _I32 or t.dim() != 1 or not t.is_contiguous() or t.get_device() != dev or dev < 0 or t.shape[0] < 1:
                raise ValueError("PackedSeqs: want contiguous int32 CUDA tensors [n + 1] on one device")
        if q_start.shape != k_start.shape:
            raise ValueError("PackedSeqs: starts of different numbers of sequences")
        max_k = max_q if max_k is None else max_k
        if max_q < 0 or max_k < 0:
            raise ValueError("PackedSeqs: bounds must not be negative")
        self._q_start, self._k_start, self.max_q, self.max_k, self._device = q_start, k_start, max_q, max_k, dev
        self._args = (q_start.data_ptr(), k_start.data_ptr(), q_start.shape[0] - 1)

    def __reduce__(self):   # (copies take the addresses of their own tensors)
        return PackedSeqs, (self._q_start, self.max_q, self._k_start, self.max_k)


def _operands(name, q, k, v, seqs, mask, causal):
    """(device, d, heads, kv_heads, strides of q, k, v, mask numbers) of a call, checked."""
    dev = seqs._device
    _on(dev, name)
    if q.dim() != 3:
        raise ValueError(f"{name}: want q [tokens, heads, d]")
    d = q.shape[2]
    heads, qs = _tokens(q, "q", 0, d, dev)
    kvh, ks = _tokens(k, "k", 0, d, dev)
    vs = _tokens(v, "v", kvh, d, dev)[1]
    if v.shape[0] != k.shape[0]:
        raise ValueError(f"{name}: k and v differ in tokens")
    if not causal and mask is not None:
        raise ValueError(f"{name}: a mask is causal")
    return dev, d, heads, kvh, qs, ks, vs, (mask.block_tokens, mask.window, mask.sink) if mask is not None else (1, 0, 0)


def _dense(t, name, shape, dtypes, device):
    if t.dtype not in dtypes or t.shape != shape or not t.is_contiguous() or t.get_device() != device:
        raise ValueError(f"{name} must be a contiguous tensor {list(shape)} of {' or '.join(str(x) for x in dtypes)} on cuda:{device}")


def packed_attention(q, k, v, seqs, mask=None, causal=True, scale=None, out_bf16=True, out=None, with_lse=False):
    """softmax(scale q k^T) v inside each sequence: q [tokens, heads, d], k, v [keys, kv_heads, d] (bf16; tokens may lie apart, as slices of a
    projection do) -> [tokens, heads, d]. causal: by token, the last row at the last key, or by a BlockCausal `mask` whose sink blocks are not
    seen before their time; not causal: every key of the sequence. with_lse: also f32 [tokens, heads], the logarithm of every row's
    sum, for packed_attention_backward. Rows behind the last sequence are not written."""
    if _watched(q, k, v):
        return _NoGraph.apply("packed_attention", lambda: packed_attention(q, k, v, seqs, mask, causal, scale, out_bf16, out, with_lse), q, k, v)
    dev, d, heads, kvh, qs, ks, vs, m = _operands("packed_attention", q, k, v, seqs, mask, causal)
    tokens, keys = q.shape[0], k.shape[0]
    dtype = _BF16 if out_bf16 else _F32
    given = out is not None
    if not given:
        out = _like(q, dtype)
    else:
        _dense(out, "out", (tokens, heads, d), (dtype,), dev)
    lse = torch.empty((tokens, heads), device=q.device, dtype=_F32) if with_lse else None
    lib, n = _lib.lib(), seqs._args[2]
    numbers = (heads, kvh, d, n, tokens, keys, seqs.max_q, seqs.max_k, 1 if causal else 0, *m)
    nbytes = lib.fv_packed_attention_workspace_bytes(*numbers)
    work = torch.empty(nbytes, device=q.device, dtype=_U8) if nbytes else None
    _lib.check(lib.fv_packed_attention(
        q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, out.data_ptr(), 1 if out_bf16 else 0, lse.data_ptr() if with_lse else None, heads, kvh, d,
        *seqs._args, tokens, keys, seqs.max_q, seqs.max_k, 1.0 / math.sqrt(d or 1) if scale is None else scale, 1 if causal else 0, *m,
        work.data_ptr() if nbytes else None, nbytes, _lib.stream()))
    if given:
        increment_version(out)
    return (out, lse) if with_lse else out


def packed_attention_backward(dout, q, k, v, out, lse, seqs, mask=None, causal=True, scale=None, grads_bf16=True):
    """The gradients (dq, dk, dv), contiguous, of a scalar from its gradient dout [tokens, heads, d] (f32 or bf16) by packed_attention's result:
    q, k, v, seqs, mask, causal and scale as that call had them, out and lse as it returned them. An f32 dout is rounded to bf16 first. By an f32
    out rows that see few keys are nearer (in calls whose rows see 64 keys at most they are so by either). Rows and keys behind the last
    sequence are not written."""
    if _watched(dout):   # (gradients of gradients)
        return _NoGraph.apply("packed_attention_backward", lambda: packed_attention_backward(dout, q, k, v, out, lse, seqs, mask, causal, scale, grads_bf16), dout)
    dev, d, heads, kvh, qs, ks, vs, m = _operands("packed_attention_backward", q, k, v, seqs, mask, causal)
    tokens, keys = q.shape[0], k.shape[0]
    _dense(dout, "dout", (tokens, heads, d), (_BF16, _F32), dev)
    _dense(out, "out", (tokens, heads, d), (_BF16, _F32), dev)
    _dense(lse, "lse", (tokens, heads), (_F32,), dev)
    dtype = _BF16 if grads_bf16 else _F32
    dq, dk, dv = _like(q, dtype), _like(k, dtype), _like(v, dtype)
    lib, n, g16 = _lib.lib(), seqs._args[2], 1 if dout.dtype is _BF16 else 0
    numbers = (heads, kvh, d, n, tokens, keys, seqs.max_q, seqs.max_k, 1 if causal else 0, *m)
    nbytes = lib.fv_packed_attention_backward_workspace_bytes(g16, *numbers)
    work = torch.empty(nbytes, device=q.device, dtype=_U8) if nbytes else None
    _lib.check(lib.fv_packed_attention_backward(
        dout.data_ptr(), g16, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, out.data_ptr(), 1 if out.dtype is _BF16 else 0, lse.data_ptr(),
        dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), 1 if grads_bf16 else 0, heads, kvh, d, *seqs._args, tokens, keys, seqs.max_q, seqs.max_k,
        1.0 / math.sqrt(d or 1) if scale is None else scale, 1 if causal else 0, *m, work.data_ptr() if nbytes else None, nbytes, _lib.stream()))
    return dq, dk, dv
