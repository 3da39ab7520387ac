"""A paged KV cache and the attention over it (include/fv_sdpa_hip.h, `fv_paged_*`; no counterpart in the reference): many
sequences of different lengths in one pool of pages of bf16 or of 4 bits, new tokens appended with the rotation of their
positions applied on the way, attention under the block mask with a window and sinks, single tokens to long prompts.
"""
import math
from operator import attrgetter

import torch

from . import _lib

__all__ = ["PagedKv", "PagedBatch", "paged_append", "paged_read", "paged_attention"]

_BF16, _F32, _U8, _I32 = torch.bfloat16, torch.float32, torch.uint8, torch.int32
_ONLY_BF16 = (_BF16,)


class PagedKv:
    """One layer's pool: k, v [pages, kv_heads, page_tokens, d] bf16, or 4-bit codes [.., d / 2] with k_scales, v_scales
    [.., d / 32] (uint8 all four). The tensors are the caller's, used in place; their addresses are taken here, so that the
    fields cannot be set (other tensors are another PagedKv)."""

    __slots__ = ("_k", "_v", "_k_scales", "_v_scales", "_d", "_kv_heads", "_args", "_device")
    k, v, k_scales, v_scales, d, kv_heads = (property(attrgetter(n)) for n in __slots__[:6])

    def __init__(self, k, v, k_scales=None, v_scales=None):
        four = k_scales is not None
        shape = k.shape
        if (v_scales is None) == four or len(shape) != 4 or v.shape != shape:
            raise ValueError("PagedKv: want k and v [pages, kv_heads, page_tokens, d] of one shape, with scales for both or neither")
        dtype, dev = (_U8 if four else _BF16), k.get_device()
        if k.dtype is not dtype or v.dtype is not dtype or not k.is_contiguous() or not v.is_contiguous() or dev < 0 or v.get_device() != dev:
            raise ValueError(f"PagedKv: want contiguous CUDA tensors of {dtype} on one device")
        d = shape[3] * 2 if four else shape[3]
        if four:
            want = (shape[0], shape[1], shape[2], d // 32)
            for t in (k_scales, v_scales):
                if t.dtype is not _U8 or t.shape != want or not t.is_contiguous() or t.get_device() != dev:
                    raise ValueError(f"PagedKv: want contiguous uint8 scales {want} on the pages' device")
        self._k, self._v, self._k_scales, self._v_scales, self._d, self._kv_heads, self._device = k, v, k_scales, v_scales, d, shape[1], dev
        self._args = (k.data_ptr(), v.data_ptr(), k_scales.data_ptr() if four else None, v_scales.data_ptr() if four else None,
                      shape[0], shape[2], shape[1], d)

    def __reduce__(self):   # (copies take the addresses of their own tensors)
        return PagedKv, (self._k, self._v, self._k_scales, self._v_scales)

    @staticmethod
    def new(pages, page_tokens, kv_heads, d, four_bits=False, device="cuda"):
        """A pool of zeros."""
        shape = (pages, kv_heads, page_tokens)
        if not four_bits:
            return PagedKv(*(torch.zeros((*shape, d), dtype=_BF16, device=device) for _ in range(2)))
        return PagedKv(*(torch.zeros((*shape, n), dtype=_U8, device=device) for n in (d // 2, d // 2, d // 32, d // 32)))

    @property
    def four_bits(self):
        return self._k_scales is not None

    @property
    def page_tokens(self):
        return self._k.shape[2]


class PagedBatch:
    """The sequences of a call: int32 CUDA tensors q_start [n + 1] (rows of sequence s: q_start[s] .. q_start[s + 1]), lens [n]
    (tokens in the cache, the new ones among them) and table [n, columns] (page numbers); max_q and max_len bound the rows of
    a sequence and its length (host numbers: the launches are sized by them; max_len None: what the table's columns hold). The
    tensors' addresses are taken here: other numbers go into them, other tensors are another PagedBatch."""

    __slots__ = ("_q_start", "_lens", "_table", "max_q", "max_len", "_args", "_device")
    q_start, lens, table = (property(attrgetter(n)) for n in __slots__[:3])

    def __init__(self, q_start, lens, table, max_q, max_len=None):
        dev = lens.get_device()
        if not (q_start.dtype is lens.dtype is table.dtype is _I32) or dev < 0 or q_start.get_device() != dev or table.get_device() != dev:
            raise ValueError("PagedBatch: want int32 CUDA tensors on one device")
        if lens.dim() != 1 or q_start.dim() != 1 or table.dim() != 2:
            raise ValueError("PagedBatch: want q_start [n + 1], lens [n] and table [n, columns]")
        n, (rows, columns), (step, inner) = lens.shape[0], table.shape, table.stride()
        if q_start.shape[0] != n + 1 or rows != n:
            raise ValueError("PagedBatch: want q_start [n + 1], lens [n] and table [n, columns]")
        if not q_start.is_contiguous() or not lens.is_contiguous() or (columns > 1 and inner != 1) or (n > 1 and step < columns):
            raise ValueError("PagedBatch: want contiguous arrays (of the table: rows)")
        if max_q < 0 or (max_len is not None and max_len < 0):
            raise ValueError("PagedBatch: bounds must not be negative")
        self._q_start, self._lens, self._table, self.max_q, self.max_len, self._device = q_start, lens, table, max_q, max_len, dev
        self._args = (q_start.data_ptr(), lens.data_ptr(), table.data_ptr(), step if n > 1 else columns, columns, n)

    def __reduce__(self):
        return PagedBatch, (self._q_start, self._lens, self._table, self.max_q, self.max_len)


def _rows(t, name, heads, d, dtypes, device):
    """(heads, elements between the tokens) of t [tokens, heads, d], whose heads are contiguous."""
    shape = t.shape
    if len(shape) != 3 or t.dtype not in dtypes or t.get_device() != device:
        raise ValueError(f"{name}: want a [tokens, heads, d] tensor of {' or '.join(str(x) for x in dtypes)} on the pool's device")
    n, h, dd = shape
    if (heads and h != heads) or dd != d:
        raise ValueError(f"{name}: want [tokens, {heads or 'heads'}, {d}], got {tuple(shape)}")
    if t.is_contiguous():
        return h, h * d
    a, b, c = t.stride()
    if c != 1 or (h > 1 and b != d):
        raise ValueError(f"{name}: the heads of a token must be contiguous")
    return h, a if n > 1 else h * d


def _on(device, name):
    if torch._C._cuda_getDevice() != device:
        raise ValueError(f"{name}: the tensors are on cuda:{device}, which is not the current device")


def paged_append(pool, batch, k, v, rope=None, halves=False, rope_at=None, q=None):
    """The new tokens' k, v [tokens, kv_heads, d] (f32 or bf16) into the pool, the keys turned by their positions (rows of
    rope = (cos, sin), f32 [rows, d]; rope_at: int32 [tokens], rows in place of the positions). q [tokens, heads, d]: turned
    likewise and returned, bf16. halves: pairs (i, i + d / 2) instead of (2i, 2i + 1). A token past the table's columns is not
    stored; positions are counted from lens, whatever max_len says."""
    dev, kvh, d = pool._device, pool._kv_heads, pool._d
    _on(dev, "paged_append")
    tokens, dtype = k.shape[0], k.dtype
    dtypes = (dtype,) if dtype is _BF16 or dtype is _F32 else (_F32, _BF16)
    ks, vs = _rows(k, "k", kvh, d, dtypes, dev)[1], _rows(v, "v", kvh, d, dtypes, dev)[1]
    if v.shape[0] != tokens or batch._device != dev:
        raise ValueError("paged_append: k and v differ in tokens, or the batch is on another device")
    qs, heads, q_out = 0, 0, None
    if q is not None:
        heads, qs = _rows(q, "q", 0, d, dtypes, dev)
        if q.shape[0] != tokens:
            raise ValueError("paged_append: q and k differ in tokens")
        q_out = torch.empty_like(q) if dtype is _BF16 and q.is_contiguous() else torch.empty((tokens, heads, d), device=q.device, dtype=_BF16)
    cos = sin = None
    rows = 0
    if rope is not None:
        cos, sin = rope
        rows = cos.shape[0]
        if rows == 0 and tokens:   # (no address: the entry would take them for none, and turn nothing)
            raise ValueError("paged_append: rope tables without rows")
        for t in rope:
            if t.dtype is not _F32 or t.shape != (rows, d) or not t.is_contiguous() or t.get_device() != dev:
                raise ValueError(f"paged_append: rope tables must be contiguous f32 [rows, {d}] on the pool's device")
        if rope_at is not None and (rope_at.dtype is not _I32 or rope_at.shape != (tokens,) or not rope_at.is_contiguous() or rope_at.get_device() != dev):
            raise ValueError("paged_append: rope_at must be contiguous int32 [tokens] on the pool's device")
    elif rope_at is not None:
        raise ValueError("paged_append: rope_at without tables")
    _lib.check(_lib.lib().fv_paged_append(
        k.data_ptr(), ks, v.data_ptr(), vs, q.data_ptr() if q is not None else None, qs, q_out.data_ptr() if q is not None else None,
        1 if dtype is _BF16 else 0, heads, cos.data_ptr() if rows else None, sin.data_ptr() if rows else None, rows,
        rope_at.data_ptr() if rope_at is not None else None, 1 if halves else 0, *pool._args, *batch._args, tokens, _lib.stream()))
    return q_out


def paged_read(pool, batch, tokens, out_bf16=True):
    """(k, v) [tokens, kv_heads, d] of the batch's tokens; rows behind the last sequence are not written."""
    dev = pool._device
    _on(dev, "paged_read")
    if batch._device != dev:
        raise ValueError("paged_read: the batch is on another device")
    k = torch.empty((tokens, pool._kv_heads, pool._d), device=pool._k.device, dtype=_BF16 if out_bf16 else _F32)
    v = torch.empty_like(k)
    _lib.check(_lib.lib().fv_paged_read(k.data_ptr(), v.data_ptr(), 1 if out_bf16 else 0, *pool._args, *batch._args, tokens, _lib.stream()))
    return k, v


def paged_attention(q, pool, batch, mask=None, scale=None, out_bf16=True, out=None):
    """softmax(scale q k^T) v of the rows q [tokens, heads, d] (bf16) over the cached keys of their sequences, [tokens, heads, d].
    mask: a BlockCausal; None: causal by token. A sink block is not seen before its time (BlockCausal.allows has it always
    seen). Rows behind the last sequence are not written."""
    dev, kvh, d = pool._device, pool._kv_heads, pool._d
    _on(dev, "paged_attention")
    heads, qs = _rows(q, "q", 0, d, _ONLY_BF16, dev)
    if batch._device != dev:
        raise ValueError("paged_attention: the batch is on another device")
    tokens = q.shape[0]
    dtype = _BF16 if out_bf16 else _F32
    if out is None:   # (half the time of an empty() by shape)
        out = torch.empty_like(q) if out_bf16 and q.is_contiguous() else torch.empty((tokens, heads, d), device=q.device, dtype=dtype)
    elif out.dtype is not dtype or out.shape != q.shape or not out.is_contiguous() or out.get_device() != dev:
        raise ValueError(f"out must be a contiguous {dtype} tensor of shape {tuple(q.shape)} on {q.device}")
    max_len = batch.max_len if batch.max_len is not None else batch._table.shape[1] * pool._k.shape[2]
    bt, window, sink = (mask.block_tokens, mask.window, mask.sink) if mask is not None else (1, 0, 0)
    n = batch._args[5]
    lib = _lib.lib()
    nbytes = lib.fv_paged_attention_workspace_bytes_for(pool._k_scales is not None, heads, kvh, d, n, tokens, batch.max_q, max_len, bt, window, sink)
    work = torch.empty(nbytes, device=q.device, dtype=_U8) if nbytes else None
    _lib.check(lib.fv_paged_attention(
        q.data_ptr(), qs, out.data_ptr(), 1 if out_bf16 else 0, heads, *pool._args, *batch._args, tokens, batch.max_q, max_len,
        1.0 / math.sqrt(d) if scale is None else scale, bt, window, sink, work.data_ptr() if nbytes else None, nbytes, _lib.stream()))
    return out
