"""The operators of a paged KV cache, as data: what to prepare, one pass through each, its plain form in elementary torch
operations, the same from the definitions in 64 bits, and the bytes and operations a pass cannot do without.

append: the keys (rotated by their positions), the values and, where they are given, the queries (rotated) of new tokens,
ragged over the sequences, into pages of bf16 or of 4 bits (e2m1 codes with a power-of-two scale for 32 channels).
attend: the new tokens' queries against the cache: causal by blocks, a sliding window with the first blocks kept in
sight, query heads that share key heads. step: both, as a serving loop calls them.

The shapes: latent frames of 1560 tokens (480p), 12 or 40 heads of 128 and 24 of 64, as the attention calls beside this file
have them, clips of up to 21 frames (32760 tokens); text-like sequences of generic lengths with shared key heads.
"""
import math
import os
import sys

import numpy as np
import torch

DEVICE = "cuda:0"
own = False

BF16, F32 = "bf16", "f32"


def _case(name, kind, **kw):
    base = {"name": name, "kind": kind, "bits": 16, "seqs": 1, "heads": 12, "kv_heads": 12, "d": 128, "page": 64, "q": 1, "len": 1,
            "ragged": False, "block": 1, "window": 0, "sink": 0, "dtype": BF16, "halves": False, "with_q": False}
    return {**base, **kw}


def listed():
    return [
        # one token each of 32 sessions, queries rotated with the keys: latency
        _case("append_tokens", "append", seqs=32, len=1500, ragged=True, with_q=True),
        # prompts of very different lengths, keys shared by groups, the rotation of halves
        _case("append_prompts", "append", seqs=24, heads=32, kv_heads=8, q=4000, len=4000, ragged=True, halves=True, with_q=True),
        # three latent frames of two clips at the end of the window, f32 activations, into 4 bits
        _case("append_frames_4bit", "append", bits=4, seqs=2, q=4680, len=32760, dtype=F32),
        # a few short sessions, one token each: latency of the attention alone
        _case("tokens_few", "attend", seqs=4, heads=24, kv_heads=24, d=64, len=777, ragged=True),
        # many sessions with shared key heads: the cache's bandwidth
        _case("tokens_many", "attend", seqs=64, heads=40, kv_heads=8, len=8192, ragged=True),
        # five drafted tokens a session, pages of 16, a window with four sinks
        _case("drafts_window", "attend", seqs=48, heads=32, kv_heads=8, page=16, q=5, len=6000, ragged=True, window=2048, sink=4),
        # one latent frame against a clip of 21 frames: every query sees its whole frame and what came before
        _case("frame_480p", "attend", q=1560, len=32760, block=1560),
        # prompts under a window with sinks
        _case("prompts_window", "attend", seqs=3, heads=32, kv_heads=8, q=6001, len=6001, ragged=True, window=1024, sink=4),
        # one long session at a time over 4 bits: few rows, a long axis
        _case("token_long_4bit", "attend", bits=4, heads=40, kv_heads=8, len=131000),
        # the largest caches: 4 bits, long sessions, shared key heads
        _case("tokens_many_4bit", "attend", bits=4, seqs=40, heads=40, kv_heads=8, len=32760, ragged=True),
        # three frames of two clips over 4 bits
        _case("frames_4bit", "attend", bits=4, seqs=2, q=4680, len=32760, block=4680),
        # a serving step of 128 sessions: append to 4-bit pages, attend under a window with sinks
        _case("step_4bit", "step", bits=4, seqs=128, heads=32, kv_heads=8, len=9000, ragged=True, window=4096, sink=16, halves=True, with_q=True),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "step"])
    heads, kv_heads, d = rng.choice([(12, 12, 128), (40, 40, 128), (24, 24, 64), (32, 8, 128), (40, 8, 128), (32, 4, 64), (16, 1, 128)])
    c = {"kind": kind, "bits": rng.choice([16, 4]), "heads": heads, "kv_heads": kv_heads, "d": d, "page": rng.choice([16, 32, 64, 128]),
         "ragged": rng.random() < 0.7, "block": 1, "window": 0, "sink": 0, "dtype": rng.choice([BF16, BF16, F32]),
         "halves": rng.random() < 0.5, "with_q": kind == "step" or rng.random() < 0.5}
    form = rng.choice(["tokens", "drafts", "prompts", "frames"])
    if form in ("tokens", "drafts"):
        c["q"] = 1 if form == "tokens" else rng.randint(2, 9)
        c["len"] = _between(rng, 64, 30000)
        c["seqs"] = _between(rng, 1, max(1, min(128, 4_000_000 // (c["len"] * kv_heads))))
    elif form == "prompts":
        c["q"] = c["len"] = _between(rng, 100, 5000)
        c["seqs"] = _between(rng, 1, max(1, min(12, 12000 // c["len"])))
    else:
        frame, per_block = rng.choice([390, 880, 1560]), rng.choice([1, 3])
        c["block"] = c["q"] = frame * per_block
        c["len"] = c["q"] * rng.randint(1, max(1, min(7, 16000 // c["q"])))
        c["seqs"], c["ragged"] = rng.choice([1, 1, 2]), False
    if form != "frames" and rng.random() < 0.5:
        c["window"], c["sink"] = _between(rng, 16, 4096), rng.choice([0, 1, 4, 64])
    elif form == "frames" and rng.random() < 0.3:
        c["window"], c["sink"] = rng.randint(1, 4), rng.choice([0, 1])
    return c


# ---- the batch of a case: fixed by the case alone --------------------------------------------------------------------

def _counts(case):
    """(tokens in the cache, new tokens) of every sequence."""
    out = []
    for s in range(case["seqs"]):
        part = 1.0 - 0.85 * ((s * 0.6180339887498949) % 1.0) if case["ragged"] else 1.0
        n = max(1, int(round(case["len"] * part)))
        if case["q"] == case["len"]:
            q = n
        elif case["block"] == case["q"]:
            q = min(n, case["q"])
        else:
            q = min(n, max(1, case["q"] - (s % 3 if case["ragged"] else 0)))
        out.append((n, q))
    return out


def _seen(case, p):
    """The keys a query at position p sees: [0, a) and [lo, hi), a <= lo."""
    b = case["block"]
    hi = (p // b + 1) * b
    lo = max(0, p // b - case["window"] + 1) * b if case["window"] else 0
    return min(case["sink"] * b, lo), lo, hi


def work(case):
    size, kvh, h, d = (2 if case["dtype"] == BF16 else 4), case["kv_heads"], case["heads"], case["d"]
    row = 2 * d if case["bits"] == 16 else d // 2 + d // 32
    counts = _counts(case)
    new = sum(q for _, q in counts)
    nbytes = flops = 0
    if case["kind"] in ("append", "step"):
        nbytes += new * (2 * kvh * (d * size + row) + 4 * d)
        if case["with_q"]:
            nbytes += new * h * d * (size + 2)
        if case["bits"] == 4:
            nbytes += new * 2 * kvh * (row + 2 * d)   # what was stored, read back
    if case["kind"] in ("attend", "step"):
        for n, q in counts:
            a, lo, _ = _seen(case, n - q)
            nbytes += (a + n - lo) * 2 * kvh * row
            p = np.arange(n - q, n)
            b = case["block"]
            his = np.minimum((p // b + 1) * b, n)
            los = np.maximum(0, p // b - case["window"] + 1) * b if case["window"] else np.zeros_like(p)
            flops += 4 * d * h * int((his - los + np.minimum(case["sink"] * b, los)).sum())
        nbytes += new * h * d * 4
    return {"bytes": nbytes, "flops": flops}


# ---- 4 bits ----------------------------------------------------------------------------------------------------------

_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _to_4bit(x):
    """x [.., d] f32 -> codes [.., d/2] (channel 2i in the low half of byte i) and scales [.., d/32] (2^(s - 127), the smallest
    power of two that takes no value past the largest code), nearest code, ties to the even one."""
    b = x.unflatten(-1, (-1, 32))
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True))          # a = m 2^e, m in [0.5, 1)
    e = torch.where(m > 0.75, e - 2, e - 3).clamp(-126, 126)    # a <= 6 2^e
    a = torch.ldexp(b, -e)
    mag = a.abs()
    code = (mag > 0.25).to(torch.uint8)
    code += mag >= 0.75
    code += mag > 1.25
    code += mag >= 1.75
    code += mag > 2.5
    code += mag >= 3.5
    code += mag > 5.0
    code += (a < 0).to(torch.uint8) * 8
    code = code.flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).squeeze(-1).to(torch.uint8)


def _from_4bit(codes, scales):
    levels = torch.tensor(_LEVELS + tuple(-x for x in _LEVELS), device=codes.device)
    x = torch.stack((levels[(codes & 15).long()], levels[(codes >> 4).long()]), -1).flatten(-2)
    return (x.unflatten(-1, (-1, 32)) * torch.exp2(scales.float() - 127.0).unsqueeze(-1)).flatten(-2)


# ---- inputs ----------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kvh, h, d, page = case["kv_heads"], case["heads"], case["d"], case["page"]
    counts = _counts(case)
    need = [-(-n // page) for n, _ in counts]
    width, pages = max(need), sum(need) + 3      # a few pages are somebody else's
    order = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    i32 = {"dtype": torch.int32, "device": DEVICE}
    starts = np.concatenate([[0], np.cumsum([q for _, q in counts])])
    state = {"case": case, "table": table, "lens": torch.tensor([n for n, _ in counts], **i32),
             "q_start": torch.tensor(starts.tolist(), **i32), "max_q": max(q for _, q in counts), "max_len": max(n for n, _ in counts)}

    def normal(*shape, dtype=torch.bfloat16):
        x = torch.empty(shape, device=DEVICE, dtype=dtype)
        for part in x.split(max(1, (1 << 28) // max(1, x[0].numel()))):
            part.copy_(torch.randn(part.shape, generator=gen, device=DEVICE))
        return x

    shape = (pages, kvh, page, d)
    if case["bits"] == 16:
        state["k_pages"], state["v_pages"] = normal(*shape), normal(*shape)
        state["k_scales"] = state["v_scales"] = None
    else:
        for n in ("k", "v"):
            state[n + "_pages"] = torch.empty(*shape[:3], d // 2, device=DEVICE, dtype=torch.uint8)
            state[n + "_scales"] = torch.empty(*shape[:3], d // 32, device=DEVICE, dtype=torch.uint8)
            step = max(1, (1 << 26) // (kvh * page * d))
            for i in range(0, pages, step):
                codes, scales = _to_4bit(torch.randn((min(step, pages - i), *shape[1:]), generator=gen, device=DEVICE))
                state[n + "_pages"][i:i + step], state[n + "_scales"][i:i + step] = codes, scales
    new = int(starts[-1])
    dtype = torch.bfloat16 if case["dtype"] == BF16 else torch.float32
    if case["kind"] in ("append", "step"):
        state["k"], state["v"] = normal(new, kvh, d, dtype=dtype), normal(new, kvh, d, dtype=dtype)
        # rotation angles position / 10000^(2i/d), made in 64 bits; one per pair, for each of its channels
        pos = torch.arange(state["max_len"], device=DEVICE, dtype=torch.float64)[:, None]
        angle = pos * 10000.0 ** (-torch.arange(0, d, 2, device=DEVICE, dtype=torch.float64) / d)[None, :]
        spread = (lambda t: torch.cat((t, t), 1)) if case["halves"] else (lambda t: t.repeat_interleave(2, dim=1))
        state["rope"] = tuple(spread(f(angle)).float().contiguous() for f in (torch.cos, torch.sin))
    if case["kind"] != "append" or case["with_q"]:
        state["q"] = normal(new, h, d, dtype=dtype if case["kind"] != "attend" else torch.bfloat16)
    return state


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    if "fastvideo-rs_amd" not in sys.path[0]:
        sys.path.insert(0, os.path.abspath("fastvideo-rs_amd"))   # the working folder is the repository's root
    import fv_sdpa

    case = state["case"]
    pool = fv_sdpa.PagedKv(state["k_pages"], state["v_pages"], state["k_scales"], state["v_scales"])
    batch = fv_sdpa.PagedBatch(state["q_start"], state["lens"], state["table"], state["max_q"], state["max_len"])
    out, q = {}, state.get("q")
    if case["kind"] in ("append", "step"):
        q = fv_sdpa.paged_append(pool, batch, state["k"], state["v"], rope=state["rope"], halves=case["halves"], q=q)
        if q is not None:
            out["q"] = q
        if case["bits"] == 16:
            out["k"], out["v"] = pool.k, pool.v
        else:
            out["k"], out["v"] = fv_sdpa.paged_read(pool, batch, state["k"].shape[0])
    if case["kind"] in ("attend", "step"):
        out["out"] = fv_sdpa.paged_attention(q, pool, batch, fv_sdpa.BlockCausal(case["block"], case["window"], case["sink"]))
    return out


def _places(state):
    """For every new token: its sequence, its number among the sequence's new ones, its position, page and slot."""
    start, lens = state["q_start"].long(), state["lens"].long()
    new = start.new_ones(state["q"].shape[0] if "q" in state else state["k"].shape[0]).cumsum(0) - 1
    seq = torch.searchsorted(start, new, right=True) - 1
    i = new - start[seq]
    pos = lens[seq] - (start[seq + 1] - start[seq]) + i
    page = state["case"]["page"]
    return seq, i, pos, state["table"][seq, pos // page].long(), pos % page


def _rotate_plain(x, rope, pos, halves):
    c, s = rope[0][pos], rope[1][pos]
    half = x.shape[-1] // 2
    if halves:
        c, s = c[:, None, :half], s[:, None, :half]
        a, b = x[..., :half], x[..., half:]
        return torch.cat((a * c - b * s, a * s + b * c), -1)
    c, s = c[:, None, 0::2], s[:, None, 0::2]
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def _rows_plain(state, name, page, slot):
    """f32 [.., kv_heads, d] of the tokens at (page, slot)."""
    x = state[name + "_pages"][page, :, slot]
    return x.float() if state["case"]["bits"] == 16 else _from_4bit(x, state[name + "_scales"][page, :, slot])


def _run_plain(state):
    case = state["case"]
    out, q = {}, state.get("q")
    seq, i, pos, page, slot = _places(state)
    if case["kind"] in ("append", "step"):
        for name, x in (("k", _rotate_plain(state["k"].float(), state["rope"], pos, case["halves"])), ("v", state["v"].float())):
            if case["bits"] == 16:
                state[name + "_pages"][page, :, slot] = x.bfloat16()
                out[name] = state[name + "_pages"]
            else:
                state[name + "_pages"][page, :, slot], state[name + "_scales"][page, :, slot] = _to_4bit(x)
                out[name] = _rows_plain(state, name, page, slot).bfloat16()
        if q is not None:
            q = out["q"] = _rotate_plain(q.float(), state["rope"], pos, case["halves"]).bfloat16()
    if case["kind"] in ("attend", "step"):
        kvh, h, d, b = case["kv_heads"], case["heads"], case["d"], case["block"]
        start, lens = state["q_start"].long(), state["lens"].long()
        seqs, nq, nk = case["seqs"], state["max_q"], state["max_len"]
        # keys and values of every sequence, padded to the longest: [seqs, kv_heads, nk, d]
        j = torch.arange(nk, device=DEVICE)
        at = state["table"].long()[:, j // case["page"]].clamp(min=0), (j % case["page"])[None, :].expand(seqs, nk)
        keys, values = (_rows_plain(state, n, *at).transpose(1, 2).contiguous() for n in ("k", "v"))
        # queries padded likewise, rows of one key head together: [seqs, kv_heads, nq * group, d]
        r = torch.arange(nq, device=DEVICE)
        rows = (start[:-1, None] + r[None, :]).clamp(max=q.shape[0] - 1)
        queries = q.float()[rows].unflatten(2, (kvh, h // kvh)).transpose(1, 2).reshape(seqs, kvh, -1, d)
        scores = torch.matmul(queries, keys.transpose(2, 3)).mul_(1.0 / math.sqrt(d)).unflatten(2, (nq, h // kvh))
        tq = ((lens - (start[1:] - start[:-1]))[:, None] + r[None, :])[:, :, None] // b
        tk = (j // b)[None, None, :]
        seen = (tk <= tq) & (j[None, None, :] < lens[:, None, None])
        if case["window"]:
            seen &= (tq - tk < case["window"]) | (tk < case["sink"])
        scores.masked_fill_(~seen[:, None, :, None, :], -math.inf)
        scores.sub_(scores.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
        total = scores.sum(-1, keepdim=True)
        values.masked_fill_((j[None, :] >= lens[:, None])[:, None, :, None], 0.0)
        o = torch.matmul(scores.flatten(2, 3), values).unflatten(2, (nq, h // kvh)) / total.clamp(min=1e-38)
        out["out"] = o[seq, :, i].reshape(-1, h, d).bfloat16()
    return out


# ---- from the definitions, in 64 bits --------------------------------------------------------------------------------

def _nearest_4bit(x):
    """The value that 4 bits keep of each element of x [.., d], in 64 bits."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = b.abs().max(-1, keepdim=True).values
    scale = torch.exp2(torch.ceil(torch.log2(top.clamp(min=1e-300) / 6.0)).clamp(-126, 126))
    scale = torch.where(top > 6 * scale, 2 * scale, torch.where(top <= 3 * scale, scale / 2, scale)).clamp(min=2.0 ** -126)
    a = (b / scale).abs()
    # the spacing of the codes at a: 1/2 up to 2, 1 up to 4, then 2; rounding to the nearest multiple, ties to even
    gap = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return (torch.round(a / gap) * gap * b.sign() * scale).reshape(x.shape)


def _turn(x, angle_rows, halves):
    """x [tokens, heads, d] turned by the angles whose cosines and sines are given per pair."""
    c, s = (t[:, None, :] for t in angle_rows)
    z = torch.stack((x[..., :x.shape[-1] // 2], x[..., x.shape[-1] // 2:]), -1) if halves else x.reshape(*x.shape[:-1], -1, 2)
    turned = torch.view_as_real(torch.view_as_complex(z.contiguous()) * torch.complex(c, s))
    return torch.cat((turned[..., 0], turned[..., 1]), -1) if halves else turned.reshape(x.shape)


def exact(case, seed):
    state = prepare(case, seed)
    counts, page, d = _counts(case), case["page"], case["d"]
    h, kvh = case["heads"], case["kv_heads"]
    cached = {}
    levels = torch.tensor(_LEVELS, dtype=torch.float64, device=DEVICE)

    def stored(name, ids):
        x = state[name + "_pages"][ids]                                        # [n, kv_heads, page, ..]
        if case["bits"] == 16:
            return x.double()
        low, high = x.bitwise_and(15), x.bitwise_right_shift(4)
        v = torch.stack((low, high), -1).flatten(-2).long()
        v = levels[v % 8] * (1 - 2 * (v // 8)).double()
        return v * torch.exp2(state[name + "_scales"][ids].double() - 127).repeat_interleave(32, -1)

    first = np.concatenate([[0], np.cumsum([q for _, q in counts])])
    new = {"k": [], "v": [], "q": []}
    if case["kind"] in ("append", "step"):
        pools = {n: state[n + "_pages"].double() for n in ("k", "v")} if case["bits"] == 16 else None
        for s, (n, q) in enumerate(counts):
            part = slice(int(first[s]), int(first[s + 1]))
            pos = torch.arange(n - q, n, device=DEVICE)
            each = slice(0, d // 2) if case["halves"] else slice(0, d, 2)
            rows = [t[n - q:n, each].double() for t in state["rope"]]
            ids = state["table"][s].long()[pos // page]
            for name in ("k", "v"):
                x = state[name][part].double()
                x = _turn(x, rows, case["halves"]) if name == "k" else x
                if case["bits"] == 4:
                    x = _nearest_4bit(x)
                else:
                    pools[name].index_put_((ids[:, None], torch.arange(kvh, device=DEVICE)[None, :], (pos % page)[:, None]), x)
                new[name].append(x)
            if "q" in state:
                new["q"].append(_turn(state["q"][part].double(), rows, case["halves"]))
        cached = {"k": pools["k"], "v": pools["v"]} if pools else {n: torch.cat(new[n]) for n in ("k", "v")}
        if "q" in state:
            cached["q"] = torch.cat(new["q"])
    if case["kind"] == "append":
        return cached
    total = torch.empty(int(first[-1]), h, d, dtype=torch.float64, device=DEVICE)
    for s, (n, q) in enumerate(counts):
        ids = state["table"][s, :-(-n // page)].long()
        if case["kind"] == "step":
            queries = new["q"][s].bfloat16().double()
        else:
            queries = state["q"][int(first[s]):int(first[s + 1])].double()
        keys, values = (stored(name, ids).transpose(0, 1).reshape(kvh, -1, d)[:, :n].clone() for name in ("k", "v"))
        if case["kind"] == "step":
            for x, name in ((keys, "k"), (values, "v")):
                fresh = new[name][s] if case["bits"] == 4 else new[name][s].bfloat16().double()
                x[:, n - q:] = fresh.transpose(0, 1)
        for t0 in range(0, q, 1024):      # queries by the thousand, head by head
            t1 = min(q, t0 + 1024)
            tq = torch.arange(n - q + t0, n - q + t1, device=DEVICE).div(case["block"], rounding_mode="floor")[:, None]
            tk = torch.arange(n, device=DEVICE).div(case["block"], rounding_mode="floor")[None, :]
            hidden = tk > tq
            if case["window"]:
                hidden |= (tk <= tq - case["window"]) & (tk >= case["sink"])
            for x in range(h):
                p = queries[t0:t1, x] @ keys[x * kvh // h].t() * d ** -0.5
                p = torch.softmax(p.masked_fill(hidden, -math.inf), -1)
                total[int(first[s]) + t0:int(first[s]) + t1, x] = p @ values[x * kvh // h]
    return {**cached, "out": total}
