"""The operators between the projections of a gated attention block, as cases that can be timed.

  append   ``kernels.rope_append``: rotates queries and keys, writes keys and values to their slots of a paged cache
  gather   ``kernels.kv_gather``: rows of a paged cache as packed keys and values (a prompt chunk on a cached prefix)
  prompt   ``kernels.attention_prompt``: causal attention with grouped heads over packed sequences
  paged    ``kernels.attention_paged``: one query token of each sequence over its pages

``own`` false: elementary torch operations in 32 bits, rounded once at the end.  ``own`` true: the library's calls.

A case is a dict of plain values:

  op       "append", "gather", "prompt", "paged"
  dtype    type of queries, keys and values ("bf16", "f16")
  bits     16 or 4: what a cached element is held in
  heads, kv_heads, dim (of a head), rotary (channels that turn; "append")
  page     tokens of a page; pages lie in no order
  tokens   rows of the call ("append", "gather")
  count, longest, mix   sequences, the longest one's length, and the seed of the other lengths, which are spread
           over the logarithm of 1 .. longest (mix 0: all as long as the longest)
  fresh    "prompt": new tokens of each sequence (at most its length); 0: the whole prompt

A page of a 16-bit cache is [page, kv_heads, dim].  A 4-bit cache holds codes, [kv_heads, page, dim / 2] bytes a
page, and for each token and group of 64 channels a scale and a minimum in float16, [kv_heads, page, dim / 64, 2] for
keys and [kv_heads, dim / 64, page, 2] for values; an element stands for code * scale + minimum.  A unit of codes is
a 32-bit word: of a key 8 channels, the even ones in the low half; of values 2 channels of 4 tokens, a byte a token,
the even channel low, [page / 4, dim / 2] units a head.  The units of two groups lie two and two by turns.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
GROUP = 64          # channels that share a scale and a minimum
LARGEST = 65504.0   # the largest float16: what a 4-bit cache clamps to


def _kernels():
    import __graft_entry__
    return __graft_entry__.load_package().kernels


def listed():
    return [
        # One token of one sequence: the smallest call of a decode loop.
        {"name": "append 1", "op": "append", "dtype": "bf16", "bits": 16, "heads": 8, "kv_heads": 2, "dim": 256,
         "rotary": 64, "page": 256, "tokens": 1},
        # A batch of prompts into a 4-bit cache.
        {"name": "append 8000 4 bit", "op": "append", "dtype": "f16", "bits": 4, "heads": 16, "kv_heads": 4,
         "dim": 128, "rotary": 128, "page": 64, "tokens": 8000},
        # The cached prefix of one sequence, read back for a prompt chunk.
        {"name": "gather 700 4 bit", "op": "gather", "dtype": "bf16", "bits": 4, "heads": 8, "kv_heads": 2,
         "dim": 256, "page": 256, "tokens": 700},
        # Prefixes of a batch, 16-bit pages.
        {"name": "gather 20000", "op": "gather", "dtype": "bf16", "bits": 16, "heads": 16, "kv_heads": 4, "dim": 128,
         "page": 16, "tokens": 20000},
        # One prompt of 2048 tokens.
        {"name": "prompt 2048", "op": "prompt", "dtype": "bf16", "heads": 8, "kv_heads": 2, "dim": 256, "count": 1,
         "longest": 2048, "mix": 0, "fresh": 0},
        # Prompts of many lengths, one token among them, packed.
        {"name": "prompts ragged f16", "op": "prompt", "dtype": "f16", "heads": 16, "kv_heads": 4, "dim": 128,
         "count": 24, "longest": 3001, "mix": 3, "fresh": 0},
        # A chunk of 512 tokens on a cached prefix.
        {"name": "prompt chunk 512", "op": "prompt", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128,
         "count": 1, "longest": 8700, "mix": 0, "fresh": 512},
        # The largest prompt.
        {"name": "prompt 16384", "op": "prompt", "dtype": "bf16", "heads": 8, "kv_heads": 2, "dim": 256, "count": 1,
         "longest": 16384, "mix": 0, "fresh": 0},
        # Decode of one sequence: latency counts.
        {"name": "paged 1x4000 4 bit", "op": "paged", "dtype": "bf16", "bits": 4, "heads": 8, "kv_heads": 2,
         "dim": 256, "page": 256, "count": 1, "longest": 4000, "mix": 0},
        # A decode batch of sequences of many lengths.
        {"name": "paged 64 ragged 4 bit", "op": "paged", "dtype": "bf16", "bits": 4, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "count": 64, "longest": 16000, "mix": 5},
        # One long context: the work is split over its length.
        {"name": "paged 1x131072 4 bit", "op": "paged", "dtype": "f16", "bits": 4, "heads": 8, "kv_heads": 2,
         "dim": 256, "page": 256, "count": 1, "longest": 131072, "mix": 0},
        # A decode batch on 16-bit pages.
        {"name": "paged 32x4100", "op": "paged", "dtype": "bf16", "bits": 16, "heads": 8, "kv_heads": 2, "dim": 256,
         "page": 256, "count": 32, "longest": 4100, "mix": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "gather", "prompt", "prompt", "paged", "paged", "paged"])
    kv_heads, dim = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128, 256])
    case = {"op": op, "dtype": rng.choice(["bf16", "f16"]), "heads": kv_heads * rng.choice([1, 2, 3, 4, 5, 8]),
            "kv_heads": kv_heads, "dim": dim}
    if op == "prompt":
        while True:
            case |= {"count": _log(rng, 1, 40), "longest": _log(rng, 1, 12000), "mix": rng.randint(0, 1000),
                     "fresh": rng.choice([0, 0, _log(rng, 1, 1024)])}
            longest = min(case["longest"], case["fresh"] or case["longest"])
            # The plain form's scores, and the kernel's work, stay below those of the largest listed case.
            if (case["heads"] * case["count"] * longest * case["longest"] <= 1.2e9
                    and work(case)["flops"] <= 1.0e12):
                return case
    case |= {"bits": rng.choice([4, 4, 16]), "page": 16 * rng.choice([1, 2, 3, 4, 8, 16])}
    if op == "append":
        case["rotary"] = rng.choice([dim, dim // 2, dim // 4])
    if op in ("append", "gather"):
        case["tokens"] = max(1, min(_log(rng, 1, 20000), int(8e6) // (kv_heads * dim)))
        return case
    while True:
        case |= {"count": _log(rng, 1, 128), "longest": _log(rng, 1, 131072), "mix": rng.randint(0, 1000)}
        # All caches fit beside the plain form's copies of them in 32 bits.
        if case["count"] * case["longest"] * kv_heads * dim <= 5e8:
            return case


def _lengths(case):
    """Tokens of each sequence (keys), the longest first."""
    rng, longest = random.Random(case["mix"]), case["longest"]
    if not case["mix"]:
        return [longest] * case["count"]
    return [longest] + [_log(rng, 1, longest) for _ in range(case["count"] - 1)]


def _fresh(case):
    """New tokens of each sequence (queries)."""
    return [min(n, case["fresh"] or n) for n in _lengths(case)]


# ---------------------------------------------------------------------------
# Inputs: activations are standard normal, as behind a norm; keys carry an
# offset by channel, as biased projections give them.
# ---------------------------------------------------------------------------
class _Inputs:
    def __init__(self, seed, dtype):
        self.gen = torch.Generator(device=DEV).manual_seed(int(seed))
        self.rng = random.Random(int(seed))
        self.dtype = dtype

    def normal(self, *shape):
        return torch.randn(shape, generator=self.gen, device=DEV).to(self.dtype)

    def keys(self, *shape):
        offset = torch.randn(shape[-2:], generator=self.gen, device=DEV)
        return (torch.randn(shape, generator=self.gen, device=DEV) + offset).to(self.dtype)

    def order(self, n):
        return torch.randperm(n, generator=self.gen, device=DEV)


def _cos_sin(positions, rotary):
    """[positions, rotary] cosines and sines, the angles in 64 bits (far positions turn many times)."""
    rate = 10000.0 ** (-torch.arange(0, rotary, 2, device=DEV, dtype=torch.float64) / rotary)
    angle = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * rate
    return torch.cat((angle.cos(), angle.sin()), -1).float()


def _new_cache(case, pages):
    """Empty caches of `pages` pages: (k, v) or, in 4 bits, (k, v, k_scales, v_scales)."""
    heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    if case["bits"] == 16:
        return [torch.zeros(pages, page, heads, dim, dtype=DTYPES[case["dtype"]], device=DEV) for _ in range(2)]
    return ([torch.zeros(pages, heads, page, dim // 2, dtype=torch.uint8, device=DEV) for _ in range(2)]
            + [torch.zeros(pages, heads, *shape, 2, dtype=torch.float16, device=DEV)
               for shape in ((page, dim // GROUP), (dim // GROUP, page))])


def _full_cache(inp, case, pages):
    """Caches whose every slot holds a row."""
    cache = _new_cache(case, pages)
    heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    at = 0
    while at < pages:      # in pieces: the rows in 16 and 32 bits are larger than the cache
        n = min(pages - at, max(1, int(1e8) // (page * heads * dim)))
        slots = torch.arange(at * page, (at + n) * page, device=DEV)
        _store(case, cache, slots, inp.keys(n * page, heads, dim), inp.normal(n * page, heads, dim))
        at += n
    return cache


def prepare(case, seed):
    inp = _Inputs(seed, DTYPES[case["dtype"]])
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    state = {"case": case, "scale": dim ** -0.5}
    if case["op"] == "append":
        tokens, page = case["tokens"], case["page"]
        pages = -(-tokens // page) + 1
        # Queries, keys and values are columns of one projection; the last row of a batch may be padding.
        rows = inp.normal(tokens, (heads + 2 * kv_heads) * dim)
        q, k, v = (x.view(tokens, -1, dim) for x in rows.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
        slots = inp.order(pages * page)[:tokens].to(torch.int32) if tokens < 512 else (
            inp.order(pages)[:, None] * page + torch.arange(page, device=DEV)).view(-1)[:tokens].to(torch.int32)
        if tokens > 1:
            slots[-1] = -1
        positions = torch.randint(0, 32768, (tokens,), generator=inp.gen, device=DEV)
        return state | {"q": q, "k": k, "v": v, "positions": positions, "cos_sin": _cos_sin(32768, case["rotary"]),
                        "slots": slots, "cache": _new_cache(case, pages),
                        "every": torch.arange(pages * page, device=DEV, dtype=torch.int32)}
    if case["op"] == "gather":
        tokens, page = case["tokens"], case["page"]
        pages = -(-tokens // page) + 1
        slots = (inp.order(pages)[:, None] * page + torch.arange(page, device=DEV)).view(-1)[:tokens]
        return state | {"slots": slots.to(torch.int32), "cache": _full_cache(inp, case, pages)}
    lengths = _lengths(case)
    if case["op"] == "prompt":
        fresh = _fresh(case)
        cu = [torch.tensor([0] + list(_sums(x)), dtype=torch.int32, device=DEV) for x in (fresh, lengths)]
        kv = inp.normal(sum(lengths), 2 * kv_heads * dim)
        k, v = (x.view(-1, kv_heads, dim) for x in kv.chunk(2, 1))
        return state | {"q": inp.normal(sum(fresh), heads, dim), "k": k, "v": v, "cu_q": cu[0], "cu_k": cu[1]}
    page = case["page"]
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + 1
    order, at = inp.order(pages).to(torch.int32), 0
    tables = torch.full((len(need), max(need)), -1, dtype=torch.int32, device=DEV)
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        at += n
    return state | {"q": inp.normal(len(lengths), heads, dim), "cache": _full_cache(inp, case, pages),
                    "tables": tables, "lens": torch.tensor(lengths, dtype=torch.int32, device=DEV)}


def _sums(values):
    total = 0
    for v in values:
        total += v
        yield total


# ---------------------------------------------------------------------------
# The plain forms.
# ---------------------------------------------------------------------------
def _halves(x, rotary):
    return x[..., :rotary // 2], x[..., rotary // 2:rotary], x[..., rotary:]


def _rotate(x, cos, sin):
    x1, x2, rest = _halves(x.float(), 2 * cos.shape[-1])
    return torch.cat((x1 * cos - x2 * sin, x2 * cos + x1 * sin, rest), -1).to(x.dtype)


def _quantise(x):
    """Rows [T, heads, dim] as codes [T, heads, dim] and float16 scales and minima [T, heads, dim / 64, 2]."""
    g = x.float().clamp(-LARGEST, LARGEST).unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s, m = ((hi - lo) / 15).half(), lo.half()
    codes = ((g - m.float()) / s.float()).round().clamp(0, 15)
    codes = torch.where(s == 0, 0.0, codes).to(torch.uint8)
    return codes.flatten(-2), torch.cat((s, m), -1)


_SHIFT = [4 * (j // 2) + 16 * (j % 2) for j in range(8)]      # of channel j in a key's word


def _by_turns(units, groups):
    """Units of a row, group after group, in the order a cache holds them: those of two groups two and two."""
    return units.unflatten(-1, (-1, min(2, groups), units.shape[-1] // groups // 2, 2)).transpose(-3, -2).flatten(-4)


def _in_order(units, groups):
    return units.unflatten(-1, (-1, units.shape[-1] // groups // 2, min(2, groups), 2)).transpose(-3, -2).flatten(-4)


def _store(case, cache, slots, k, v):
    """Writes rows to their slots; a negative slot takes none."""
    page, dim = case["page"], case["dim"]
    kept = slots >= 0
    slots, k, v = slots[kept].long(), k[kept], v[kept]
    at, row = slots // page, slots % page
    if case["bits"] == 16:
        cache[0][at, row], cache[1][at, row] = k, v
        return
    codes, scales = _quantise(k)
    shift = torch.tensor(_SHIFT, device=DEV)
    words = _by_turns((codes.long().unflatten(-1, (-1, 8)) << shift).sum(-1), dim // GROUP)
    cache[0][at, :, row] = ((words[..., None] >> (8 * torch.arange(4, device=DEV))) & 255).flatten(-2).to(torch.uint8)
    cache[2][at, :, row] = scales
    codes, scales = _quantise(v)
    pair = codes.unflatten(-1, (-1, 2))
    words = cache[1].view(-1, case["kv_heads"], page // 4, dim // 2, 4)
    words[at, :, row // 4, :, row % 4] = _by_turns(pair[..., 0] | pair[..., 1] << 4, dim // GROUP)
    cache[3][at, :, :, row] = scales


def _load(case, cache, slots):
    """Rows [..., kv_heads, dim] of keys and of values, in 32 bits."""
    page, dim = case["page"], case["dim"]
    at, row = slots // page, slots % page
    if case["bits"] == 16:
        return cache[0][at, row].float(), cache[1][at, row].float()
    word = _in_order(cache[0].view(torch.int32).transpose(1, 2)[at, row], dim // GROUP)
    k = ((word[..., None] >> torch.tensor(_SHIFT, dtype=torch.int32, device=DEV)) & 15).flatten(-2)
    words = cache[1].view(-1, case["kv_heads"], page // 4, dim // 2, 4).permute(0, 2, 4, 1, 3)
    byte = _in_order(words[at, row // 4, row % 4], dim // GROUP)
    v = torch.stack((byte & 15, byte >> 4), -1).flatten(-2)
    scales = [cache[2].transpose(1, 2)[at, row].float(), cache[3].permute(0, 3, 1, 2, 4)[at, row].float()]
    return [(c.unflatten(-1, (-1, GROUP)) * s[..., :1] + s[..., 1:]).flatten(-2) for c, s in zip((k, v), scales)]


def _attend(q, k, v, allowed, scale):
    """q [B, Lq, heads, dim], k and v [B, Lk, kv_heads, dim] in 32 bits; allowed [B, Lq, Lk]."""
    b, lq, heads, dim = q.shape
    kv_heads = k.shape[2]
    q = q.unflatten(2, (kv_heads, -1)).permute(0, 2, 3, 1, 4).reshape(b, kv_heads, -1, dim)      # [B, kv, G Lq, dim]
    s = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).mul_(scale)
    s = s.view(b, kv_heads, -1, lq, k.shape[1])
    s.masked_fill_(~allowed[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(b, kv_heads, -1, k.shape[1]), v.permute(0, 2, 1, 3).contiguous())
    o = o.view(b, kv_heads, -1, lq, dim) / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).reshape(b, lq, heads, dim)


def _padded(cu, longest):
    """Rows [B, longest] of each sequence (0 behind its end), and which of them exist."""
    at = torch.arange(longest, device=DEV)
    there = at < (cu[1:] - cu[:-1])[:, None]
    return torch.where(there, cu[:-1, None] + at, 0), there


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "append":
        half = case["rotary"] // 2
        turn = state["cos_sin"][state["positions"]][:, None]
        q, k = (_rotate(state[x], turn[..., :half], turn[..., half:]) for x in "qk")
        _store(case, state["cache"], state["slots"], k, state["v"])
        if case["bits"] == 16:
            return {"q": q, "k": k, "k_cache": state["cache"][0], "v_cache": state["cache"][1]}
        kept = _load(case, state["cache"], state["every"].long())
        return {"q": q, "k": k, "k_cache": kept[0].to(q.dtype), "v_cache": kept[1].to(q.dtype)}
    if case["op"] == "gather":
        return [x.to(DTYPES[case["dtype"]]) for x in _load(case, state["cache"], state["slots"].long())]
    if case["op"] == "prompt":
        q, k, v, cu_q, cu_k = (state[x] for x in ("q", "k", "v", "cu_q", "cu_k"))
        rows_q, there_q = _padded(cu_q, max(_fresh(case)))
        rows_k, there_k = _padded(cu_k, case["longest"])
        # Row i of Lq queries stands at position i + Lk - Lq of the sequence.
        behind = ((cu_k[1:] - cu_k[:-1]) - (cu_q[1:] - cu_q[:-1]))[:, None, None]
        allowed = (torch.arange(rows_k.shape[1], device=DEV)
                   <= torch.arange(rows_q.shape[1], device=DEV)[:, None] + behind) & there_k[:, None]
        o = _attend(q.float()[rows_q], k.float()[rows_k], v.float()[rows_k], allowed, state["scale"])
        return o[there_q].to(q.dtype)
    page, lens = case["page"], state["lens"]
    at = torch.arange(case["longest"], device=DEV)
    there = at < lens[:, None]
    slots = torch.where(there, state["tables"].clamp(min=0)[:, at // page] * page + at % page, 0)
    k, v = _load(case, state["cache"], slots)
    o = _attend(state["q"].float()[:, None], k, v, there[:, None], state["scale"])
    return o[:, 0].to(state["q"].dtype)


def _run_own(case, state):
    ops = _kernels()
    if case["op"] == "append":
        cache = state["cache"]
        q, k = ops.rope_append(state["q"], state["k"], state["v"], state["positions"], state["cos_sin"],
                               state["slots"], *cache)
        if case["bits"] == 16:
            return {"q": q, "k": k, "k_cache": cache[0], "v_cache": cache[1]}
        kept = ops.kv_gather(*cache[:2], state["every"], *cache[2:], out_dtype=q.dtype)
        return {"q": q, "k": k, "k_cache": kept[0], "v_cache": kept[1]}
    if case["op"] == "gather":
        cache = state["cache"]
        return ops.kv_gather(*cache[:2], state["slots"], *cache[2:], out_dtype=DTYPES[case["dtype"]])
    if case["op"] == "prompt":
        return ops.attention_prompt(state["q"], state["k"], state["v"], state["cu_q"], state["cu_k"], state["scale"])
    cache = state["cache"]
    return ops.attention_paged(state["q"], *cache[:2], state["tables"], state["lens"], state["scale"], *cache[2:])


# ---------------------------------------------------------------------------
# What a pass cannot do without.
# ---------------------------------------------------------------------------
def _row_bytes(case):
    """Bytes of one cached token, keys and values."""
    per = case["dim"] * 2 if case["bits"] == 16 else case["dim"] // 2 + case["dim"] // GROUP * 4
    return 2 * case["kv_heads"] * per


def work(case):
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        t = case["tokens"]
        moved = 2 * t * dim * (2 * heads + 3 * kv_heads) + t * (_row_bytes(case) + 4 * case["rotary"] + 12)
        return {"bytes": moved, "flops": 3 * t * (heads + kv_heads) * case["rotary"]}
    if case["op"] == "gather":
        return {"bytes": case["tokens"] * (_row_bytes(case) + 4 * kv_heads * dim + 4), "flops": 0}
    lengths = _lengths(case)
    if case["op"] == "prompt":
        fresh = _fresh(case)
        pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(fresh, lengths))
        return {"bytes": 4 * dim * (heads * sum(fresh) + kv_heads * sum(lengths)), "flops": 4 * dim * heads * pairs}
    pages = sum(-(-n // case["page"]) for n in lengths)
    return {"bytes": sum(lengths) * _row_bytes(case) + 4 * len(lengths) * heads * dim + 4 * (pages + len(lengths)),
            "flops": 4 * dim * heads * sum(lengths)}


# ---------------------------------------------------------------------------
# The definition in 64 bits, sequence by sequence.
# ---------------------------------------------------------------------------
def _stands_for(row):
    """What a 4-bit cache keeps of rows [T, heads, dim], in 64 bits."""
    x = row.double().clamp(-LARGEST, LARGEST).unflatten(-1, (-1, GROUP))
    low = x.min(-1, keepdim=True).values.half().double()
    step = ((x.max(-1, keepdim=True).values - x.min(-1, keepdim=True).values) / 15).half().double()
    code = torch.where(step > 0, ((x - low) / torch.where(step > 0, step, 1.0)).round().clamp(0, 15), 0.0)
    return (code * step + low).flatten(-2)


def _slot_rows(case, cache, slots):
    """The rows of slots in 64 bits, element by element from the cache's bytes."""
    dim, page = case["dim"], case["page"]
    slots = slots.long()
    at, row = slots // page, slots % page
    if case["bits"] == 16:
        return [c[at, row].double() for c in cache]
    channel = torch.arange(dim, device=DEV)
    # Unit u of its group, in a block of one or two groups.
    def place(u, per_group):
        if dim == GROUP:
            return u
        return channel // (2 * GROUP) * 2 * per_group + u // 2 * 4 + channel // GROUP % 2 * 2 + u % 2
    bit = channel % 8 // 2 * 4 + channel % 2 * 16
    byte = cache[0][at, :, row][:, :, place(channel % GROUP // 8, GROUP // 8) * 4 + bit // 8]
    k = (byte >> (bit % 8).to(torch.uint8)) & 15
    index = (row // 4)[:, None] * (2 * dim) + place(channel % GROUP // 2, GROUP // 2) * 4 + (row % 4)[:, None]
    whole = cache[1].flatten(2)[at]
    byte = torch.gather(whole, 2, index[:, None].expand(-1, whole.shape[1], -1))
    v = (byte >> (channel % 2 * 4).to(torch.uint8)) & 15
    rows = []
    for code, pair in zip((k, v), (cache[2][at, :, row], cache[3][at, :, :, row])):
        pair = pair.double()[:, :, channel // GROUP]
        rows.append(code.double() * pair[..., 0] + pair[..., 1])
    return rows


def _softmax_rows(q, k, v, scale, first):
    """q [Lq, G, dim], k and v [Lk, dim]: row i over keys 0 .. first + i."""
    s = torch.einsum("igd,jd->gij", q, k) * scale
    at = torch.arange(k.shape[0], device=DEV)
    s = s.masked_fill(at > first + torch.arange(q.shape[0], device=DEV)[:, None], -math.inf)
    return torch.einsum("gij,jd->igd", torch.softmax(s, -1), v)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "append":
        half = case["rotary"] // 2
        angle = state["cos_sin"].double()[state["positions"]]
        turn = torch.complex(angle[:, :half], angle[:, half:])[:, None]
        out = {}
        for name in "qk":
            x = state[name].double()
            y = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
            out[name] = torch.cat((y.real, y.imag, x[..., 2 * half:]), -1)
        where = state["slots"].long()
        for name, rows in (("k_cache", out["k"]), ("v_cache", state["v"].double())):
            rows = rows.to(DTYPES[case["dtype"]])      # a cache keeps the rounded row
            kept = torch.zeros(state["every"].numel(), *rows.shape[1:], dtype=torch.float64, device=DEV)
            kept[where[where >= 0]] = (_stands_for(rows) if case["bits"] == 4 else rows.double())[where >= 0]
            out[name] = kept if case["bits"] == 4 else kept.view(state["cache"][0].shape)
        return out
    if case["op"] == "gather":
        return _slot_rows(case, state["cache"], state["slots"])
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    group, outs, at_q, at_k = heads // kv_heads, [], 0, 0
    lengths = _lengths(case)
    for b, n in enumerate(lengths):
        if case["op"] == "prompt":
            m = _fresh(case)[b]
            q, k, v = (state[x][at:at + size].double() for x, at, size in
                       (("q", at_q, m), ("k", at_k, n), ("v", at_k, n)))
            at_q, at_k = at_q + m, at_k + n
        else:
            m, token = 1, torch.arange(n, device=DEV)
            q = state["q"][b:b + 1].double()
            k, v = _slot_rows(case, state["cache"],
                              state["tables"][b].long()[token // case["page"]] * case["page"] + token % case["page"])
        o = torch.empty(m, heads, dim, dtype=torch.float64, device=DEV)
        for h in range(kv_heads):
            some = slice(h * group, (h + 1) * group)
            for i in range(0, m, 2048):      # rows in pieces: the scores of a long prompt are large
                o[i:i + 2048, some] = _softmax_rows(q[i:i + 2048, some], k[:n - m + min(m, i + 2048), h],
                                                    v[:n - m + min(m, i + 2048), h], state["scale"], n - m + i)
        outs.append(o)
    return torch.cat(outs)
