"""The attention operators from their definitions, on the CPU: rotation, the
4-bit form of a cached row, and attention in 64 bits with the bound that each
type's roundings allow.

The reference's layers (nanovllm/layers/rotary_embedding.py,
nanovllm/layers/attention.py) need flash-attn and cannot run here: parity with
their outputs is unpinned; these are the formulas they compute.
"""
from __future__ import annotations

import numpy as np
import torch

GROUP = 64


def rotate(x: torch.Tensor, positions, cos_sin: torch.Tensor) -> torch.Tensor:
    """x [T, heads, dim] rotated: float32 products and sums rounded one by one, one rounding to x.dtype."""
    half = cos_sin.shape[1] // 2
    table = cos_sin.numpy()
    out = x.float().numpy().copy()
    for t, pos in enumerate(positions):
        turn = table[pos] if 0 <= pos < len(table) else np.full(2 * half, np.nan, np.float32)
        c, s = turn[:half], turn[half:]
        x1, x2 = out[t, :, :half].copy(), out[t, :, half:2 * half].copy()
        out[t, :, :half] = (x1 * c).astype(np.float32) - (x2 * s).astype(np.float32)
        out[t, :, half:2 * half] = (x2 * c).astype(np.float32) + (x1 * s).astype(np.float32)
    return torch.from_numpy(out).to(x.dtype)


def code_row(row: np.ndarray):
    """One head's row (float32 [dim]) in 4 bits: codes [dim], float16 scales and minima [dim / 64]."""
    codes, scales, minima = [], [], []
    for g in np.clip(row.astype(np.float32), -65504, 65504).reshape(-1, GROUP):
        if np.isnan(g).any():
            codes += [0] * GROUP
            scales.append(np.float16(np.nan))
            minima.append(np.float16(np.nan))
            continue
        s = np.float16((g.max() - g.min()) / np.float32(15))
        m = np.float16(g.min())
        if 15.0 * float(s) + float(m) > 65504.0:      # a finite row stays finite: code 15 in float16's range
            s = np.nextafter(s, np.float16(0))
        if s > 0:
            q = np.rint((g - np.float32(m)) / np.float32(s))
            codes += [int(v) for v in np.clip(q, 0, 15)]
        else:
            codes += [0] * GROUP
        scales.append(s)
        minima.append(m)
    return np.array(codes, np.uint8), np.array(scales, np.float16), np.array(minima, np.float16)


def word_place(dim: int, channel: int, per_group: int, word: int) -> int:
    """Place of a group's word in its row: those of two neighbouring groups take turns two by two."""
    groups, g = dim // GROUP, channel // GROUP
    if groups == 1:
        return word
    return g // 2 * 2 * per_group + word // 2 * 4 + g % 2 * 2 + word % 2


def write_row(cache, slot: int, head: int, key: np.ndarray, value: np.ndarray) -> None:
    """Codes one row of keys and of values into a 4-bit cache of numpy arrays (k, v, k_scales, v_scales)."""
    k, v, ks, vs = cache
    size, dim = k.shape[2], 2 * k.shape[3]
    block, at = divmod(slot, size)
    codes, s, m = code_row(key)
    line = np.zeros(dim // 8, np.uint32)
    for c in range(dim):
        j = c % 8
        line[word_place(dim, c, 8, c % GROUP // 8)] |= np.uint32(int(codes[c]) << (4 * (j // 2) + 16 * (j % 2)))
    k[block, head, at] = line.view(np.uint8)
    ks[block, head, at, :, 0], ks[block, head, at, :, 1] = s, m
    codes, s, m = code_row(value)
    whole = v[block, head].reshape(size // 4, dim // 2, 4)
    for c in range(0, dim, 2):
        whole[at // 4, word_place(dim, c, 32, c % GROUP // 2), at % 4] = codes[c] | codes[c + 1] << 4
    vs[block, head, :, at, 0], vs[block, head, :, at, 1] = s, m


def read_row(cache, slot: int, head: int):
    """(key, value) of a slot in 64 bits, and (codes times scale, minimum) of the value."""
    k, v, ks, vs = cache
    size, dim = k.shape[2], 2 * k.shape[3]
    block, at = divmod(slot, size)
    c = np.arange(dim)
    place = np.array([word_place(dim, x, 8, x % GROUP // 8) for x in range(dim)])
    word = np.ascontiguousarray(k[block, head, at]).view(np.uint32)[place]
    code = (word >> (4 * (c % 8 // 2) + 16 * (c % 2)).astype(np.uint32)) & 15
    pair = ks[block, head, at].astype(np.float64)
    key = code * pair[c // GROUP, 0] + pair[c // GROUP, 1]
    place = np.array([word_place(dim, x, 32, x % GROUP // 2) for x in range(dim)])
    byte = v[block, head].reshape(size // 4, dim // 2, 4)[at // 4, place, at % 4]
    code = (byte >> (4 * (c % 2)).astype(np.uint8)) & 15
    pair = vs[block, head, :, at].astype(np.float64)
    high, low = code * pair[c // GROUP, 0], pair[c // GROUP, 1]
    return key, high + low, high, low


def attend(q, k, v, scale, first=None):
    """float64 q [m, heads, dim], k and v [n, kv_heads, dim] -> (out, weights, scores' magnitude).

    Row i sees keys 0 .. first + i, or all of them; a row that sees none is 0.
    weights: [heads, m, n]; magnitude: the largest scale sum |q| |k| of a row, [m, heads, 1]."""
    group = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    seen = torch.ones(q.shape[0], k.shape[0], dtype=torch.bool)
    if first is not None:
        seen = torch.arange(k.shape[0]) <= first + torch.arange(q.shape[0])[:, None]
    s = torch.einsum("ihd,jhd->hij", q, k) * scale
    s = torch.where(seen, s, -torch.inf)
    w = torch.where(seen.any(-1)[:, None], torch.softmax(s, -1), 0.0) if k.shape[0] else s
    w = torch.where(seen, w, 0.0)
    # A key that is not seen has no part, whatever its value holds.
    out = torch.zeros(q.shape, dtype=torch.float64)
    for i in range(q.shape[0]):
        n = int(seen[i].sum())
        out[i] = torch.einsum("hj,jhd->hd", w[:, i, :n], v[:n])
    big = torch.where(seen, torch.einsum("ihd,jhd->hij", q.abs(), k.abs()) * scale, 0.0)
    big = big.amax(-1).T[..., None] if k.shape[0] else torch.zeros(*q.shape[:2], 1, dtype=torch.float64)
    return out, w, big


def tolerance(out, absolute, big, dtype, dim: int, *, p_half_step: float):
    """How far a correct kernel's output may be from `out`.

    absolute: sum_j w_j |what P multiplies|.  One rounding of the output; one of each P (p_half_step, in the
    numerator and, where the total is of rounded P, in the denominator); scores are fp32 sums of dim products whose
    error e shifts a weight by a factor 1 + 2 e (numerator and denominator); 2^-20 for base-2 exponentials, the
    scaling and fp32 sums of weights."""
    half_step = torch.finfo(dtype).eps / 2
    w = 2 * (dim + 16) * 2.0 ** -24 * big + 2.0 ** -20
    return half_step * out.abs() + (p_half_step + w) * (absolute + out.abs()) * (1 + half_step) + 1e-30


def read_rows(cache, slots):
    """Rows of a 4-bit cache of numpy arrays, for slots [n]: (codes, scales, minima) of keys and of values, float64
    [n, heads, dim] each."""
    k, v, ks, vs = cache
    size, dim = k.shape[2], 2 * k.shape[3]
    block, at = np.divmod(np.asarray(slots, dtype=np.int64), size)
    c = np.arange(dim)
    word = np.ascontiguousarray(k[block, :, at]).view(np.uint32)
    word = word[..., [word_place(dim, x, 8, x % GROUP // 8) for x in c]]
    code_k = (word >> (4 * (c % 8 // 2) + 16 * (c % 2)).astype(np.uint32)) & 15
    byte = v.reshape(*v.shape[:2], size // 4, dim // 2, 4)[block, :, at // 4, :, at % 4]
    byte = byte[..., [word_place(dim, x, 32, x % GROUP // 2) for x in c]]
    code_v = (byte >> (4 * (c % 2)).astype(np.uint8)) & 15
    pairs = [p.astype(np.float64)[:, :, c // GROUP] for p in (ks[block, :, at], vs[block, :, :, at])]
    return [[torch.from_numpy(x) for x in (code.astype(np.float64), p[..., 0], p[..., 1])]
            for code, p in zip((code_k, code_v), pairs)]


def attend_4bit(q, keys, values, scale, dtype, tiles: int):
    """One query row float64 [1, heads, dim] over 4-bit rows (`read_rows`): (out, how far a correct kernel may be off).

    With key c s + m, a kernel may sum products on 16 + c and take m - 16 s apart, in fp32: a product goes through
    the 64 sums of its group and 16 further roundings, each of half a last place (2^-24) of what is added up.  An error
    e of a score changes its weight by a factor 1 + e, of which the total has the mean.  2^-20: base-2 exponentials and
    the scaling.
    With value (c - 7.5) s + (m + 7.5 s) and weight p: p s, p and m + 7.5 s are rounded to float16 (2^-11 each, or
    2^-25 in its subnormal range: of p and p s held 2^10 fold where all scales are at most 32), the total of the
    rounded p divides.  Sums of (64 + c) p s and of 64 + 7.5 times the p s run over `tiles` tiles of 32 tokens: 32
    and 8 additions a tile and 8 to join lanes, of at most one last place (2^-23) of (64 + 15) p s.  Then one rounding
    to dtype.  1 + 2^-6: products of these errors."""
    (ck, sk, mk), (cv, sv, mv) = keys, values
    group = q.shape[1] // ck.shape[1]
    out, w, _ = attend(q, ck * sk + mk, cv * sv + mv, scale)
    heads = lambda x: x.repeat_interleave(group, 1)      # noqa: E731
    spread = lambda x: torch.einsum("hij,jhd->ihd", w, heads(x))      # noqa: E731
    score = torch.einsum("ihd,jhd->hij", q.abs(), heads((16 + ck) * sk + (mk - 16 * sk).abs())) * scale
    error = w * (80 * 2.0 ** -24 * score + 2.0 ** -20)
    value = (cv * sv + mv).abs()
    n, around, middle = ck.shape[0], (cv - 7.5).abs() * sv, (mv + 7.5 * sv).abs()
    half = 2.0 ** -11
    least = 2.0 ** -35 if bool((sv <= 32).all()) else 2.0 ** -25
    off = half * (spread(around) + 2 * spread(middle) + out.abs())
    off = off + torch.einsum("hij,jhd->ihd", error, heads(value)) + error.sum(-1).T[..., None] * out.abs()
    off = off + least * (7.5 * n + heads(middle).sum(0, keepdim=True) + n * out.abs()) + 2.0 ** -25
    off = off + (40 * tiles + 8) * 2.0 ** -23 * 79 * spread(sv)
    off = off * (1 + 2.0 ** -6)
    return out, off + torch.finfo(dtype).eps / 2 * (out.abs() + off)
