"""A 4-bit cache byte for byte, and attention over it within a bound derived
from its scales: the bound itself on the CPU, the kernels on the GPU."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from conftest import PKG
from oracle import attention_oracle as orc

K = PKG.kernels
BF16, F16 = torch.bfloat16, torch.float16
IDS = {BF16: "bf16", F16: "f16"}


def _say(*what):
    print(*what, flush=True)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _numpy(cache):
    return [t.cpu().numpy().copy() for t in cache]


def _still(device):
    """A table that turns by nothing."""
    return torch.cat((torch.ones(1, 16), torch.zeros(1, 16)), 1).to(device)


def _append(k, v, slots, cache, backend):
    at = torch.zeros(k.shape[0], dtype=torch.int64, device=k.device)
    K.rope_append_kv(k, k, v, at, _still(k.device), slots, cache, backend=backend)


# ---------------------------------------------------------------------------
# rope_append: every byte
# ---------------------------------------------------------------------------
def _noisy(cache, gen):
    """Contents that no call may change: any codes, scales with NaN among them."""
    out = []
    for t in cache:
        if t.dtype == torch.uint8:
            out.append(torch.randint(0, 256, t.shape, generator=gen, dtype=torch.uint8))
        else:
            x = torch.randn(t.shape, generator=gen).to(t.dtype)
            out.append(torch.where(torch.rand(t.shape, generator=gen) < 0.3, torch.nan, x))
    return out


def _slots(kind, tokens, capacity, gen):
    if kind == "random":
        return torch.randperm(capacity, generator=gen)[:tokens]
    slots = torch.arange(tokens) + (0 if kind == "aligned" else 3)
    if tokens > 9:
        slots[tokens // 2], slots[tokens // 2 + 4] = -1, capacity + 7
    return slots


def _append_and_compare(device, backend, dtype, dim, kv, size, tokens, kind):
    gen = _gen(tokens * dim + kv)
    blocks = -(-60 // size)
    k, v = (torch.randn((tokens, kv, dim), generator=gen).to(dtype) for _ in range(2))
    if tokens > 5:
        v[3, 0, dim // 2], v[5] = torch.nan, 2.0
    table, positions = K.rope_table(500, 32), torch.randint(0, 500, (tokens,), generator=gen)
    if tokens > 2:
        positions[1], positions[2] = 500, -1       # outside the table: NaN in the group that turns
    slots = _slots(kind, tokens, blocks * size, gen)
    want = _noisy(K.new_kv_cache(blocks, size, kv, dim, bits=4), gen)
    cache = K.KVCache(*[t.to(device) for t in want])
    want = [t.numpy() for t in want]
    K.rope_append_kv(k.to(device), k.to(device), v.to(device), positions.to(device), table.to(device),
                     slots.to(torch.int32).to(device), cache, backend=backend)
    turned = orc.rotate(k, positions.tolist(), table)
    for t, s in enumerate(slots.tolist()):
        for h in range(kv):
            if 0 <= s < blocks * size:
                orc.write_row(want, s, h, turned[t, h].float().numpy(), v[t, h].float().numpy())
    got = _numpy(cache)
    for name, a, b in zip(("k", "v"), got, want):
        assert np.array_equal(a, b), name      # codes of a group with a NaN are 0
    for name, a, b in zip(("k_scales", "v_scales"), got[2:], want[2:]):
        same = (a.view(np.uint16) == b.view(np.uint16)) | (np.isnan(a) & np.isnan(b))
        assert same.all(), name


APPENDED = [(tokens, kind) for tokens in (1, 7, 41) for kind in ("aligned", "shifted", "random")]


@pytest.mark.parametrize("dim,kv,size", [(64, 3, 16), (128, 2, 48)])
@pytest.mark.parametrize("tokens,kind", APPENDED)
def test_torch_backend_leaves_every_other_byte(dim, kv, size, tokens, kind):
    _append_and_compare("cpu", "torch", BF16, dim, kv, size, tokens, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("dim,kv,size", [(64, 3, 16), (128, 2, 48), (256, 1, 16), (128, 5, 256)])
@pytest.mark.parametrize("tokens,kind", APPENDED)
def test_append_leaves_every_other_byte(dtype, dim, kv, size, tokens, kind):
    """Written rows by the oracle, every other byte as it was: words that four tokens share among them."""
    _say("every byte", dtype, dim, kv, size, tokens, kind)
    _append_and_compare("cuda:0", "hip", dtype, dim, kv, size, tokens, kind)


# ---------------------------------------------------------------------------
# attention_paged over 4-bit pages
# ---------------------------------------------------------------------------
# (lengths, page, heads, kv_heads, dim, magnitude of the values)
PAGED = [(lens, size, heads, kv, dim, 1.0)
         for lens, size, heads, kv in (([1, 15, 16, 17], 16, 4, 4), ([31, 32, 33, 127, 128, 129], 48, 8, 2),
                                       ([257, 1000], 256, 5, 1), ([700], 32, 40, 2))
         for dim in (64, 128, 256)]
PAGED += [([300, 40], 16, 4, 2, 128, m) for m in (1e-3, 300.0, 20000.0)]      # scales above 32 in the last two
PAGED += [([9000] + [1 + 7 * i % 60 for i in range(140)], 16, 4, 2, 64, 1.0)]
PAGED_IDS = [f"{len(p[0])}x{p[0][0]}-{p[4]}-{p[5]:g}" for p in PAGED]


def _paged_case(lens, size, heads, kv, dim, magnitude, dtype, device, backend):
    gen = _gen(sum(lens) + dim)
    need = [-(-n // size) for n in lens]
    blocks = sum(need) + 2
    order = torch.randperm(blocks, generator=gen).tolist()
    tables, slots, at = torch.full((len(lens), max(need)), -1, dtype=torch.int32), [], 0
    for b, n in enumerate(lens):
        pages = order[at:at + need[b]]
        tables[b, :need[b]] = torch.tensor(pages, dtype=torch.int32)
        slots.append([pages[t // size] * size + t % size for t in range(n)])
        at += need[b]
    q = torch.randn((len(lens), heads, dim), generator=gen).to(dtype)
    total = sum(lens)
    k = (torch.randn((total, kv, dim), generator=gen) + torch.randn((kv, dim), generator=gen)).to(dtype)
    v = (torch.randn((total, kv, dim), generator=gen) * magnitude).to(dtype)
    cache = K.KVCache(*[t.to(device) for t in _noisy(K.new_kv_cache(blocks, size, kv, dim, bits=4), gen)])
    _append(k.to(device), v.to(device), _i32([s for x in slots for s in x], device), cache, backend)
    return q.to(device), cache, tables.to(device), slots


def _tiles(lens, kv, heads):
    """Most tiles of 32 tokens that one wave adds up: a pair (sequence, key-value head, 16 query heads) has a unit per
    128 tokens and 3 to begin, a unit is one tile of each of 4 waves, and 512 workgroups or more share them evenly."""
    units = sum(3 + -(-n // 128) for n in lens) * kv * -(-heads // kv // 16)
    return min(-(-max(lens) // 128), -(-units // 512))


def _bounds(q, cache, slots, lens, scale):
    """out and tolerance [batch, heads, dim]."""
    kv, now, rows = cache.k.shape[1], _numpy(cache), []
    for b, mine in enumerate(slots):
        keys, values = orc.read_rows(now, mine)
        rows.append(orc.attend_4bit(q[b:b + 1].cpu().double(), keys, values, scale, q.dtype,
                                    _tiles(lens, kv, q.shape[1])))
    return [torch.cat(x) for x in zip(*rows)]


def _outside(got, out, tol):
    return ~((got.cpu().double() - out).abs() <= tol)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("case", PAGED, ids=PAGED_IDS)
def test_the_bound_rejects_what_is_wrong(dtype, case):
    """Zeros leave the bound in nearly all elements, outputs 3% off in a fifth or more (small sums of large parts may be
    that far off); what the torch backend computes in 32 bits does not."""
    lens, heads, dim = case[0], case[2], case[4]
    q, cache, tables, slots = _paged_case(*case, dtype, "cpu", "torch")
    out, tol = _bounds(q, cache, slots, lens, dim ** -0.5)
    got = K.paged_attention(q, cache, tables, _i32(lens, "cpu"), dim ** -0.5, backend="torch")
    assert not _outside(got, out, tol).any()
    assert _outside(torch.zeros_like(out), out, tol).float().mean() > 0.95
    assert _outside(out * 1.03, out, tol).float().mean() > 0.2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("case", PAGED, ids=PAGED_IDS)
def test_paged_4bit_within_the_bound(dtype, case):
    lens, dim = case[0], case[4]
    _say("paged 4 bit", dtype, case[1:], lens[:6])
    q, cache, tables, slots = _paged_case(*case, dtype, "cuda:0", "hip")
    out, tol = _bounds(q, cache, slots, lens, dim ** -0.5)
    got = K.attention_paged(q, cache.k, cache.v, tables, _i32(lens, "cuda:0"), dim ** -0.5, cache.k_scales,
                            cache.v_scales)
    bad = _outside(got, out, tol)
    worst = ((got.cpu().double() - out).abs() / tol).max()
    _say("largest share of the bound", float(worst))
    assert not bad.any(), (int(bad.sum()), float(worst))


def _one_large_score(n, down, dim, dtype, device):
    """q, keys, values, scale: key 0 scores `down` powers of two above all others, and its value is 0."""
    q, k = torch.ones((1, 1, dim)), torch.zeros((n, 1, dim))
    k[0] = 1.0
    v = torch.linspace(0.5, 1.5, dim).expand(n, 1, dim).clone()
    v[0] = 0.0
    return *(x.to(dtype).to(device) for x in (q, k, v)), down * math.log(2) / dim


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,page", [(5, 16), (20, 16), (45, 32), (140, 48)])
def test_paged_4bit_depends_on_its_own_scales_only(dim, n, page):
    """What scales hold behind a sequence's end, and in pages it has none of, changes no bit of its output.  (Its
    weights, 2^-17 of the largest, would lose bits if such a scale took the factor off that P is held with.)"""
    _say("own scales", dim, n, page)
    q, k, v, scale = _one_large_score(n, 17.3, dim, F16, "cuda:0")
    blocks = -(-n // page)
    pages = list(range(1, blocks + 1))
    slots = _i32([pages[t // page] * page + t % page for t in range(n)], "cuda:0")
    outs = []
    for left in (0.0, 33.0, 1000.0, 60000.0, torch.inf, torch.nan):
        cache = K.new_kv_cache(blocks + 2, page, 1, dim, bits=4, device="cuda:0")
        cache.v_scales.fill_(left)
        cache.k_scales.fill_(left)
        _append(k, v, slots, cache, "hip")
        outs.append(K.attention_paged(q, cache.k, cache.v, _i32([pages + [0]], "cuda:0"), _i32([n], "cuda:0"), scale,
                                      cache.k_scales, cache.v_scales))
    assert not torch.isnan(outs[0]).any() and outs[0].any()
    for x in outs[1:]:
        assert torch.equal(x, outs[0])


# ---------------------------------------------------------------------------
# The ends of float16's range
# ---------------------------------------------------------------------------
def _extreme_rows(dim, dtype):
    """Groups whose top code is at, or near, the largest float16."""
    top, at = 65504.0, torch.arange(dim)
    ranges = [(-top, top), (0.0, top), (-top, 0.0), (top, top), (-top, -top), (60000.0, top), (-3000.0, top),
              (-50000.0, 65000.0), (-20000.0, 65472.0), (-65472.0, 65472.0), (torch.finfo(dtype).min, torch.finfo(dtype).max)]
    rows = [torch.where(at % 3 == 0, hi, torch.where(at % 3 == 1, lo, (lo + hi) / 2)) for lo, hi in ranges[:-1]]
    lo, hi = ranges[-1]
    rows.append(torch.where(at % 2 == 0, torch.full((dim,), hi), torch.full((dim,), lo)))
    rows.append(torch.where(at % 2 == 0, torch.inf, -torch.inf) * torch.ones(dim))
    return torch.stack(rows)[:, None].to(dtype)


def _finite_rows_stay_finite(device, backend, dtype, dim):
    rows = _extreme_rows(dim, dtype)
    n = rows.shape[0]
    slots = [(5 * t + 3) % 32 for t in range(n)]
    cache = K.new_kv_cache(2, 16, 1, dim, bits=4, device=device)
    want = _numpy(K.new_kv_cache(2, 16, 1, dim, bits=4))
    x = rows.to(device)
    still = torch.cat((torch.ones(1, 16), torch.zeros(1, 16)), 1)
    keys = torch.where(torch.isinf(rows), 0.0, rows)      # an infinity turns by 0 x infinity
    K.rope_append_kv(keys.to(device), keys.to(device), x, torch.zeros(n, dtype=torch.int64, device=device),
                     still.to(device), _i32(slots, device), cache, backend=backend)
    turned = orc.rotate(keys, [0] * n, still)
    for t, s in enumerate(slots):
        orc.write_row(want, s, 0, turned[t, 0].float().numpy(), rows[t, 0].float().numpy())
    for a, b in zip(_numpy(cache), want):
        assert np.array_equal(a, b)
    _, (code, step, low) = orc.read_rows(want, slots)
    stands_for = code * step + low
    assert float(stands_for.abs().max()) <= 65504.0
    # Half of a code's step, and what rounding the scale down adds at code 15.
    off = (stands_for - rows.double().clamp(-65504, 65504)).abs()
    assert (off <= 0.5 * step + 15 * 8 + 16).all()
    for out_dtype in (F16, BF16):
        for got in K.gather_kv(cache, _i32(slots, device), out_dtype, backend=backend):
            assert torch.isfinite(got).all()


@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("dim", [64, 256])
def test_torch_backend_keeps_finite_rows_finite(dtype, dim):
    _finite_rows_stay_finite("cpu", "torch", dtype, dim)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_finite_rows_stay_finite(dtype, dim):
    """Rows are clamped to float16's range so that they stay finite; what their codes stand for stays in it too."""
    _say("ends of the range", dtype, dim)
    _finite_rows_stay_finite("cuda:0", "hip", dtype, dim)
