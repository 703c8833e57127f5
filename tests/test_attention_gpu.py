"""GPU tests of the attention operators (rotation and cache append, cache
reads, prompt and paged attention) against oracle/attention_oracle.py.

Rotation, codes and cached rows are compared bit for bit.  Attention is held
to the bound of its roundings: P is rounded to the operands' type (float16
next to 4-bit values), the output once, everything else is fp32."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import PKG
from oracle import attention_oracle as orc

pytestmark = pytest.mark.gpu

K = PKG.kernels
DEV = torch.device("cuda:0")
BF16, F16 = torch.bfloat16, torch.float16
IDS = {BF16: "bf16", F16: "f16"}


def _say(*what):
    print(*what, flush=True)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _bits(t):
    """The tensor's bytes on the CPU: comparison of NaNs and of signs too."""
    return t.cpu().contiguous().view(torch.uint8)


def _numpy(cache):
    return [t.cpu().numpy().copy() for t in cache]


def _noise(shape, dtype, gen):
    """Contents that no call may change or use: NaN among them."""
    if dtype == torch.uint8:
        return torch.randint(0, 256, shape, generator=gen, dtype=torch.uint8).to(DEV)
    x = torch.randn(shape, generator=gen).to(dtype)
    return torch.where(torch.rand(shape, generator=gen) < 0.3, torch.nan, x).to(DEV)


def _noisy_cache(blocks, size, heads, dim, bits, dtype, gen):
    empty = K.new_kv_cache(blocks, size, heads, dim, bits=bits, dtype=dtype)
    return K.KVCache(*[None if t is None else _noise(t.shape, t.dtype, gen) for t in empty])


# ---------------------------------------------------------------------------
# rope_append and kv_gather
# ---------------------------------------------------------------------------
def _slots(kind, tokens, capacity, gen):
    if kind == "random":
        return torch.randperm(capacity, generator=gen)[:tokens]
    start = 0 if kind == "aligned" else 3
    slots = torch.arange(start, start + tokens)
    if tokens > 4:
        slots[tokens // 2] = -1
    if tokens > 9:
        slots[tokens // 2 + 4] = capacity + 7      # behind the cache: takes no row either
    return slots


@pytest.mark.parametrize("bits,size", [(16, 16), (16, 23), (4, 16), (4, 48)])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("dim,rotary,heads,kv", [(64, 64, 3, 3), (128, 16, 6, 2), (256, 64, 8, 1), (128, 128, 5, 5)])
@pytest.mark.parametrize("tokens,kind", [(1, "random"), (7, "aligned"), (41, "shifted"), (40, "random")])
def test_rope_append(bits, size, dtype, dim, rotary, heads, kv, tokens, kind):
    _say("rope_append", bits, size, dtype, dim, rotary, heads, kv, tokens, kind)
    gen = _gen(tokens * dim + heads)
    blocks = -(-60 // size)
    rows = torch.randn((tokens, (heads + 2 * kv) * dim), generator=gen).to(dtype)
    q, k, v = (x.view(tokens, -1, dim) for x in rows.to(DEV).split([heads * dim, kv * dim, kv * dim], 1))
    table = K.rope_table(500, rotary)
    positions = torch.randint(0, 500, (tokens,), generator=gen)
    if tokens > 2:
        positions[1], positions[2] = 500, -1       # outside the table
    slots = _slots(kind, tokens, blocks * size, gen)
    cache = _noisy_cache(blocks, size, kv, dim, bits, dtype, gen)
    before = _numpy([t.view(torch.int16) if t.dtype == BF16 else t for t in cache if t is not None])

    got_q, got_k = K.rope_append(q, k, v, positions.to(DEV), table.to(DEV), slots.to(torch.int32).to(DEV), *cache)
    torch.cuda.synchronize()

    want_q, want_k = (orc.rotate(x.cpu().contiguous(), positions.tolist(), table) for x in (q, k))
    for got, want in ((got_q, want_q), (got_k, want_k)):
        got = got.cpu()
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(got), nan)
        assert torch.equal(torch.where(nan, 0, got), torch.where(nan, 0, want))
    # The cache: written rows by the oracle, every other byte as it was.
    got_rows, value_rows = got_k.cpu(), v.cpu()
    if bits == 16:
        want = [torch.from_numpy(a).view(dtype).clone() if dtype == BF16 else torch.from_numpy(a) for a in before]
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < blocks * size:
                want[0][s // size, s % size], want[1][s // size, s % size] = got_rows[t], value_rows[t]
        assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip(cache[:2], want))
        return
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < blocks * size:
            for h in range(kv):
                orc.write_row(before, s, h, got_rows[t, h].float().numpy(), value_rows[t, h].float().numpy())
    for a, b, codes in zip(cache, before, (True, True, False, False)):
        a = a.cpu().numpy()
        # A group with a NaN reads back as NaN whatever its codes are.
        same = (a == b) if codes else (a.view(np.uint16) == b.view(np.uint16)) | (np.isnan(a) & np.isnan(b))
        if codes and np.isnan(before[2]).any():
            continue
        assert same.all()
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < blocks * size and tokens > 2:
            now = _numpy(cache)
            for h in range(kv):
                for a, b in zip(orc.read_row(now, s, h)[:2], orc.read_row(before, s, h)[:2]):
                    np.testing.assert_array_equal(a, b)
            if t > 6:
                break


@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
def test_rope_append_4bit_values_at_the_edges(dtype):
    """Groups that are constant, of one step, tiny, huge, infinite or hold a NaN."""
    _say("edges", dtype)
    dim, top = 128, torch.finfo(dtype).max
    rows = torch.zeros((9, 1, dim))
    rows[0] = 3.0
    rows[1] = torch.arange(dim) % 2 * 2.0 ** -24
    rows[2] = torch.randn((1, dim), generator=_gen(1)) * 1e-6
    rows[3] = torch.where(torch.arange(dim) % 3 == 0, top, -top)
    rows[4, 0, 5], rows[4, 0, 70] = torch.inf, -torch.inf
    rows[5, 0, 9] = torch.nan
    rows[6] = torch.arange(dim) / 7.0
    rows[7] = -1000.0 + torch.arange(dim) * 0.01
    rows[8] = torch.linspace(-1, 1, dim)
    x = rows.to(dtype).to(DEV)
    cache = K.new_kv_cache(2, 16, 1, dim, bits=4, device=DEV)
    table = torch.cat((torch.ones(1, 16), torch.zeros(1, 16)), 1).to(DEV)     # turns by nothing
    slots = _i32([5, 6, 7, 8, 9, 10, 11, 12, 17])
    K.rope_append(x, x, x, torch.zeros(9, dtype=torch.int64, device=DEV), table, slots, *cache)
    want = _numpy(K.new_kv_cache(2, 16, 1, dim, bits=4))
    for t, s in enumerate(slots.tolist()):
        orc.write_row(want, s, 0, x[t, 0].cpu().float().numpy(), x[t, 0].cpu().float().numpy())
    got = _numpy(cache)
    for s in slots.tolist():
        for a, b in zip(orc.read_row(got, s, 0)[:2], orc.read_row(want, s, 0)[:2]):
            if s != 9:      # infinite rows turn by 0 x infinity in the rotated channels of the key
                np.testing.assert_array_equal(a, b)
    assert np.array_equal(orc.read_row(got, 9, 0)[1], orc.read_row(want, 9, 0)[1])


@pytest.mark.parametrize("bits,size", [(16, 16), (16, 5), (4, 32)])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("dim,kv", [(64, 3), (128, 1), (256, 2)])
def test_kv_gather(bits, size, dtype, dim, kv):
    _say("kv_gather", bits, size, dtype, dim, kv)
    gen = _gen(dim + size)
    cache = K.KVCache(*[None if t is None else (torch.randint(0, 256, t.shape, generator=gen, dtype=torch.uint8)
                                                if t.dtype == torch.uint8 else
                                                torch.randn(t.shape, generator=gen).to(t.dtype)).to(DEV)
                        for t in K.new_kv_cache(4, size, kv, dim, bits=bits, dtype=dtype)])
    # Whole runs of four, runs that start inside a word, repeats, and slots outside the cache.
    slots = [0, 1, 2, 3, 4, 5, 6, 7, 9, 10, 11, 12, 13, 3, 3, -1, 4 * size, 2 ** 31 - 1, 4 * size - 1, 8, 9, 10, 11, 2]
    slots = [s % (4 * size) if 0 <= s < 4 * size + 20 and s != 4 * size else s for s in slots]
    k, v = K.kv_gather(cache.k, cache.v, _i32(slots), cache.k_scales, cache.v_scales, dtype)
    now = _numpy([t.float() if t.dtype == BF16 else t for t in cache if t is not None])
    for i, s in enumerate(slots):
        for h in range(kv):
            if not 0 <= s < 4 * size:
                want = np.zeros(dim), np.zeros(dim)
            elif bits == 16:
                want = [now[j][s // size, s % size, h].astype(np.float64) for j in range(2)]
            else:
                want = orc.read_row(now, s, h)[:2]
            for got, w in zip((k, v), want):
                # code * scale + minimum is rounded to float32, then to the type.
                w = torch.from_numpy(w).float().to(dtype)
                assert torch.equal(got[i, h].cpu(), w), (i, s, h)


@pytest.mark.parametrize("bits,size", [(16, 23), (4, 48)])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("dim,tokens", [(64, 4500), (128, 2301), (256, 2070)])
def test_rope_append_of_many_tokens(bits, size, dtype, dim, tokens):
    """A call of prompts (several heads and rows of values to a team) writes bit for bit what calls of at most 50 tokens
    write: sequences that begin at any slot of a page, rows that are kept nowhere, odd counts of heads."""
    _say("many tokens", bits, size, dtype, dim, tokens)
    gen, heads, kv = _gen(dim + bits), 10, 5
    rows = torch.randn((tokens, heads + 2 * kv, dim), generator=gen).to(dtype).to(DEV)
    q, k, v = rows.split([heads, kv, kv], 1)
    table = K.rope_table(1000, 32, device=DEV)
    positions = torch.randint(0, 1000, (tokens,), generator=gen).to(DEV)
    blocks = tokens // size + 20
    slots = torch.arange(tokens) + torch.repeat_interleave(torch.randint(0, 7, (tokens // 90 + 1,), generator=gen).cumsum(0),
                                                           90)[:tokens]
    slots[500:530] = slots[500:530].flip(0)
    slots[torch.randint(0, tokens, (9,), generator=gen)] = -1
    assert int(slots.max()) < blocks * size
    slots = slots.to(torch.int32).to(DEV)
    whole = _noisy_cache(blocks, size, kv, dim, bits, dtype, gen)
    parts = K.KVCache(*[None if x is None else x.clone() for x in whole])
    outs = K.rope_append(q, k, v, positions, table, slots, *whole)
    at = 0
    while at < tokens:
        n = at + int(torch.randint(1, 51, (1,), generator=gen))
        piece = K.rope_append(q[at:n], k[at:n], v[at:n], positions[at:n], table, slots[at:n], *parts)
        assert all(torch.equal(a[at:n], b) for a, b in zip(outs, piece)), at
        at = n
    for a, b in zip(whole, parts):
        assert a is b is None or torch.equal(_bits(a), _bits(b))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("dim,rows", [(64, 3300), (128, 2801), (256, 2760)])
def test_kv_gather_of_many_rows(dtype, dim, rows):
    """A long 4-bit gather (64 rows of values to a workgroup) reads bit for bit what calls of at most 50 rows read:
    runs that begin at any slot, slots outside the cache, the same slot twice."""
    _say("many rows", dtype, dim, rows)
    gen, kv, size = _gen(dim + rows), 3, 48
    blocks = rows // size + 4
    cache = _noisy_cache(blocks, size, kv, dim, 4, dtype, gen)
    slots = torch.arange(rows) + torch.repeat_interleave(torch.randint(0, 4, (rows // 90 + 1,), generator=gen).cumsum(0),
                                                         90)[:rows]
    slots[500:530] = slots[500:530].flip(0)
    slots[1000:1100] = torch.randint(0, blocks * size, (100,), generator=gen)
    slots[40:44] = slots[44:48]
    slots[torch.randint(0, rows, (9,), generator=gen)] = -1
    slots[2000], slots[rows - 1] = blocks * size, 2 ** 31 - 1
    slots = slots.to(torch.int32).to(DEV)
    k, v = K.kv_gather(cache.k, cache.v, slots, cache.k_scales, cache.v_scales, out_dtype=dtype)
    at = 0
    while at < rows:
        n = at + int(torch.randint(1, 51, (1,), generator=gen))
        pk, pv = K.kv_gather(cache.k, cache.v, slots[at:n], cache.k_scales, cache.v_scales, out_dtype=dtype)
        assert torch.equal(_bits(k[at:n]), _bits(pk)) and torch.equal(_bits(v[at:n]), _bits(pv)), at
        at = n


def test_appended_rows_read_back():
    """A cache written in pieces reads back as written at once, through blocks that are slices of a larger allocation."""
    _say("read back")
    gen = _gen(3)
    whole = torch.zeros((6, 2, 32, 2, 128), dtype=BF16, device=DEV)
    k_cache, v_cache = whole[:, 0], whole[:, 1]
    k, v = (torch.randn((100, 2, 128), generator=gen).to(BF16).to(DEV) for _ in range(2))
    table = K.rope_table(100, 128, device=DEV)
    slots = torch.randperm(192, generator=gen)[:100].to(torch.int32).to(DEV)
    at = torch.arange(100, device=DEV)
    keys = []
    for i, j in ((0, 1), (1, 60), (60, 100)):
        keys.append(K.rope_append(k[i:j], k[i:j], v[i:j], at[i:j], table, slots[i:j], k_cache, v_cache)[1])
    got_k, got_v = K.kv_gather(k_cache, v_cache, slots)
    assert torch.equal(got_k, torch.cat(keys)) and torch.equal(got_v, v)


# ---------------------------------------------------------------------------
# attention_prompt
# ---------------------------------------------------------------------------
def _check(got, out, absolute, big, dtype, dim, p_half_step, what):
    got = got.cpu().double()
    tol = orc.tolerance(out, absolute, big, dtype, dim, p_half_step=p_half_step)
    assert torch.equal(torch.isnan(got), torch.isnan(out)), what
    off = (got - out).abs() - tol
    bad = torch.where(torch.isnan(out) | (got == out), -1.0, off) > 0
    assert not bad.any(), (what, int(bad.sum()), float((got - out).abs().max()))


def _check_prompt(got, q, k, v, lq, lk, scale, causal, what):
    a = c = 0
    for n, m in zip(lq, lk):
        qs, ks, vs = q[a:a + n].cpu().double(), k[c:c + m].cpu().double(), v[c:c + m].cpu().double()
        if n:
            out, w, big = orc.attend(qs, ks, vs, scale, m - n if causal else None)
            size = vs.abs().nan_to_num(0, 0, 0).repeat_interleave(q.shape[1] // k.shape[1], 1)
            absolute = torch.einsum("hij,jhd->ihd", w, size)
            _check(got[a:a + n], out, absolute, big, q.dtype, q.shape[2], torch.finfo(q.dtype).eps / 2, (what, n, m))
        a, c = a + n, c + m


def _cu(lengths):
    return _i32([0] + list(np.cumsum(lengths)))


LENGTHS = [
    ([1], [1]),
    ([33, 1, 0, 64], [33, 1, 0, 64]),
    ([5, 130, 31], [5, 130, 31]),
    ([257], [257]),
    ([1, 7, 129], [40, 200, 300]),          # new tokens on cached ones
    ([20, 0, 3, 140], [3, 9, 0, 70]),       # more queries than keys: rows that see none
]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("dim,heads,kv", [(64, 4, 4), (128, 6, 2), (256, 8, 1)])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda x: "-".join(map(str, x[0])))
def test_attention_prompt(dtype, dim, heads, kv, causal, lengths):
    lq, lk = lengths
    _say("prompt", dtype, dim, heads, kv, causal, lengths)
    gen = _gen(sum(lq) + dim)
    q = torch.randn((sum(lq), heads, dim), generator=gen).to(dtype).to(DEV)
    kv_rows = torch.randn((sum(lk), 2 * kv * dim), generator=gen).to(dtype).to(DEV)
    k, v = (x.view(sum(lk), kv, dim) for x in kv_rows.chunk(2, 1))
    scale = dim ** -0.5
    got = K.attention_prompt(q, k, v, _cu(lq), _cu(lk), scale, causal)
    _check_prompt(got, q, k, v, lq, lk, scale, causal, "prompt")


@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
def test_attention_prompt_scores_of_every_size(dtype):
    """Sharp and flat rows, growing maxima (the sums are rescaled), a head whose scores are all equal."""
    _say("scores", dtype)
    gen = _gen(11)
    n, dim = 300, 128
    q = torch.randn((n, 3, dim), generator=gen)
    k = torch.randn((n, 3, dim), generator=gen) * torch.linspace(0.01, 6.0, n)[:, None, None]
    q[:, 1] = 0.0
    k[:, 2] = k[:, 2] - 4.0
    q, k, v = (x.to(dtype).to(DEV) for x in (q, k, torch.randn((n, 3, dim), generator=gen)))
    got = K.attention_prompt(q, k, v, _cu([n]), _cu([n]), 0.3)
    _check_prompt(got, q, k, v, [n], [n], 0.3, True, "scores")


@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_prompt_keeps_to_what_a_row_sees(dtype, dim):
    """NaN and infinities in keys and values that a row does not see change nothing in it: rows of other sequences,
    later tokens, rows behind the last sequence.  Where they are seen they spread as the sums do."""
    _say("masked places", dtype, dim)
    gen = _gen(dim)
    lens, spare = [70, 45, 1], 20
    n = sum(lens)
    q, k, v = (torch.randn((n + spare, 2, dim), generator=gen).to(dtype) for _ in range(3))
    clean_k, clean_v = k.clone(), v.clone()
    v[30, 0, 3], v[33, 1, 5], v[90, :, :] = torch.nan, torch.inf, -torch.inf
    k[60], k[n:], v[n:] = torch.nan, torch.nan, torch.inf
    got = K.attention_prompt(q.to(DEV), k.to(DEV), v.to(DEV), _cu(lens), _cu(lens), dim ** -0.5).cpu()
    want = K.attention_prompt(q.to(DEV), clean_k.to(DEV), clean_v.to(DEV), _cu(lens), _cu(lens), dim ** -0.5).cpu()
    assert not torch.isnan(want).any() and torch.equal(want[n:], torch.zeros_like(want[n:]))
    same = torch.ones(n + spare, 2, dim, dtype=torch.bool)
    same[30:70, 0, 3] = same[33:70, 1, 5] = False
    same[60:70] = same[90:115] = False
    assert torch.equal(got[same], want[same])
    assert torch.isnan(got[30:70, 0, 3]).all() and torch.isnan(got[60:70]).all()
    assert (got[33:60, 1, 5] == torch.inf).all()
    assert (got[90:115] == -torch.inf).all()


def test_attention_prompt_scores_that_are_not_finite():
    """Scores of -infinity drop their keys; a row whose every score is -infinity, or one with +infinity, is NaN."""
    _say("infinite scores")
    gen = _gen(5)
    q, k, v = (torch.randn((40, 1, 64), generator=gen).to(BF16) for _ in range(3))
    q[:, 0, 0], k[:, 0, 0] = 1.0, 0.0
    k[3, 0, 0], k[0, 0, 0], k[35, 0, 0] = -torch.inf, -torch.inf, torch.inf
    got = K.attention_prompt(q.to(DEV), k.to(DEV), v.to(DEV), _cu([40]), _cu([40]), 0.125).cpu()
    out, _, _ = orc.attend(q.double(), k.double(), v.double(), 0.125, 0)
    assert torch.isnan(got[0]).all() and torch.isnan(got[35:]).all()
    assert torch.equal(torch.isnan(got), torch.isnan(out))


def test_attention_prompt_many_sequences():
    """More sequences than a wave looks through at once."""
    _say("many sequences")
    gen = _gen(8)
    lens = torch.randint(0, 40, (150,), generator=gen).tolist()
    q, k, v = (torch.randn((sum(lens), h, 64), generator=gen).to(BF16).to(DEV) for h in (4, 2, 2))
    got = K.attention_prompt(q, k, v, _cu(lens), _cu(lens), 0.125)
    _check_prompt(got, q, k, v, lens, lens, 0.125, True, "many")


# Keys enough that blocks are cut into equal runs.
RUNS = [
    ([5, 130, 31, 0, 900], [5, 130, 31, 0, 1200]),
    ([1, 7, 129], [40, 200, 1300]),
    ([20, 0, 3, 140, 1], [3, 9, 0, 70, 1400]),
    ([1], [1250]),
]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("dim,heads,kv", [(64, 4, 4), (128, 6, 2), (256, 8, 1)])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("lengths", RUNS, ids=lambda x: "-".join(map(str, x[0])))
def test_attention_prompt_in_runs(dtype, dim, heads, kv, causal, lengths):
    lq, lk = lengths
    _say("prompt in runs", dtype, dim, heads, kv, causal, lengths)
    gen = _gen(sum(lk) + dim)
    q, k, v = (torch.randn((sum(n), h, dim), generator=gen).to(dtype).to(DEV) for n, h in ((lq, heads), (lk, kv), (lk, kv)))
    got = K.attention_prompt(q, k, v, _cu(lq), _cu(lk), dim ** -0.5, causal)
    _check_prompt(got, q, k, v, lq, lk, dim ** -0.5, causal, "runs")


@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_prompt_in_runs_keeps_to_what_a_row_sees(dtype, dim):
    """As test_attention_prompt_keeps_to_what_a_row_sees, blocks cut into runs; growing scores rescale the sums."""
    _say("runs, masked places", dtype, dim)
    gen = _gen(dim)
    lens = [70, 45, 1, 1300]
    n = sum(lens)
    q, k, v = (torch.randn((n, 2, dim), generator=gen) for _ in range(3))
    k[116:] *= torch.linspace(0.01, 6.0, 1300)[:, None, None]
    q, k, v = (x.to(dtype) for x in (q, k, v))
    bad_k, bad_v = k.clone(), v.clone()
    bad_v[30, 0, 3], bad_v[90], bad_k[60], bad_v[800, 1], bad_k[1000, 0] = torch.nan, -torch.inf, torch.nan, torch.inf, torch.nan
    got, want = (K.attention_prompt(q.to(DEV), a.to(DEV), b.to(DEV), _cu(lens), _cu(lens), dim ** -0.5).cpu()
                 for a, b in ((bad_k, bad_v), (k, v)))
    _check_prompt(want, q, k, v, lens, lens, dim ** -0.5, True, "runs")
    same = torch.ones(n, 2, dim, dtype=torch.bool)
    same[30:70, 0, 3] = same[60:70] = same[90:115] = same[800:, 1] = same[1000:, 0] = False
    assert torch.equal(got[same], want[same])
    assert torch.isnan(got[30:70, 0, 3]).all() and torch.isnan(got[60:70]).all()
    assert (got[90:115] == -torch.inf).all() and torch.isnan(got[1000:, 0]).all()
    # Where its P is 0, by rounding, an infinity makes a NaN.
    assert (torch.isnan(got[800:, 1]) | (got[800:, 1] == torch.inf)).all()


@pytest.mark.parametrize("dim,heads,kv,lq,lk", [(64, 2, 1, 130, 5000), (128, 3, 3, 515, 2500), (256, 2, 2, 300, 3400)])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
def test_attention_prompt_long_keys(dim, heads, kv, lq, lk, causal):
    """Few blocks of queries against many keys: a block's keys are taken by many workgroups and joined."""
    _say("long keys", dim, lq, lk, causal)
    gen = _gen(lk)
    q, k, v = (torch.randn((n, h, dim), generator=gen).to(BF16).to(DEV) for n, h in ((lq, heads), (lk, kv), (lk, kv)))
    got = K.attention_prompt(q, k, v, _cu([lq]), _cu([lk]), dim ** -0.5, causal)
    _check_prompt(got, q, k, v, [lq], [lk], dim ** -0.5, causal, "long keys")


# Enough blocks that each has a workgroup of its own.
MANY = [(64, 4, 2, 400), (128, 4, 1, 400), (256, 2, 2, 400)]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("dim,heads,kv,count", MANY)
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
def test_attention_prompt_many_blocks(dtype, dim, heads, kv, count, causal):
    _say("many blocks", dtype, dim, causal)
    gen = _gen(dim + count)
    lq = torch.randint(0, 7, (count,), generator=gen).tolist()
    lk = [n + int(x) for n, x in zip(lq, torch.randint(0, 9, (count,), generator=gen))]
    lq[10], lk[10], lq[200], lk[200], lq[399], lk[399] = 300, 300, 140, 700, 150, 70
    q, k, v = (torch.randn((sum(n), h, dim), generator=gen).to(dtype).to(DEV) for n, h in ((lq, heads), (lk, kv), (lk, kv)))
    spare = torch.ones((200, heads, dim), dtype=dtype, device=DEV)      # rows behind the last sequence
    got = K.attention_prompt(torch.cat((q, spare)), k, v, _cu(lq), _cu(lk), dim ** -0.5, causal)
    assert not got[sum(lq):].any()
    _check_prompt(got, q, k, v, lq, lk, dim ** -0.5, causal, "many blocks")


@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("dim,heads,kv,count", MANY)
def test_attention_prompt_many_blocks_keep_to_what_a_row_sees(dtype, dim, heads, kv, count):
    """As test_attention_prompt_keeps_to_what_a_row_sees, a workgroup a block."""
    _say("many blocks, masked places", dtype, dim)
    gen = _gen(dim)
    lens = [70, 45] + [1] * count
    n = sum(lens)
    q, k, v = (torch.randn((n, h, dim), generator=gen).to(dtype) for h in (heads, kv, kv))
    bad_k, bad_v = k.clone(), v.clone()
    bad_v[30, 0, 3], bad_v[90], bad_k[60], bad_v[200], bad_k[201] = torch.nan, -torch.inf, torch.nan, torch.inf, torch.nan
    got, want = (K.attention_prompt(q.to(DEV), a.to(DEV), b.to(DEV), _cu(lens), _cu(lens), dim ** -0.5).cpu()
                 for a, b in ((bad_k, bad_v), (k, v)))
    assert not torch.isnan(want).any()
    same = torch.ones(n, heads, dim, dtype=torch.bool)
    same[30:70, :heads // kv, 3] = same[60:70] = same[90:115] = same[200:202] = False
    assert torch.equal(got[same], want[same])
    assert torch.isnan(got[30:70, :heads // kv, 3]).all() and torch.isnan(got[60:70]).all()
    assert (got[90:115] == -torch.inf).all() and (got[200] == torch.inf).all() and torch.isnan(got[201]).all()


# ---------------------------------------------------------------------------
# attention_paged
# ---------------------------------------------------------------------------
def _paged_case(lens, size, heads, kv, dim, bits, dtype, gen, extra_blocks=3, magnitude=1.0):
    """(q, noisy cache with the sequences' rows in it, tables, per-sequence keys, values, their parts)."""
    need = [-(-n // size) for n in lens]
    blocks = sum(need) + extra_blocks
    cache = _noisy_cache(blocks, size, kv, dim, bits, dtype, gen)
    order = torch.randperm(blocks, generator=gen).tolist()
    tables = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    slots, at = [], 0
    for b, n in enumerate(lens):
        tables[b, :need[b]] = torch.tensor(order[at:at + need[b]], dtype=torch.int32)
        slots += [order[at + t // size] * size + t % size for t in range(n)]
        at += need[b]
    q = torch.randn((len(lens), heads, dim), generator=gen).to(dtype).to(DEV)
    if slots:
        rows = [(torch.randn((len(slots), kv, dim), generator=gen) * m + o).to(dtype).to(DEV)
                for m, o in ((1.0, torch.randn((kv, dim), generator=gen)), (magnitude, 0.0))]
        table = torch.cat((torch.ones(1, 16), torch.zeros(1, 16)), 1).to(DEV)
        K.rope_append(rows[0], rows[0], rows[1], torch.zeros(len(slots), dtype=torch.int64, device=DEV), table,
                      _i32(slots), *cache)
    return q, cache, tables.to(DEV), slots


def _check_paged(got, q, cache, slots, lens, scale, what):
    kv = (cache.k.shape[2] if cache.k_scales is None else cache.k.shape[1])
    dim, group, at = q.shape[2], q.shape[1] // kv, 0
    coded = cache.k_scales is not None
    now = _numpy(cache) if coded else [t.cpu().double() for t in cache[:2]]
    for b, n in enumerate(lens):
        if n == 0:
            assert torch.equal(got[b].cpu(), torch.zeros_like(got[b].cpu())), (what, b)
            continue
        mine = slots[at:at + n]
        at += n
        if coded:
            rows = [[orc.read_row(now, s, h) for h in range(kv)] for s in mine]
            k, v, high, low = (torch.from_numpy(np.array([[r[i] for r in row] for row in rows])) for i in range(4))
            step = torch.from_numpy(np.array([[np.repeat(now[3][s // cache.k.shape[2], h, :, s % cache.k.shape[2], 0],
                                                         64) for h in range(kv)] for s in mine])).double()
        else:
            size = cache.k.shape[1]
            k, v = (torch.stack([c[s // size, s % size] for s in mine]) for c in now)
            high, low = v.abs(), torch.zeros_like(v)
        out, w, big = orc.attend(q[b:b + 1].cpu().double(), k, v, scale)
        spread = lambda x: torch.einsum("hij,jhd->ihd", w, x.repeat_interleave(group, 1))  # noqa: E731
        absolute = spread(high.abs() + low.abs())
        if coded:
            # Keys: products of codes, whose parts code s and minimum are each larger than the key.
            parts = torch.einsum("ihd,jhd->hij", q[b:b + 1].cpu().double().abs(),
                                 (k.abs() + 32 * step.amax()).repeat_interleave(group, 1)) * scale
            big = parts.amax(-1).T[..., None]
            # Values: 1024 + code in the products, 1024 P taken off again in fp32.
            absolute = absolute + spread(step) * 1040 * (n / 32 + 64) * 2.0 ** -24 / 2.0 ** -11
            half_step = 2.0 ** -11
        else:
            half_step = torch.finfo(q.dtype).eps / 2
        _check(got[b:b + 1], out, absolute, big, q.dtype, dim, half_step, (what, b, n))


PAGED = [
    ([0, 1, 15, 16, 17], 16, 4, 4),
    ([31, 32, 33, 127, 128, 129], 48, 8, 2),
    ([257, 0, 1000], 256, 5, 1),
    ([700], 32, 40, 2),                     # 20 query heads per key-value head: two blocks of columns
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens,size,heads,kv", PAGED, ids=lambda x: str(x).replace(" ", ""))
def test_attention_paged(bits, dtype, dim, lens, size, heads, kv):
    _say("paged", bits, dtype, dim, lens, size, heads, kv)
    q, cache, tables, slots = _paged_case(lens, size, heads, kv, dim, bits, dtype, _gen(dim + sum(lens)))
    got = K.attention_paged(q, cache.k, cache.v, tables, _i32(lens), dim ** -0.5, cache.k_scales, cache.v_scales)
    _check_paged(got, q, cache, slots, lens, dim ** -0.5, "paged")


@pytest.mark.parametrize("bits", [16, 4])
def test_attention_paged_long_and_many(bits):
    """A sequence over many workgroups next to short ones; more sequences than a wave looks through at once."""
    _say("paged long", bits)
    gen = _gen(bits)
    lens = [9000] + torch.randint(0, 60, (140,), generator=gen).tolist()
    q, cache, tables, slots = _paged_case(lens, 16, 4, 2, 64, bits, F16, gen)
    got = K.attention_paged(q, cache.k, cache.v, tables, _i32(lens), 0.125, cache.k_scales, cache.v_scales)
    _check_paged(got, q, cache, slots, lens, 0.125, "long")


@pytest.mark.parametrize("dim,kv", [(64, 16), (128, 8), (256, 8)])
def test_attention_paged_more_work_than_the_chip_holds(dim, kv):
    """16-bit pages, units enough that half of the workgroups take them all."""
    _say("paged much", dim)
    gen = _gen(dim)
    lens = [900, 0, 1, 128, 129] + torch.randint(1, 900, (20,), generator=gen).tolist()
    assert kv * sum(3 + max(1, -(-n // 128)) for n in lens) >= 2 * (1024 if dim == 64 else 512)
    q, cache, tables, slots = _paged_case(lens, 16, 2 * kv, kv, dim, 16, BF16, gen)
    got = K.attention_paged(q, cache.k, cache.v, tables, _i32(lens), dim ** -0.5)
    _check_paged(got, q, cache, slots, lens, dim ** -0.5, "much")


@pytest.mark.parametrize("magnitude", [1e-3, 300.0, 20000.0])
def test_attention_paged_4bit_values_of_every_size(magnitude):
    """Scales for which the probabilities keep their factor of 2^10, and larger ones for which they cannot."""
    _say("paged sizes", magnitude)
    lens = [300, 40]
    q, cache, tables, slots = _paged_case(lens, 16, 4, 2, 128, 4, F16, _gen(4), magnitude=magnitude)
    got = K.attention_paged(q, cache.k, cache.v, tables, _i32(lens), 0.09, cache.k_scales, cache.v_scales)
    _check_paged(got, q, cache, slots, lens, 0.09, "sizes")


@pytest.mark.parametrize("bits", [16, 4])
def test_attention_paged_bad_pages(bits):
    """A page number outside the cache and a length behind the table make that sequence NaN and no other; entries
    behind a sequence's end are not looked at."""
    _say("bad pages", bits)
    lens = [100, 100, 100, 30]
    q, cache, tables, slots = _paged_case(lens, 16, 4, 2, 64, bits, BF16, _gen(6))
    good = K.attention_paged(q, cache.k, cache.v, tables, _i32(lens), 0.125, cache.k_scales, cache.v_scales)
    tables[0, 3], tables[1, 0], tables[3, 3] = cache.k.shape[0], -1, 10 ** 9
    bad = K.attention_paged(q, cache.k, cache.v, tables, _i32([100, 100, 113, 30]), 0.125, cache.k_scales,
                            cache.v_scales)
    assert not torch.isnan(good).any()
    assert torch.isnan(bad[:3]).all()
    assert torch.equal(bad[3], good[3])


def test_attention_paged_far_offsets():
    """Pages whose byte offsets pass 32 bits, in both caches."""
    _say("far offsets")
    blocks = 9000           # 9000 x 256 x 2 x 256 x 2 bytes: 2.4 GB each
    cache = K.KVCache(*(torch.empty((blocks, 256, 2, 256), dtype=BF16, device=DEV) for _ in range(2)))
    n, gen = 300, _gen(2)
    k, v, q = (torch.randn((m, h, 256), generator=gen).to(BF16).to(DEV) for m, h in ((n, 2), (n, 2), (1, 8)))
    slots = [8999 * 256 + t if t < 256 else 8500 * 256 + t - 256 for t in range(n)]
    table = torch.cat((torch.ones(1, 16), torch.zeros(1, 16)), 1).to(DEV)
    K.rope_append(k, k, v, torch.zeros(n, dtype=torch.int64, device=DEV), table, _i32(slots), *cache)
    assert torch.equal(K.kv_gather(*cache[:2], _i32(slots))[0], k)
    got = K.attention_paged(q, cache.k, cache.v, _i32([[8999, 8500]]), _i32([n]), 0.0625)
    out, w, big = orc.attend(q.cpu().double(), k.cpu().double(), v.cpu().double(), 0.0625)
    absolute = torch.einsum("hij,jhd->ihd", w, v.cpu().double().abs().repeat_interleave(4, 1))
    _check(got, out, absolute, big, BF16, 256, 2.0 ** -8, "far")


# ---------------------------------------------------------------------------
# Streams, graphs, registration, the run of them together
# ---------------------------------------------------------------------------
def test_graph_replays_follow_their_inputs():
    """A decode step (append, attention) captured once and replayed with other lengths, slots and rows, eager work in
    between; a second graph captured on the same sizes does not disturb it."""
    _say("graphs")
    gen, heads, kv, dim, size, blocks = _gen(9), 8, 2, 128, 16, 40
    cache = K.new_kv_cache(blocks, size, kv, dim, bits=4, device=DEV)
    twin = K.KVCache(*[t.clone() for t in cache])
    table = K.rope_table(600, 64, device=DEV)
    tables = torch.randperm(blocks, generator=gen)[:36].view(2, 18).to(torch.int32).to(DEV)
    rows = torch.zeros((2, (heads + 2 * kv) * dim), dtype=BF16, device=DEV)
    positions = torch.zeros(2, dtype=torch.int64, device=DEV)
    slots, lens = _i32([-1, -1]), _i32([0, 0])

    def step(cache):
        q, k, v = (x.view(2, -1, dim) for x in rows.split([heads * dim, kv * dim, kv * dim], 1))
        q, k = K.rope_append(q, k, v, positions, table, slots, *cache)
        return K.attention_paged(q, cache.k, cache.v, tables, lens, 0.09, cache.k_scales, cache.v_scales)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(cache))
    for i in range(6):
        rows.copy_(torch.randn(rows.shape, generator=gen).to(BF16))
        n = [i + 1, 20 * i + 1]
        positions.copy_(torch.tensor([x - 1 for x in n]))
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        slots.copy_(torch.stack([tables[b, (x - 1) // size] * size + (x - 1) % size for b, x in enumerate(n)]))
        want = step(twin)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i % 2], want), i
        assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip(cache, twin)), i


@pytest.mark.parametrize("heads,batch", [(4, 3), (8, 250)])
def test_prompt_graph_replays_follow_their_offsets(heads, batch):
    """attention_prompt captured once (equal runs of keys; a workgroup a block) and replayed with other rows and
    offsets, eager calls in between, as it answers eagerly."""
    _say("prompt graph", heads, batch)
    gen, rows, dim = _gen(batch), 1900, 128
    q, k, v = (torch.zeros((rows, h, dim), dtype=BF16, device=DEV) for h in (heads, 2, 2))
    cu = torch.zeros(batch + 1, dtype=torch.int32, device=DEV)
    K.attention_prompt(q, k, v, cu, cu, 0.09)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = K.attention_prompt(q, k, v, cu, cu, 0.09)
    for i in range(5):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=gen).to(BF16))
        cu[1:].copy_(torch.randint(0, rows + 1, (batch,), generator=gen).sort().values.to(torch.int32))
        want = K.attention_prompt(q, k, v, cu, cu, 0.09)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


def test_calls_on_another_stream():
    _say("stream")
    gen = _gen(1)
    q, k, v = (torch.randn((500, h, 128), generator=gen).to(BF16).to(DEV) for h in (8, 2, 2))
    cu = _cu([500])
    want = K.attention_prompt(q, k, v, cu, cu, 0.09)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = K.attention_prompt(q, k, v, cu, cu, 0.09)
    side.synchronize()
    assert torch.equal(got, want)


def test_empty_calls():
    _say("empty")
    none = torch.empty((0, 2, 64), dtype=BF16, device=DEV)
    cache = K.new_kv_cache(1, 16, 2, 64, device=DEV)
    table = K.rope_table(4, 64, device=DEV)
    at, slots = torch.empty(0, dtype=torch.int64, device=DEV), _i32([])
    q, k = K.rope_append(none, none, none, at, table, slots, *cache[:2])
    assert q.shape == k.shape == (0, 2, 64)
    assert K.kv_gather(cache.k, cache.v, slots)[0].shape == (0, 2, 64)
    assert K.attention_prompt(none, none, none, _i32([0]), _i32([0]), 1.0).shape == (0, 2, 64)
    assert K.attention_paged(none, cache.k, cache.v, torch.empty((0, 1), dtype=torch.int32, device=DEV), slots,
                             1.0).shape == (0, 2, 64)
    one = torch.randn((3, 2, 64), device=DEV).to(BF16)
    assert not K.attention_prompt(one, none, none, _i32([0, 3]), _i32([0, 0]), 1.0).any()
    assert not K.attention_prompt(one, one, one, _i32([0]), _i32([0]), 1.0).any()     # rows of no sequence
    got = K.attention_paged(one, cache.k, cache.v, torch.empty((3, 0), dtype=torch.int32, device=DEV),
                            _i32([0, 0, 1]), 1.0)
    assert not got[:2].any() and torch.isnan(got[2]).all()


@pytest.mark.parametrize("bits", [16, 4])
def test_layer_prompt_then_chunk_then_decode(bits):
    """Qwen35Attention on the ops against the same layer in plain torch: prompts, a chunk on the cached prefix, then
    decode steps of a padded batch.  The hidden states are compared in norm: projections and norms round alike, the
    attention's P and 4-bit codes at a rounding's edge do not."""
    _say("layer", bits)
    gen = _gen(bits)
    layers = []
    for backend in ("hip", "torch"):
        layer = PKG.layers.Qwen35Attention(256, 8, 2, 128)
        g = _gen(77)
        for p in layer.parameters():
            p.requires_grad_(False)
            p.copy_(torch.randn(p.shape, generator=g) * (0.05 if p.dim() == 2 else 0.1))
        layer = layer.to(DEV, BF16)
        layer.gemm_backend = backend
        layers.append(layer)
    table, size = K.rope_table(400, 64, device=DEV), 16
    caches = [K.new_kv_cache(60, size, 2, 128, bits=bits, device=DEV) for _ in layers]
    pages = torch.randperm(60, generator=gen)[:56].view(2, 28)
    slot = lambda b, t: int(pages[b, t // size]) * size + t % size  # noqa: E731

    def both(count, positions, slots, **where):
        x = torch.randn((count, 256), generator=gen).to(BF16).to(DEV)
        got, want = (layer(x, torch.tensor(positions, device=DEV), table, cache, _i32(slots), **where).float()
                     for layer, cache in zip(layers, caches))
        return float((got - want).norm() / want.norm())

    lens = [150, 37]
    steps = [both(sum(lens), [t for n in lens for t in range(n)], [slot(b, t) for b, n in enumerate(lens) for t in range(n)],
                  cu_seqlens=_cu(lens))]
    more = [20, 33]
    after = [n + m for n, m in zip(lens, more)]
    steps.append(both(sum(more), [n + t for n, m in zip(lens, more) for t in range(m)],
                      [slot(b, n + t) for b, (n, m) in enumerate(zip(lens, more)) for t in range(m)],
                      cu_seqlens=_cu(more), cu_seqlens_k=_cu(after),
                      context_slots=_i32([slot(b, t) for b, n in enumerate(after) for t in range(n)])))
    tables = torch.cat((pages, torch.full((1, 28), -1))).to(torch.int32).to(DEV)
    for i in range(3):
        now = [n + i for n in after]
        steps.append(both(3, now + [0], [slot(b, n) for b, n in enumerate(now)] + [-1], block_tables=tables,
                          context_lens=_i32([n + 1 for n in now] + [0])))
    _say(steps)
    # Roundings to bf16 (half a step is 2^-8) along the layer: q, k, P, the output, the gate, the product.
    assert max(steps) < 6 * 2.0 ** -8
