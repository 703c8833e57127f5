"""The plain torch backend keeps the contracts of the ops: what pages, lengths,
masks and infinities give is the same on either backend (on the GPU, both)."""
from __future__ import annotations

import pytest
import torch

from conftest import PKG

K = PKG.kernels
BF16, F16 = torch.bfloat16, torch.float16
BACKENDS = [pytest.param(("cpu", "torch"), id="torch"),
            pytest.param(("cuda:0", "torch"), id="torch-gpu", marks=pytest.mark.gpu),
            pytest.param(("cuda:0", "hip"), id="hip", marks=pytest.mark.gpu)]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _filled(bits, device, gen, blocks=6, size=16, heads=2, dim=64):
    """A cache whose every slot holds a row of random keys and values."""
    cache = K.new_kv_cache(blocks, size, heads, dim, bits=bits, device=device)
    k, v = (torch.randn((blocks * size, heads, dim), generator=gen).to(BF16).to(device) for _ in range(2))
    table = torch.cat((torch.ones(1, 16), torch.zeros(1, 16)), 1).to(device)
    K.rope_append_kv(k, k, v, torch.zeros(blocks * size, dtype=torch.int64, device=device), table,
                     torch.arange(blocks * size, dtype=torch.int32, device=device), cache, backend="torch")
    return cache


@pytest.mark.parametrize("where", BACKENDS)
@pytest.mark.parametrize("bits", [16, 4])
def test_paged_bad_pages_and_lengths(where, bits):
    """A page outside the cache or a length behind the table makes that sequence NaN and no other, whatever the entries
    behind a sequence's end hold; no token gives 0, a negative length too."""
    device, backend = where
    print("bad pages", device, backend, bits, flush=True)
    gen = _gen(bits)
    cache = _filled(bits, device, gen)
    q = torch.randn((8, 4, 64), generator=gen).to(BF16).to(device)
    good = [[0, 1, 2], [3, 4, 5], [5, 0, 3], [1, 2, 4], [4, 3, 2], [2, 1, 0], [0, 2, 4], [1, 3, 5]]
    lens = [33, 48, 17, 40, 16, 48, 5, 30]
    want = K.paged_attention(q, cache, _i32(good, device), _i32(lens, device), 0.125, backend=backend)
    bad = [row[:] for row in good]
    bad[0][2], bad[1][0], bad[2][1] = -1, 6, 2 ** 31 - 1      # inside the length
    bad[4][1], bad[4][2], bad[6][1] = -7, 6, 10 ** 9          # behind it
    lens[3], lens[5], lens[7] = 49, 0, -3
    got = K.paged_attention(q, cache, _i32(bad, device), _i32(lens, device), 0.125, backend=backend)
    assert not torch.isnan(want).any()
    assert torch.isnan(got[:4]).all()
    assert torch.equal(got[[4, 6]], want[[4, 6]])
    assert not got[[5, 7]].any()


@pytest.mark.parametrize("where", BACKENDS)
def test_paged_empty_table(where):
    device, backend = where
    print("empty table", device, backend, flush=True)
    cache = _filled(16, device, _gen(1))
    q = torch.ones((3, 2, 64), dtype=BF16, device=device)
    table = torch.empty((3, 0), dtype=torch.int32, device=device)
    got = K.paged_attention(q, cache, table, _i32([0, 1, -2 ** 31], device), 0.125, backend=backend)
    assert torch.isnan(got[1]).all() and not got[[0, 2]].any()


@pytest.mark.parametrize("where", BACKENDS)
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_keeps_to_what_a_row_sees(where, causal):
    """NaN and infinities in keys and values that a row does not see change nothing in it."""
    device, backend = where
    print("masked places", device, backend, causal, flush=True)
    gen = _gen(7)
    lens, spare = [70, 45, 1], 20
    n = sum(lens)
    q, k, v = (torch.randn((n + spare, 2, 64), generator=gen).to(BF16) for _ in range(3))
    bad_k, bad_v = k.clone(), v.clone()
    bad_v[30, 0, 3], bad_v[33, 1, 5], bad_v[90] = torch.nan, torch.inf, -torch.inf
    bad_k[60], bad_k[n:], bad_v[n:] = torch.nan, torch.nan, torch.inf
    cu = _i32([0, 70, 115, 116], device)
    want, got = (K.prompt_attention(*(x.to(device) for x in (q, *kv)), cu, cu, 0.125, causal, backend=backend).cpu()
                 for kv in ((k, v), (bad_k, bad_v)))
    first = lambda i, a: i if causal else a      # noqa: E731
    same = torch.ones(n + spare, 2, 64, dtype=torch.bool)
    same[first(30, 0):70, 0, 3] = same[first(33, 0):70, 1, 5] = False
    same[first(60, 0):70] = same[first(90, 70):115] = False
    assert not torch.isnan(want).any() and not want[n:].any()
    assert torch.equal(got[same], want[same])
    assert torch.isnan(got[first(30, 0):70, 0, 3]).all() and torch.isnan(got[first(60, 0):70]).all()
    assert (got[first(90, 70):115] == -torch.inf).all()
    if causal:
        assert (got[33:60, 1, 5] == torch.inf).all()


@pytest.mark.parametrize("where", BACKENDS)
def test_scores_that_are_not_finite(where):
    """A score of -infinity drops its key; rows whose every score is -infinity, or one with +infinity, are NaN; a row
    with no key to see is 0."""
    device, backend = where
    print("infinite scores", device, backend, flush=True)
    gen = _gen(5)
    q, k, v = (torch.randn((40, 1, 64), generator=gen).to(BF16) for _ in range(3))
    q[:, 0, 0], k[:, 0, 0] = 1.0, 0.0
    k[3, 0, 0], k[0, 0, 0], k[35, 0, 0] = -torch.inf, -torch.inf, torch.inf
    cu = _i32([0, 40], device)
    got = K.prompt_attention(*(x.to(device) for x in (q, k, v)), cu, cu, 0.125, backend=backend).cpu()
    assert torch.isnan(got[0]).all() and torch.isnan(got[35:]).all() and not torch.isnan(got[1:35]).any()
    # More queries than keys: the first three rows see none, the fourth one of -infinity only.
    cu_k = _i32([0, 37], device)
    got = K.prompt_attention(*(x.to(device) for x in (q, k[:37], v[:37])), cu, cu_k, 0.125, backend=backend).cpu()
    assert not got[:3].any() and torch.isnan(got[3]).all() and not torch.isnan(got[4:38]).any()
    # The same over pages.
    cache = K.new_kv_cache(4, 16, 1, 64, device=device)
    cache.k.view(-1, 1, 64)[:40], cache.v.view(-1, 1, 64)[:40] = k.to(device), v.to(device)
    table, lens = _i32([[0, 1, 2, 3]] * 3, device), _i32([1, 35, 36], device)
    got = K.paged_attention(q[:3].to(device), cache, table, lens, 0.125, backend=backend).cpu()
    assert torch.isnan(got[0]).all() and not torch.isnan(got[1]).any() and torch.isnan(got[2]).all()
