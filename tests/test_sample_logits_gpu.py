"""sample_logits on the GPU against the oracle: tokens are equal, log-probabilities within their rounding."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import int8_oracle as orc

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF = float("inf")


@pytest.fixture(scope="module")
def ops(pkg):
    return pkg.kernels


def rows_of(m, vocab, seed, spread=2.0, peak=10.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, vocab, generator=g) * spread
    if peak:
        at = torch.randint(0, vocab, (m, 12), generator=g)
        x.scatter_add_(1, at, peak * torch.rand(m, 12, generator=g))
    return x, 0.5 + torch.rand(m, generator=g), torch.rand(m, generator=g)


def check(ops, logits, t, u, top_k=None, top_p=None, min_p=None, view=None):
    def param(x, dtype):
        if x is None:
            return None
        x = torch.as_tensor(x, dtype=dtype)
        return x.expand(logits.shape[:-1]).contiguous()
    t, u = param(t, F32), param(u, F32)
    k, p, q = param(top_k, torch.int32), param(top_p, F32), param(min_p, F32)
    dev = [None if x is None else x.to(DEV) for x in (t, u, k, p, q)]
    source = logits.to(DEV) if view is None else view
    tokens, logprobs = ops.sample_logits(source, *dev)
    assert tokens.dtype == torch.int64 and tokens.shape == logits.shape[:-1] and logprobs.dtype == F32
    again = ops.sample_logits(source, *dev)
    assert torch.equal(tokens, again[0]) and torch.equal(logprobs.nan_to_num(7), again[1].nan_to_num(7))
    x = logits.double().numpy().reshape(-1, logits.shape[-1])
    got = tokens.cpu().numpy().reshape(-1), logprobs.cpu().double().numpy().reshape(-1)
    for i in range(x.shape[0]):
        given = [None if a is None else float(a.reshape(-1)[i]) for a in (t, u, k, p, q)]
        token, share = orc.sample(x[i], *given)
        assert got[0][i] == token, (i, given, got[0][i], token, share)
        # A logarithm in 64 bits of weights good to 2^-40, rounded once.
        if np.isnan(share):
            assert np.isnan(got[1][i])
        else:
            assert abs(got[1][i] - share) <= abs(share) * 2.0 ** -24 + 1e-11, (i, given, got[1][i], share)
    return tokens


FILTERS = [dict(), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05), dict(top_k=200, top_p=0.8),
           dict(top_k=30, min_p=0.02), dict(top_p=0.95, min_p=0.01), dict(top_k=500, top_p=0.97, min_p=0.001)]


@pytest.mark.parametrize("filters", FILTERS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 8191, 8193, 32000])
def test_sample_logits(ops, vocab, dtype, filters):
    x, t, u = rows_of(9, vocab, vocab)
    check(ops, x.to(dtype), t, u, **filters)


@pytest.mark.parametrize("filters", FILTERS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sample_logits_flat_rows(ops, dtype, filters):
    """No token stands out: the borders fall among tens of thousands, many of them equal in 16 bits."""
    x, t, u = rows_of(6, 50021, 3, spread=1.0, peak=0.0)
    check(ops, x.to(dtype), t, u, **filters)


@pytest.mark.parametrize("vocab", [151936, 262144])
def test_sample_logits_large_vocabulary(ops, vocab):
    x, t, u = rows_of(5, vocab, 11)
    k = torch.tensor([0, 1, 50, 5000, vocab], dtype=torch.int32)
    check(ops, x.to(BF16), t, u, top_k=k, top_p=torch.tensor([0.9, 0.5, 0.99, 0.999, 1.0]))
    check(ops, x, t, u, top_p=torch.tensor([0.9, 0.5, 0.99, 0.999, 1.0]), min_p=0.01)


def test_sample_logits_many_rows(ops):
    x, t, u = rows_of(700, 3000, 12)
    check(ops, x, t, u, top_k=torch.randint(0, 300, (700,), generator=torch.Generator().manual_seed(1), dtype=torch.int32),
          top_p=torch.rand(700, generator=torch.Generator().manual_seed(2)))


@pytest.mark.parametrize("vocab", [40, 6000, 30000])
def test_sample_logits_equal_logits(ops, vocab):
    """Every token equal: each filter counts, the lowest indices first."""
    x = torch.full((6, vocab), 1.5)
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.9, 0.999])
    check(ops, x, 1.0, u)
    check(ops, x, 1.0, u, top_k=vocab // 3)
    check(ops, x, 1.0, u, top_p=0.5)
    check(ops, x, 0.7, u, top_k=vocab // 2, top_p=0.25, min_p=1.0)
    # Two values, thousands of holders each.
    x[:, ::2] = 1.0
    check(ops, x, 0.5, u, top_k=vocab // 2 + 5)
    check(ops, x, 0.5, u, top_p=0.9)
    check(ops, x, 0.5, u, top_k=vocab // 2 + 5, top_p=0.95)


def test_sample_logits_bins_with_many_members(ops):
    """A high temperature puts thousands of different logits into one bin."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(4, 60000, generator=g)
    u = torch.rand(4, generator=g)
    for filters in (dict(top_k=20000), dict(top_p=0.37), dict(top_k=31000, top_p=0.9), dict(min_p=0.999)):
        check(ops, x, torch.tensor([50.0, 1000.0, 3e7, INF]), u, **filters)


def test_sample_logits_temperatures(ops):
    x, _, u = rows_of(8, 5000, 5)
    x[2, 17] = x[2, 4000] = x[2].max() + 1
    t = torch.tensor([0.0, 1e-10, -1.0, float("nan"), 1e-9, 1e-3, 0.05, 1e30])
    tokens = check(ops, x, t, u, top_p=0.9)
    assert tokens[2] == 17


def test_sample_logits_numbers_at_the_ends(ops):
    x, t, _ = rows_of(8, 3000, 6)
    u = torch.tensor([0.0, -1.0, float("nan"), 1.0, 2.0, 1 - 2.0 ** -24, 2.0 ** -24, INF])
    for filters in FILTERS:
        check(ops, x, t, u, **filters)


def test_sample_logits_parameters_at_the_ends(ops):
    x, t, u = rows_of(8, 3000, 7)
    nan = float("nan")
    check(ops, x, t, u, top_k=torch.tensor([0, -5, 1, 2, 2999, 3000, 3001, 2 ** 31 - 1], dtype=torch.int32))
    check(ops, x, t, u, top_p=torch.tensor([0.0, -1.0, 1.0, 2.0, nan, 1e-30, 1 - 2.0 ** -24, INF]))
    check(ops, x, t, u, min_p=torch.tensor([0.0, -1.0, 1.0, 2.0, nan, 1e-30, 1e-45, INF]))


def test_sample_logits_masked_rows(ops):
    """-inf, the type's lowest value, infinities and NaN in places, and rows of nothing else."""
    for dtype in (F32, F16, BF16):
        x, t, u = rows_of(12, 2500, 8)
        x = x.to(dtype)
        low = torch.finfo(dtype).min
        x[0, 100:] = -INF
        x[1, :2400] = low
        x[2] = -INF
        x[3] = low
        x[4] = -INF
        x[4, 77] = 3.0
        x[5, 300], x[5, 200] = INF, INF
        x[6] = INF
        x[7, 900], x[7, 800] = float("nan"), float("nan")
        x[8] = float("nan")
        x[9, ::3] = -INF
        x[10, 5] = -0.0
        x[11] = 0.0
        x[11, ::2] = -0.0
        for filters in FILTERS:
            check(ops, x, t, u, **filters)
        tokens = check(ops, x, torch.zeros(12), u)
        assert tokens[7] == 800 and tokens[5] == 200 and tokens[11] == 0


def test_sample_logits_large_values(ops):
    """Logits far from 0 and temperatures far from 1: l / T has no fraction left in 64 bits, or all of it matters."""
    g = torch.Generator().manual_seed(9)
    x = torch.randn(6, 4000, generator=g)
    x[0] = x[0] * 1e37
    x[1] += 1e4
    x[2] += 3e6
    x[3] *= 1e-30
    x[4] = x[4].abs() * 1e30
    t = torch.tensor([1e-9, 0.9, 0.5, 2e-30, 1e25, 1e-5])
    u = torch.rand(6, generator=g)
    for filters in (dict(), dict(top_k=60), dict(top_p=0.8), dict(min_p=0.1)):
        check(ops, x, t, u, **filters)


def test_sample_logits_views_and_dims(ops):
    g = torch.Generator().manual_seed(10)
    wide = torch.randn(10, 3001, generator=g) * 3
    for dtype in (F32, BF16):
        dev = wide.to(dtype).to(DEV)
        u = torch.rand(10, generator=g)
        check(ops, wide.to(dtype)[:, 3:2900], 0.8, u, top_p=0.9, view=dev[:, 3:2900])
        check(ops, wide.to(dtype)[::2, 1:], 0.8, u[:5], top_k=20, view=dev[::2, 1:])
        check(ops, wide.to(dtype)[:1, 5:], 0.8, u[:1], view=dev[:1, 5:])
    deep = torch.randn(2, 3, 500, generator=g)
    check(ops, deep, 1.0, torch.rand(2, 3, generator=g), top_k=10)
    check(ops, deep[0, 0], 1.0, torch.tensor(0.4), top_k=10)
    tokens, logprobs = ops.sample_logits(*(torch.empty(s, device=DEV) for s in ((0, 10), (0,), (0,))))
    assert tokens.shape == (0,) and logprobs.shape == (0,)


def test_sample_logits_follows_the_distribution(ops):
    """Evenly spread numbers give every kept token its share, to one number."""
    n = 4096
    x = torch.randn(50, generator=torch.Generator().manual_seed(13)) * 2
    u = (torch.arange(n) + 0.5) / n
    tokens, _ = ops.sample_logits(x.expand(n, 50).contiguous().to(DEV), torch.full((n,), 0.9, device=DEV), u.to(DEV))
    share = torch.bincount(tokens.cpu(), minlength=50).double() / n
    assert (share - torch.softmax(x.double() / torch.tensor(0.9).double(), 0)).abs().max() <= 1.0 / n + 1e-12


def test_sample_logits_in_a_graph_and_on_a_side_stream(ops):
    x, t, u = (a.to(DEV) for a in rows_of(20, 20000, 14))
    k = torch.full((20,), 50, dtype=torch.int32, device=DEV)
    p = torch.full((20,), 0.9, device=DEV)
    eager = ops.sample_logits(x, t, u, k, p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.sample_logits(x, t, u, k, p)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(eager[0], other[0]) and torch.equal(eager[1], other[1])
    graph = torch.cuda.CUDAGraph()
    static = [a.clone() for a in (x, t, u, k, p)]
    with torch.cuda.graph(graph):
        out = ops.sample_logits(*static)
    for seed in range(4):
        new = [a.to(DEV) for a in rows_of(20, 20000, 20 + seed)]
        k = torch.full((20,), 20 + seed, dtype=torch.int32, device=DEV)
        for dst, src in zip(static, (*new, k, p)):
            dst.copy_(src)
        graph.replay()
        want = ops.sample_logits(*new, k, p)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.parametrize("filters", [dict(), dict(top_p=0.97), dict(min_p=1e-4), dict(top_k=9000, top_p=0.99),
                                     dict(top_k=40, top_p=0.9)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sample_logits_slices_of_two_tiles(ops, dtype, filters):
    """Rows enough that each workgroup takes several slices one after the other; tails of a slice of one to 8 logits."""
    for m, vocab in ((150, 60000), (260, 32769 + 7)):
        x, t, u = rows_of(m, vocab, m)
        x[3, -1] = x[3].max() + 30      # alone in a tail
        x[5] = float("nan")
        x[7, ::2] = -INF
        check(ops, x.to(dtype), t, u, **filters)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sample_logits_longest_rows(ops, dtype):
    """Slices of four tiles: rows that two tiles a slice would cut into more than are joined."""
    vocab = 256 * 16384 + 8193
    x, t, u = rows_of(2, vocab, 21)
    x[1, vocab - 2] = x[1].max() + 3
    check(ops, x.to(dtype), t, u, top_k=torch.tensor([60, 100000], dtype=torch.int32), top_p=0.9)
    check(ops, x.to(dtype), t, u, min_p=1e-3)
    check(ops, x.to(dtype), t, u)


@pytest.mark.parametrize("filters", [dict(), dict(top_k=5), dict(top_p=0.9), dict(min_p=0.1), dict(top_k=3000, top_p=0.5)])
@pytest.mark.parametrize("vocab", [1000, 40000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sample_logits_tokens_are_in_the_vocabulary(ops, dtype, vocab, filters):
    """Whatever the temperature and the size of the logits, the token is one of the row's, and its logprob a number: rows of
    one slice and of several, the largest logit in the last of them."""
    g = torch.Generator().manual_seed(vocab)
    t = torch.cat([10.0 ** (-10.5 + 5 * torch.rand(32, generator=g)), torch.tensor([1e-9, 1e-8, 1.5e-8, 3e-9]).repeat(8)])
    x = torch.randn(64, vocab, generator=g)
    x[torch.arange(64), vocab - 1 - torch.randint(0, 900, (64,), generator=g)] = 5 + 25 * torch.rand(64, generator=g)
    x[::4] *= 10.0 ** torch.linspace(0, 37, 16)[:, None]
    given = [torch.full((64,), v, dtype=torch.int32 if k == "top_k" else F32, device=DEV) if v else None
             for k, v in ((k, filters.get(k)) for k in ("top_k", "top_p", "min_p"))]
    tokens, logprobs = ops.sample_logits(x.to(dtype).to(DEV), t.to(DEV), torch.rand(64, generator=g).to(DEV), *given)
    assert bool(((tokens >= 0) & (tokens < vocab)).all())
    assert bool((logprobs <= 0).all())


@pytest.mark.parametrize("filters", [dict(), dict(top_k=7), dict(top_p=0.9), dict(min_p=0.2)])
@pytest.mark.parametrize("vocab", [1000, 40000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sample_logits_small_temperatures(ops, dtype, vocab, filters):
    """Temperatures down to the greedy ones and logits of any size, with l / T up to 1e47: equal, near and far logits at the
    top, in a row's last slice."""
    g = torch.Generator().manual_seed(vocab + 1)
    t = torch.tensor([1.01e-10, 1e-9, 1e-9, 3e-9, 1e-8, 1.5e-8, 3e-8, 1e-6, 0.9, 40.0] * 3)
    top = torch.cat([5 + 25 * torch.rand(10, generator=g), 10.0 ** torch.linspace(-9, 0, 10), 10.0 ** torch.linspace(9, 37, 10)])
    x = torch.randn(30, vocab, generator=g) * top[:, None] / 10
    at = vocab - 1 - torch.randint(0, 900, (30, 6), generator=g)
    # Some at the top within a few weights of each other, some equal.
    x.scatter_(1, at, top[:, None] - t[:, None] * torch.tensor([0.0, 0.0, 0.3, 1.0, 2.5, 7.0]))
    check(ops, x.to(dtype), t, torch.rand(30, generator=g), **filters)


# Half of this row's weight lies in its first six tokens, to the last bit: the running sum at the bin of the sixth is a
# little below half, at the empty bins behind it, summed in another order, a little above.
HALF = """0x0.0p+0 -0x1.b15cea0000000p-6 -0x1.a7d9e60000000p-4 -0x1.8a2a920000000p-3 -0x1.be3d9c0000000p-3
-0x1.2ecf300000000p-2 -0x1.5480720000000p+0 -0x1.1e13040000000p+1 -0x1.506a400000000p+0 -0x1.ffabb40000000p-1
-0x1.0427820000000p+1 -0x1.8ffe680000000p+0 -0x1.1c52c20000000p+1 -0x1.2975820000000p+0 -0x1.5204e40000000p+0
-0x1.1c8cac0000000p+1 -0x1.ac29a20000000p+0 -0x1.abd5760000000p+0 -0x1.29c9020000000p+0 -0x1.7e316a0000000p-1
-0x1.3ca3e80000000p+1 -0x1.c2d1c20000000p-1 -0x1.2764000000000p+1 -0x1.692b340000000p+0 -0x1.40ec7e0000000p+1
-0x1.785a100000000p+0 -0x1.3d6a2c0000000p+1 -0x1.c3caa00000000p+0 -0x1.2baea20000000p+0 -0x1.0e7b240000000p+1
-0x1.2f0a620000000p+1 -0x1.3a3ae40000000p+2 -0x1.27b4b20000000p+3 -0x1.9727b80000000p+3 -0x1.1bac220000000p+4
-0x1.7f12a60000000p+4"""


@pytest.mark.parametrize("vocab", [36, 36 + 20000])
def test_sample_logits_border_behind_an_empty_bin(ops, vocab):
    """A top-p whose weight falls between two running sums of the same tokens: one token more or less, no other set."""
    x = torch.full((1, vocab), -INF)
    x[0, :36] = torch.tensor([float.fromhex(v) for v in HALF.split()])
    order = torch.sort(x[0, :36].double(), descending=True).values.exp()
    one = torch.ones(1, device=DEV)
    token, logprob = ops.sample_logits(x.to(DEV), one, 0 * one, None, 0.5 * one)
    assert token.item() == 0
    wanted = [-order[:n].sum().log().item() for n in (6, 7)]
    assert any(abs(logprob.item() - w) <= abs(w) * 2.0 ** -24 + 1e-11 for w in wanted), (logprob.item(), wanted)


@pytest.mark.parametrize("vocab", [300, 40000])
def test_sample_logits_infinite_temperature(ops, vocab):
    """Every finite logit weighs 1, so each min-p up to 1 keeps them all; infinities as at any temperature."""
    x, _, u = rows_of(6, vocab, 31)
    x[1, ::2] = -INF
    x[2] = -INF
    x[3, 5], x[3, vocab - 9] = INF, INF
    x[4] = 2.0
    for filters in (dict(), dict(min_p=1.0), dict(min_p=0.5), dict(min_p=1.0, top_k=vocab // 2), dict(min_p=1.0, top_p=0.3),
                    dict(min_p=2.0), dict(min_p=1.0 + 2.0 ** -23)):
        check(ops, x, INF, u, **filters)


@pytest.mark.parametrize("filters", [dict(), dict(top_k=30), dict(top_p=1 - 2.0 ** -24)])
@pytest.mark.parametrize("vocab", [50, 30000])
def test_sample_logits_first_token_of_small_weight(ops, vocab, filters):
    """u = 0 takes the first kept token, whatever its weight is beside its neighbours'."""
    x = torch.full((10, vocab), -INF)
    for i, down in enumerate((1.0, 20.0, 36.0, 36.8, 37.0, 38.0, 40.0, 41.0, 42.0, 43.0)):
        at = i * (vocab // 11)
        x[i, at], x[i, at + 1], x[i, at + 2] = 5.0 - down, 5.0, 5.0 - down
    for u in (0.0, -1.0, float("nan"), 2.0 ** -24):
        check(ops, x, 1.0, torch.tensor(u), **filters)


@pytest.mark.parametrize("backend", ["hip", "torch"])
@pytest.mark.parametrize("filters", [dict(), dict(top_k=900), dict(top_p=0.999)])
@pytest.mark.parametrize("m,vocab", [(600, 1500), (20, 40000)])
def test_sample_logits_last_token(ops, m, vocab, filters, backend):
    """u of 1 or more takes the last kept token: no running sum passes the total by its last bit."""
    # Weights down to 2^-60, so that many sums are the total but for its last bit.
    g = torch.Generator().manual_seed(41)
    t = 0.5 + torch.rand(m, generator=g)
    x = -41.5 * t[:, None] * torch.rand(m, vocab, generator=g)
    k, p = filters.get("top_k"), filters.get("top_p")
    given = [None if v is None else torch.full((m,), v, dtype=d, device=DEV) for v, d in ((k, torch.int32), (p, F32))]
    for u in (1.0, 1.5, INF):
        tokens, _ = ops.sample_rows(x.to(DEV), t.to(DEV), torch.full((m,), u, device=DEV), *given, backend=backend)
        for i in range(m):
            assert tokens[i] == orc.sample(x[i].double().numpy(), float(t[i]), u, k, p)[0], (i, u)
