"""GPU tests of attention rows in which one key outweighs each of very many
others: what the others add up to has to be kept, though each weight is far
below what a 16-bit float holds next to 1."""
from __future__ import annotations

import math

import pytest
import torch

from conftest import PKG

pytestmark = pytest.mark.gpu

K = PKG.kernels
DEV = torch.device("cuda:0")
BF16, F16 = torch.bfloat16, torch.float16
IDS = {BF16: "bf16", F16: "f16"}


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _case(n, down, dim, dtype, where, rows=1):
    """q, k, v, scale and the output: the key at `where` scores `down` powers of two above the others, its value is 0."""
    q, k = torch.ones((rows, 1, dim)), torch.zeros((n, 1, dim))
    k[where] = 1.0
    v = torch.linspace(0.5, 1.5, dim).expand(n, 1, dim).clone()
    v[where] = 0.0
    q, k, v = (x.to(dtype).to(DEV) for x in (q, k, v))
    scale = down * math.log(2) / dim
    others = (n - 1) * 2.0 ** -down
    out = v[where - 1, 0].double().cpu() * others / (1 + others)
    return q, k, v, scale, out


def _tolerance(out, n, down, dim, dtype, fold):
    """All weights but one are equal, so that each rounding of P weighs in full: half a step, or 2^-25 in float16's
    subnormal range where P is held 2^fold fold; fp32 sums of n weights in parts of at most a tile each, and scores of
    dim products, whose error changes a weight by a factor; one rounding to dtype."""
    half = torch.finfo(dtype).eps / 2
    p = half if dtype == BF16 else max(half, 2.0 ** (down - 25 - fold))
    fp32 = 2.0 ** -23 * (64 + n / 64) + (dim + 16) * 2.0 ** -24 * down + 2.0 ** -20
    least = 0.0 if dtype == BF16 else 2.0 ** -25
    return out * (2 * p + fp32 + half) * (1 + 2.0 ** -6) + least


# Between a float16's half step next to 1 and far below it, at lengths where the others' total still counts.
CASES = [(4097, 14.5), (16385, 18.3), (131073, 22.6), (131073, 25.4), (400001, 27.2)]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,down", CASES)
@pytest.mark.parametrize("where", ["first", "last"])
def test_prompt_keeps_small_weights(dtype, dim, n, down, where):
    print("small weights", dtype, dim, n, down, where, flush=True)
    q, k, v, scale, out = _case(n, down, dim, dtype, 0 if where == "first" else n - 1)
    got = K.attention_prompt(q, k, v, _i32([0, 1]), _i32([0, n]), scale)[0, 0].double().cpu()
    off = (got - out).abs() / _tolerance(out, n, down, dim, dtype, 12)
    print("largest share of the bound", float(off.max()), flush=True)
    assert float(off.max()) <= 1


@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompt_keeps_small_weights_a_block_a_workgroup(dtype, dim):
    """As above in a call of many short sequences, which has nothing to join."""
    print("small weights, many", dtype, dim, flush=True)
    n, down, count = 3000, 20.4, 1600
    q, k, v, scale, out = _case(n, down, dim, dtype, 0, rows=count)
    lens = [n] + [0] * (count - 1)
    cu_k = _i32([0] + [n] * count)
    got = K.attention_prompt(q, k, v, _i32(list(range(count + 1))), cu_k, scale)
    assert sum(lens) == n and not got[1:].any()
    off = (got[0, 0].double().cpu() - out).abs() / _tolerance(out, n, down, dim, dtype, 12)
    print("largest share of the bound", float(off.max()), flush=True)
    assert float(off.max()) <= 1


@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,down", CASES)
def test_paged_keeps_small_weights(dtype, dim, n, down):
    print("small weights, paged", dtype, dim, n, down, flush=True)
    q, k, v, scale, out = _case(n, down, dim, dtype, 0)
    size = 256
    blocks = -(-n // size)
    cache = K.new_kv_cache(blocks, size, 1, dim, dtype=dtype, device=DEV)
    cache.k.view(-1, 1, dim)[:n], cache.v.view(-1, 1, dim)[:n] = k, v
    got = K.attention_paged(q, cache.k, cache.v, torch.arange(blocks, dtype=torch.int32, device=DEV)[None], _i32([n]),
                            scale)[0, 0].double().cpu()
    off = (got - out).abs() / _tolerance(out, n, down, dim, dtype, 10)
    print("largest share of the bound", float(off.max()), flush=True)
    assert float(off.max()) <= 1
