"""GPU tests of attention with scores of any size that 32 bits hold exactly:
their differences decide, however large they are."""
from __future__ import annotations

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


def _case(n, dim, dtype, large, steps, gen):
    """q, k, v, scale and the weights [n].  The score of key j is 2^large + 2^(large - 23) * 8 * d_j, exact in 32 bits at
    every step of the sum (powers of two, in two groups of 64 channels); its scaled differences are `steps` * d_j.
    (2^large itself is a product 2^12 * 2^(large - 12), a power that float16 holds.)"""
    d = torch.randint(0, 4, (n,), generator=gen)
    d[:n // 2] = d[:n // 2].clamp(max=1)      # the maximum grows on the way
    unit = 2.0 ** (large - 20)
    q, k = torch.zeros((1, 2, dim)), torch.zeros((n, 1, dim))
    q[..., 0] = 2.0 ** 12
    k[..., :64] = 2.0 ** (large - 12)         # a group of equal channels: exact in 4 bits too
    q[..., 64], k[..., 64:128] = 2.0 ** 3, (d * unit / 8)[:, None, None].float()
    v = torch.randn((n, 1, dim), generator=gen)
    weights = torch.softmax(d.double() * steps, 0)
    return *(x.to(dtype).to(DEV) for x in (q, k, v)), steps / unit, weights


def _tolerance(weights, v, out, dtype, coded):
    """Scores are exact, so are their differences but for the factor: a rounding of each weight (and of its product with a
    4-bit scale, and of the middle of a group), their total, 2^-20 for exponentials and fp32 sums, one of the output."""
    half = 2.0 ** -11 if coded else torch.finfo(dtype).eps / 2
    size = torch.einsum("j,jd->d", weights, v.abs()) if not coded else v.abs().amax(0) * 2
    off = (3 if coded else 1) * half * size + (half + 2.0 ** -20) * out.abs() + 2.0 ** -20 * size
    return off * (1 + 2.0 ** -6) + torch.finfo(dtype).eps / 2 * (out.abs() + off)


# Powers of two of the scores in front of the scale; scaled, a score is 2^20 times `steps`.
LARGE = [4, 12, 20, 24, 26]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("large", LARGE)
@pytest.mark.parametrize("steps", [0.25, 3.0, 600.0])
def test_prompt(dtype, dim, large, steps):
    print("large scores, prompt", dtype, dim, large, steps, flush=True)
    n = 1500
    q, k, v, scale, weights = _case(n, dim, dtype, large, steps, torch.Generator().manual_seed(large))
    for count in (1, 1600):      # blocks cut into runs; a workgroup a block
        cu_q, cu_k = _i32(list(range(count + 1))), _i32([0] + [n] * count)
        got = K.attention_prompt(q.expand(count, -1, -1).contiguous(), k, v, cu_q, cu_k, scale)[0].double().cpu()
        rows = v[:, 0].double().cpu()
        out = torch.einsum("j,jd->d", weights, rows)
        assert ((got - out).abs() <= _tolerance(weights, rows, out, dtype, False)).all(), (count, got[0, :4], out[:4])


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("large", LARGE)
@pytest.mark.parametrize("steps", [0.25, 3.0, 600.0])
def test_paged(bits, dtype, dim, large, steps):
    print("large scores, paged", bits, dtype, dim, large, steps, flush=True)
    n, size = 1500, 64
    q, k, v, scale, weights = _case(n, dim, dtype, large, steps, torch.Generator().manual_seed(large))
    blocks = -(-n // size)
    cache = K.new_kv_cache(blocks, size, 1, dim, bits=bits, dtype=dtype, device=DEV)
    still = torch.cat((torch.ones(1, 16), torch.zeros(1, 16)), 1).to(DEV)
    slots = torch.arange(n, dtype=torch.int32, device=DEV)
    K.rope_append(k, k, v, torch.zeros(n, dtype=torch.int64, device=DEV), still, slots, *cache)
    rows = v[:, 0].double().cpu()
    if bits == 4:
        keys, values = K.gather_kv(cache, slots, torch.float32, backend="torch")
        assert torch.equal(keys, k.float())
        rows = values[:, 0].double().cpu()
    got = K.attention_paged(q, cache.k, cache.v, torch.arange(blocks, dtype=torch.int32, device=DEV)[None], _i32([n]),
                            scale, cache.k_scales, cache.v_scales)[0].double().cpu()
    out = torch.einsum("j,jd->d", weights, rows)
    assert ((got - out).abs() <= _tolerance(weights, rows, out, dtype, bits == 4)).all(), (got[0, :4], out[:4])
