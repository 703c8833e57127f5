"""quantize_rows, add_rmsnorm_quantize, gemm_int8 and gemm_int8_silu_mul on the GPU against the oracle in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import int8_oracle as orc

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24      # half a step of float32, relative


@pytest.fixture(scope="module")
def ops(pkg):
    return pkg.kernels


def gen(seed):
    return torch.Generator().manual_seed(seed)


def np64(t):
    return t.detach().double().cpu().numpy()


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half of the smallest step there is."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


# ---------------------------------------------------------------------------
# Rows in 8 bits: codes and scales are exact.
# ---------------------------------------------------------------------------
def check_rows(x, codes, scales):
    want, scale, _ = orc.quantize_rows(np64(x).reshape(-1, x.shape[-1]))
    np.testing.assert_array_equal(scales.cpu().numpy().reshape(-1), scale)
    np.testing.assert_array_equal(codes.cpu().numpy().reshape(want.shape), want)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m,k", [(1, 1), (3, 7), (33, 15), (5, 16), (17, 128), (9, 129), (2, 511), (6, 513), (8, 1024),
                                 (3, 1500), (4, 2049), (2, 4096), (3, 5000), (2, 8193), (2, 16384), (2, 16387),
                                 (1, 40001)])
def test_quantize_rows(ops, dtype, m, k):
    x = (torch.randn(m, k, generator=gen(m * 100003 + k)) * 3).to(dtype)
    x[0, -1] = 6.5      # halves of the largest value lie next to a border of two codes
    x[0, 0] = 13.0
    codes, scales = ops.quantize_rows(x.to(DEV))
    assert codes.shape == x.shape and codes.dtype == torch.int8 and scales.shape == (m,)
    check_rows(x, codes, scales)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_quantize_rows_every_half(ops, dtype):
    """Rows whose quotients are halves, or as near to them as the type allows."""
    rows = []
    for top in (127.0, 254.0, 63.5, 1.0, 3.0, 100.0, 0.0078125):
        base = torch.arange(-254, 255, dtype=torch.float64) / 254 * top
        near = base.to(dtype)
        rows.append(near)
        rows.append(torch.nextafter(near.float(), torch.tensor(float("inf"))).to(dtype))
        rows.append(torch.nextafter(near.float(), torch.tensor(-float("inf"))).to(dtype))
    x = torch.stack(rows)
    codes, scales = ops.quantize_rows(x.to(DEV))
    check_rows(x, codes, scales)


def test_quantize_rows_extremes(ops):
    """Zeros, denormal scales, the largest values, NaN and infinities."""
    k = 40
    x = torch.zeros(12, k)
    x[1, 3] = 1e-45
    x[2] = torch.arange(k) * 1.4e-45
    x[3] = torch.linspace(-1e-38, 1e-38, k)
    x[4] = torch.linspace(-3.4e38, 3.4e38, k)
    x[5] = torch.linspace(-1e-30, 2e-30, k)
    x[6, 5] = float("nan")
    x[7, 6] = float("inf")
    x[8, 7] = -float("inf")
    x[9] = torch.linspace(-1, 1, k) * 2.0 ** -64 * 127
    x[10] = torch.linspace(-1, 1, k) * 2.0 ** -60
    x[11, 0] = -0.0
    codes, scales = ops.quantize_rows(x.to(DEV))
    check_rows(x, codes, scales)
    assert bool((codes[6:9] == 0).all()) and bool(scales[6:9].isnan().all())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize_rows_views_and_dims(ops, dtype):
    wide = torch.randn(37, 301, generator=gen(5)).to(dtype).to(DEV)
    for view in (wide[:, 3:260], wide[::2, 1:], wide[:1, 7:], wide[:, :1]):
        codes, scales = ops.quantize_rows(view)
        check_rows(view, codes, scales)
    deep = torch.randn(3, 5, 48, generator=gen(6)).to(dtype).to(DEV)
    codes, scales = ops.quantize_rows(deep)
    assert codes.shape == (3, 5, 48) and scales.shape == (3, 5)
    check_rows(deep, codes, scales)
    flat = torch.randn(48, generator=gen(7)).to(dtype).to(DEV)
    codes, scales = ops.quantize_rows(flat)
    assert codes.shape == (48,) and scales.shape == ()
    check_rows(flat, codes, scales)
    codes, scales = ops.quantize_rows(torch.empty(0, 16, dtype=dtype, device=DEV))
    assert codes.shape == (0, 16) and scales.shape == (0,)


# ---------------------------------------------------------------------------
# Behind the residual add and the norm.
# ---------------------------------------------------------------------------
def check_norm(h, r, w, eps, codes, scales, residual):
    y, s = orc.add_rmsnorm(np64(h), np64(r), np64(w), eps)
    want, scale, quotient = orc.quantize_rows(y)
    k = h.shape[1]
    # s, 1 + w and their product round once each, so a quotient of two such
    # values is off by 6 half steps and its own rounding, at most 127 * 8 U.
    off = 127 * 8 * U
    diff = np.abs(codes.cpu().numpy().astype(int) - want.astype(int))
    border = np.abs(np.abs(quotient - np.trunc(quotient)) - 0.5) < off
    assert (diff <= border).all()
    # The sum of squares: a thread adds at most max(64, k / 256 + 8) of them in
    # turn, then 6 + 4 partial sums; its half, and 8 for the rest.
    chain = max(64, k / 256 + 8) + 10
    got = np64(scales)
    ref = np.abs(y).max(-1) / 127
    assert (np.abs(got - ref) <= ref * (chain / 2 + 8) * U + 2.0 ** -149).all()
    # round(h + r): rounded to float32 before it is rounded to the type.
    res = np64(residual)
    assert (np.abs(res - s) <= np.abs(s) * (half_step(h.dtype) + U) * (1 + U) + tiny(h.dtype)).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m,k", [(1, 1), (5, 9), (2, 100), (3, 128), (7, 500), (1, 1024), (65, 1024), (3, 1100),
                                 (2, 3000), (4, 4095), (2, 8192), (2, 12001), (2, 20000)])
def test_add_rmsnorm_quantize(ops, dtype, m, k):
    g = gen(k + m)
    h, r = (torch.randn(m, k, generator=g).to(dtype) for _ in range(2))
    w = (torch.randn(k, generator=g) * 0.3).to(dtype)
    out = ops.add_rmsnorm_quantize(h.to(DEV), (2 * r).to(DEV), w.to(DEV), 1e-6)
    check_norm(h, 2 * r, w, 1e-6, *out)


def test_add_rmsnorm_quantize_extremes(ops):
    k = 72
    h = torch.zeros(5, k, dtype=BF16)
    r = torch.zeros(5, k, dtype=BF16)
    h[1, 2] = 1e-3
    h[2, 3] = float("nan")
    r[3, 4] = float("inf")
    h[4] = torch.linspace(-100, 100, k).to(BF16)
    w = torch.linspace(-1, 1, k).to(BF16)
    codes, scales, residual = ops.add_rmsnorm_quantize(h.to(DEV), r.to(DEV), w.to(DEV), 1e-6)
    assert bool((codes[0] == 0).all()) and scales[0].item() == 0.0
    assert bool(scales[2:4].isnan().all()) and bool((codes[2:4] == 0).all())
    keep = [0, 1, 4]
    check_norm(h[keep], r[keep], w, 1e-6, codes[keep], scales[keep], residual[keep])


def test_add_rmsnorm_quantize_views(ops):
    wide = torch.randn(9, 300, generator=gen(8)).to(BF16).to(DEV)
    w = (torch.randn(70, generator=gen(9)) * 0.3).to(BF16).to(DEV)
    h, r = wide[:, 5:75], wide[:, 101:171]
    check_norm(h.cpu(), r.cpu(), w.cpu(), 1e-5, *ops.add_rmsnorm_quantize(h, r, w, 1e-5))


# ---------------------------------------------------------------------------
# The product: the sum is exact, three roundings in float32, one to the type.
# ---------------------------------------------------------------------------
def operands(m, n, k, seed, extreme=False):
    g = gen(seed)
    a = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
    if extreme:
        a[0], w[0] = -128, -128
        a[-1], w[-1] = 127, -128
    sa = torch.rand(m, generator=g) * 0.01 + 1e-4
    sw = torch.rand(n, generator=g) * 0.002 + 1e-5
    return a, sa, w, sw


def check_product(got, a, sa, w, sw, dtype):
    ref = orc.gemm_int8(a.numpy(), sa.numpy(), w.numpy(), sw.numpy())
    tol = np.abs(ref) * (3.01 * U + (half_step(dtype) if dtype != F32 else 0.0) * (1 + 4 * U)) + tiny(dtype)
    bad = np.abs(np64(got) - ref) > tol
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:4])


def check_silu(got, a, sa, w, sw, dtype):
    y = orc.gemm_int8(a.numpy(), sa.numpy(), w.numpy(), sw.numpy())
    g, u = np.split(y, 2, -1)
    ref = orc.silu(g) * u
    # g and u are off by 3.01 U each; |d silu| <= 1.1 |dg| and, as a share of
    # silu, at most (1 + |g|) of g's; the exponential, the sum, the quotient and
    # the product round, 2 + 1 + 1 + 1 half steps of float32.  Below g = -88.7 the
    # exponential is infinite and silu is -0, where it is under 2^-121.
    rel = 3.01 * U * (2 + np.minimum(np.abs(g), 1.1 * np.abs(g) / np.maximum(np.abs(orc.silu(g)), 1e-300))) + 6 * U
    tol = np.abs(ref) * (rel + (half_step(dtype) if dtype != F32 else 0.0) * 1.001) + tiny(dtype) + 2.0 ** -120 * np.abs(u)
    bad = np.abs(np64(got) - ref) > tol
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:4])


# Tiles by size: decode rows of 8 to 64, 32- and 64-row tiles, 128 and 256; and
# the kernel for rows that are no aligned 16-byte chunks.
PRODUCTS = [(1, 1, 1), (1, 16, 16), (2, 33, 48), (7, 100, 1024), (8, 6144, 1024), (16, 1024, 3584), (17, 2100, 512),
            (31, 4096, 1040), (33, 4100, 2048), (64, 12300, 96), (64, 2048, 2048), (65, 70, 160), (130, 576, 512),
            (200, 1024, 3584), (512, 2048, 1024), (333, 2500, 1504), (1000, 2304, 2048), (600, 3600, 256),
            (2048, 2048, 1024), (2048, 4096, 1024), (1025, 9000, 1536), (2300, 6500, 2064),
            # any rows
            (1, 5, 3), (3, 7, 15), (9, 40, 17), (4, 300, 1003), (32, 515, 100), (70, 130, 131), (333, 2501, 1003),
            (300, 1100, 2050), (700, 5000, 333)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_gemm_int8(ops, m, n, k):
    a, sa, w, sw = operands(m, n, k, m + n + k, extreme=True)
    dev = [t.to(DEV) for t in (a, sa, w, sw)]
    for dtype in (BF16, F32, F16) if m * n * k < 1e9 else (BF16,):
        out = ops.gemm_int8(*dev, dtype)
        assert out.dtype == dtype and out.shape == (m, n)
        check_product(out, a, sa, w, sw, dtype)
    check_product(ops.gemm_int8(*dev), a, sa, w, sw, BF16)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("m,n,k", [(300, 5000, 1024), (2048, 4096, 1024), (1025, 9000, 1536), (600, 3600, 256)])
def test_gemm_int8_large_tiles_other_types(ops, dtype, m, n, k):
    a, sa, w, sw = operands(m, n, k, m + n)
    check_product(ops.gemm_int8(*[t.to(DEV) for t in (a, sa, w, sw)], dtype), a, sa, w, sw, dtype)


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 16, 64), (8, 500, 1024), (16, 3584, 1024), (24, 1600, 1024),
                                   (32, 1024, 512), (50, 3584, 1024), (64, 9000, 256), (100, 3584, 1024),
                                   (200, 3584, 1024), (729, 1216, 992), (300, 2600, 96), (2048, 3584, 1024),
                                   (2048, 1800, 1024), (4100, 3600, 512),
                                   (1, 3, 5), (5, 33, 17), (40, 100, 1003), (333, 700, 501), (600, 2600, 130)])
def test_gemm_int8_silu_mul(ops, m, n, k):
    a, sa, w, sw = operands(m, 2 * n, k, m + n + k)
    sw = sw * 3
    dev = [t.to(DEV) for t in (a, sa, w, sw)]
    for dtype in (BF16, F32, F16) if m * n * k < 5e8 else (BF16,):
        out = ops.gemm_int8_silu_mul(*dev, dtype)
        assert out.dtype == dtype and out.shape == (m, n)
        check_silu(out, a, sa, w, sw, dtype)


def test_gemm_int8_longest_sum(ops):
    """K = 131071 codes of -128 on both sides: the largest sum that int32 holds."""
    for k in (131071, 131056):
        a = torch.full((2, k), -128, dtype=torch.int8)
        w = torch.full((3, k), -128, dtype=torch.int8)
        w[1] = 127
        one = torch.ones(3)
        out = ops.gemm_int8(a.to(DEV), one[:2].to(DEV), w.to(DEV), one.to(DEV), F32)
        check_product(out, a, one[:2], w, one, F32)


def test_gemm_int8_scales_and_nan(ops):
    """A NaN scale makes its row (or column) NaN and no other; zero scales give 0."""
    a, sa, w, sw = operands(70, 90, 64, 3)
    sa[5], sw[7], sa[6], sw[8] = float("nan"), float("nan"), 0.0, 0.0
    for rows in (70, 9):
        out = ops.gemm_int8(a[:rows].to(DEV), sa[:rows].to(DEV), w.to(DEV), sw.to(DEV), F32).cpu()
        nan = out.isnan()
        want = torch.zeros_like(nan)
        want[5], want[:, 7] = True, True
        assert torch.equal(nan, want)
        assert bool((out[6, [0, 1, 8]] == 0).all()) and bool((out[[0, 1, 6], 8] == 0).all())


def test_gemm_int8_unaligned_and_batched(ops):
    """Operands at odd addresses, and rows of more than two dimensions."""
    a, sa, w, sw = operands(24, 50, 96, 4)
    base_a = torch.empty(24 * 96 + 16, dtype=torch.int8, device=DEV)
    base_w = torch.empty(50 * 96 + 16, dtype=torch.int8, device=DEV)
    for off in (1, 8):
        da = base_a[off:off + 24 * 96].view(24, 96).copy_(a)
        dw = base_w[off:off + 50 * 96].view(50, 96).copy_(w)
        check_product(ops.gemm_int8(da, sa.to(DEV), dw, sw.to(DEV), F32), a, sa, w, sw, F32)
    out = ops.gemm_int8(a.view(4, 6, 96).to(DEV), sa.view(4, 6).to(DEV), w.to(DEV), sw.to(DEV), F32)
    assert out.shape == (4, 6, 50)
    check_product(out.view(24, 50), a, sa, w, sw, F32)
    out = ops.gemm_int8(a[0].to(DEV), sa[0].to(DEV), w.to(DEV), sw.to(DEV), F32)
    assert out.shape == (50,)
    check_product(out.view(1, 50), a[:1], sa[:1], w, sw, F32)
    assert ops.gemm_int8(a[:0].to(DEV), sa[:0].to(DEV), w.to(DEV), sw.to(DEV)).shape == (0, 50)
    assert ops.gemm_int8(a.to(DEV), sa.to(DEV), w[:0].to(DEV), sw[:0].to(DEV)).shape == (24, 0)


def test_int8_on_a_side_stream_and_in_a_graph(ops):
    """The chain quantise, gate/up, quantise, down: on another stream, and captured, replayed on new inputs."""
    g = gen(11)
    hidden, inner = 256, 352
    wg, sg = ops.quantize_rows(torch.randn(2 * inner, hidden, generator=g).to(DEV) * 0.05)
    wd, sd = ops.quantize_rows(torch.randn(hidden, inner, generator=g).to(DEV) * 0.05)
    x = torch.randn(40, hidden, generator=g).to(BF16).to(DEV)

    def chain(x):
        mid = ops.gemm_int8_silu_mul(*ops.quantize_rows(x), wg, sg, x.dtype)
        return ops.gemm_int8(*ops.quantize_rows(mid), wd, sd, x.dtype)

    eager = chain(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = chain(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(eager, other)
    graph, static = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        out = chain(static)
    for seed in range(3):
        new = torch.randn(40, hidden, generator=gen(seed)).to(BF16).to(DEV)
        static.copy_(new)
        graph.replay()
        assert torch.equal(out, chain(new))


def test_int8_ops_have_no_backward(ops):
    x = torch.randn(4, 32, device=DEV, requires_grad=True)
    codes, scales = ops.quantize_rows(x)
    if scales.requires_grad:
        with pytest.raises(RuntimeError):
            scales.sum().backward()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", [(1, 65536, 16), (8, 65537, 144), (9, 70001, 272), (16, 65540, 528),
                                   (17, 65550, 1040), (32, 65551, 992)])
def test_gemm_int8_wide_heads(ops, dtype, m, n, k):
    """Decode rows on the output widths of LM heads."""
    a, sa, w, sw = operands(m, n, k, m + k, extreme=True)
    check_product(ops.gemm_int8(*[t.to(DEV) for t in (a, sa, w, sw)], dtype), a, sa, w, sw, dtype)


@pytest.mark.parametrize("m,n,k", [(3, 32768, 160), (16, 33001, 272), (29, 32780, 1040)])
def test_gemm_int8_silu_mul_wide(ops, m, n, k):
    a, sa, w, sw = operands(m, 2 * n, k, m + k)
    sw = sw * 3
    for dtype in (BF16, F32):
        check_silu(ops.gemm_int8_silu_mul(*[t.to(DEV) for t in (a, sa, w, sw)], dtype), a, sa, w, sw, dtype)


def test_add_rmsnorm_quantize_sums_beyond_float32(ops):
    """Squares that overflow make a row of zeros, squares that vanish at eps = 0 one of no number, both with codes 0, as the
    formula in float32 does."""
    h = torch.zeros(4, 96, dtype=BF16)
    h[0] = torch.linspace(1e20, 3e20, 96)
    h[1] = torch.linspace(-1e-25, 1e-25, 96)
    h[2] = torch.linspace(-2, 2, 96)
    w = torch.linspace(-0.5, 0.5, 96).to(BF16)
    codes, scales, residual = (t.cpu() for t in ops.add_rmsnorm_quantize(h.to(DEV), 0 * h.to(DEV), w.to(DEV), 0.0))
    assert scales[0] == 0 and scales[1].isnan() and scales[3].isnan()
    assert bool((codes[[0, 1, 3]] == 0).all()) and torch.equal(residual, h)
    check_norm(h[2:3], 0 * h[2:3], w, 0.0, codes[2:3], scales[2:3], residual[2:3])
    codes, scales, _ = (t.cpu() for t in ops.add_rmsnorm_quantize(h.to(DEV), 0 * h.to(DEV), w.to(DEV), 1e-6))
    assert scales[0] == 0 and scales[3] == 0 and bool((codes[[0, 3]] == 0).all())
    check_norm(h[1:3], 0 * h[1:3], w, 1e-6, codes[1:3], scales[1:3], torch.empty_like(h[1:3]).copy_(h[1:3]))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_torch_quantize_rows_on_the_gpu(ops, dtype):
    """The torch backend's codes and scales are the ops', to the last bit, and the oracle's."""
    x = (torch.randn(4096, 64, generator=gen(21)) * 3).to(dtype)
    x[1] = 0
    x[2] *= 1e-3
    x[3, 5] = float("nan")
    codes, scales = ops.torch_quantize_rows(x.to(DEV))
    check_rows(x, codes, scales)
