"""CPU tests of the 8-bit ops and the sampler: registration, fake shapes, refusals, the torch backend against the
oracle, and the layers that keep their weights in 8 bits."""
from __future__ import annotations

import os
import subprocess
import sys

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from conftest import PKG, ROOT
from oracle import int8_oracle as orc

K, Lyr = PKG.kernels, PKG.layers
U = 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32


def meta(*shape, dtype=F32):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_fake_shapes():
    ops = torch.ops.nanovllm
    codes, scales = ops.quantize_rows(meta(3, 5, 64, dtype=BF16))
    assert codes.shape == (3, 5, 64) and codes.dtype == torch.int8 and scales.shape == (3, 5) and scales.dtype == F32
    h, w = meta(7, 64, dtype=BF16), meta(64, dtype=BF16)
    codes, scales, res = ops.add_rmsnorm_quantize(h, h, w, 1e-6)
    assert codes.shape == res.shape == (7, 64) and scales.shape == (7,) and res.dtype == BF16
    a, sa = meta(3, 5, 64, dtype=torch.int8), meta(3, 5)
    wt, sw = meta(96, 64, dtype=torch.int8), meta(96)
    assert ops.gemm_int8(a, sa, wt, sw).shape == (3, 5, 96) and ops.gemm_int8(a, sa, wt, sw).dtype == BF16
    out = ops.gemm_int8_silu_mul(a, sa, wt, sw, F32)
    assert out.shape == (3, 5, 48) and out.dtype == F32
    tokens, logprobs = ops.sample_logits(meta(4, 100), meta(4), meta(4))
    assert tokens.shape == logprobs.shape == (4,) and tokens.dtype == torch.int64 and logprobs.dtype == F32


class Gpu:
    """Looks like a tensor on a GPU to the contract functions."""

    def __init__(self, t, device="cuda:0"):
        self._t, self.is_cuda, self.device = t, True, torch.device(device)

    def __getattr__(self, name):
        return getattr(self._t, name)


def gpu(*shape, dtype=F32, device="cuda:0"):
    return Gpu(torch.zeros(shape, dtype=dtype), device)


def test_quantize_rows_contract():
    reason = K.quantize_rows_contract_reason
    assert reason(gpu(3, 7)) is None and reason(gpu(7, dtype=torch.float16)) is None
    assert reason(Gpu(torch.zeros(4, 20)[:, 3:9])) is None and reason(gpu(0, 5)) is None
    assert "CUDA" in reason(torch.zeros(3, 7))
    assert "float32" in reason(gpu(3, 7, dtype=torch.float64))
    assert "dimension" in reason(gpu())
    assert "K must" in reason(gpu(3, 0))
    assert "unit stride" in reason(Gpu(torch.zeros(7, 3).t()))
    assert "contiguous" in reason(Gpu(torch.zeros(2, 3, 8)[:, :, 1:]))
    assert "overlap" in reason(Gpu(torch.zeros(40).as_strided((4, 8), (4, 1))))
    assert "2^23" in reason(gpu(2 ** 23 + 1, 1, dtype=BF16))


def test_add_rmsnorm_quantize_contract():
    reason, b = K.add_rmsnorm_quantize_contract_reason, BF16
    h, w = gpu(3, 8, dtype=b), gpu(8, dtype=b)
    assert reason(h, h, w, 1e-6) is None
    assert "CUDA" in reason(h, torch.zeros(3, 8, dtype=b), w, 1e-6)
    assert "same device" in reason(h, h, gpu(8, dtype=b, device="cuda:1"), 1e-6)
    assert "float16 or bfloat16" in reason(gpu(3, 8), gpu(3, 8), gpu(8), 1e-6)
    assert "same dtype" in reason(h, h, gpu(8), 1e-6)
    assert "same shape" in reason(h, gpu(4, 8, dtype=b), w, 1e-6)
    assert "same shape" in reason(gpu(8, dtype=b), gpu(8, dtype=b), w, 1e-6)
    assert "(K,)" in reason(h, h, gpu(9, dtype=b), 1e-6)
    assert "K must" in reason(gpu(3, 0, dtype=b), gpu(3, 0, dtype=b), gpu(0, dtype=b), 1e-6)
    for eps in (-1.0, float("nan"), float("inf")):
        assert "eps" in reason(h, h, w, eps)


def test_gemm_int8_contract():
    reason, i = K.gemm_int8_contract_reason, torch.int8
    a, sa, w, sw = gpu(3, 32, dtype=i), gpu(3), gpu(6, 32, dtype=i), gpu(6)
    assert reason(a, sa, w, sw) is None and reason(a, sa, w, sw, F32, True) is None
    assert "CUDA" in reason(torch.zeros(3, 32, dtype=i), sa, w, sw)
    assert "same device" in reason(a, sa, w, gpu(6, device="cuda:1"))
    assert "must be int8" in reason(gpu(3, 32), sa, w, sw)
    assert "float32" in reason(a, gpu(3, dtype=BF16), w, sw)
    assert "out_dtype" in reason(a, sa, w, sw, torch.int32)
    assert "2-D" in reason(a, sa, gpu(32, dtype=i), sw)
    assert "w.size(1)" in reason(gpu(3, 31, dtype=i), sa, w, sw)
    assert "K (0)" in reason(gpu(3, 0, dtype=i), sa, gpu(6, 0, dtype=i), sw)
    long = gpu(1, 131072, dtype=i)
    assert "131071" in reason(long, gpu(1), long, gpu(1))
    assert "equal height" in reason(a, sa, gpu(5, 32, dtype=i), gpu(5), None, True)
    assert "contiguous" in reason(Gpu(torch.zeros(3, 40, dtype=i)[:, :32]), sa, w, sw)
    assert "a_scales" in reason(a, gpu(4), w, sw) and "w_scales" in reason(a, sa, w, gpu(5))


def test_sample_logits_contract():
    reason = K.sample_logits_contract_reason
    x, t = gpu(3, 50), gpu(3)
    k = gpu(3, dtype=torch.int32)
    assert reason(x, t, t) is None and reason(x, t, t, k, t, t) is None
    assert reason(Gpu(torch.zeros(3, 60)[:, 5:55]), t, t) is None
    assert "CUDA" in reason(torch.zeros(3, 50), t, t) and "CUDA" in reason(x, t, torch.zeros(3))
    assert "same device" in reason(x, t, t, None, gpu(3, device="cuda:1"))
    assert "logits must be float32" in reason(gpu(3, 50, dtype=torch.float64), t, t)
    assert "entries" in reason(gpu(3, 0), t, t) and "entries" in reason(gpu(), t, t)
    assert "entries" in reason(gpu(1, 2 ** 23 + 1, dtype=BF16), gpu(1), gpu(1))
    assert "2^20" in reason(gpu(2 ** 20 + 1, 1, dtype=BF16), t, t)
    assert "overlap" in reason(Gpu(torch.zeros(40).as_strided((4, 8), (4, 1))), gpu(4), gpu(4))
    assert "temperatures must be" in reason(x, gpu(3, dtype=BF16), t)
    assert "uniforms must be" in reason(x, t, gpu(4))
    assert "top_k must be torch.int32" in reason(x, t, t, gpu(3, dtype=torch.int64))
    assert "top_p must be" in reason(x, t, t, None, gpu(2))
    assert "min_p must be" in reason(x, t, t, None, None, Gpu(torch.zeros(6)[::2]))


CPU_CALLS = {
    "quantize_rows": lambda: K.quantize_rows(torch.zeros(2, 8)),
    "add_rmsnorm_quantize": lambda: K.add_rmsnorm_quantize(*(torch.zeros(2, 8, dtype=BF16),) * 2,
                                                           torch.zeros(8, dtype=BF16), 1e-6),
    "gemm_int8": lambda: K.gemm_int8(torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2),
                                     torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4)),
    "gemm_int8_silu_mul": lambda: K.gemm_int8_silu_mul(torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2),
                                                       torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4)),
    "sample_logits": lambda: K.sample_logits(torch.zeros(2, 8), torch.zeros(2), torch.zeros(2)),
}


@pytest.mark.parametrize("name", CPU_CALLS)
def test_cpu_tensors_are_refused(name):
    with pytest.raises(RuntimeError, match=f"nanovllm::{name}: .*CUDA"):
        CPU_CALLS[name]()


def test_both_registrations_have_the_same_schemas():
    code = ("import sys, json; sys.path.insert(0, {root!r}); import torch, __graft_entry__ as g; "
            "p = g.load_package(); G = sys.modules['inference_systems_amd.kernels.gemm']; "
            "print(G.REGISTRATION); [print(getattr(torch.ops.nanovllm, n).default._schema) for n in {names!r}]")
    said = {}
    for asked in ("torch_library", "custom_op"):
        proc = subprocess.run([sys.executable, "-c", code.format(root=str(ROOT), names=sorted(CPU_CALLS))],
                              env=dict(os.environ, NANOVLLM_GEMM_OPS=asked), capture_output=True, text=True)
        if proc.returncode and asked == "torch_library":
            pytest.skip("the C++ registration is not built")
        lines = proc.stdout.split("\n")
        assert lines[0] == asked, proc.stderr
        said[asked] = [line.replace("SymInt", "int") for line in lines[1:]]
    assert said["torch_library"] == said["custom_op"]


@pytest.mark.parametrize("dtype", [F32, torch.float16, BF16])
def test_torch_quantize_rows_against_the_oracle(dtype):
    x = (torch.randn(40, 33, generator=torch.Generator().manual_seed(1)) * 5).to(dtype)
    x[3] = 0
    x[4, 2] = float("nan")
    x[5, 3] = float("inf")
    x[6, 0], x[6, 1:] = 8.0, 4.0
    codes, scales = K.torch_quantize_rows(x)
    want, scale, _ = orc.quantize_rows(x.double().numpy())
    np.testing.assert_array_equal(codes.numpy(), want)
    np.testing.assert_array_equal(scales.numpy(), scale)


def test_torch_sample_logits_against_the_oracle():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(64, 300, generator=g) * 3
    x[1, 5] = float("nan")
    x[2] = -float("inf")
    x[3, 7] = float("inf")
    x[4, 10:] = -float("inf")
    t, u, p, q = (torch.rand(64, generator=g) for _ in range(4))
    t[5:9] = 0
    k = torch.randint(-5, 350, (64,), generator=g, dtype=torch.int32)
    u[10], u[11], u[12] = 1.0, -1.0, float("nan")
    p[13], p[14], p[15], q[16] = 0.0, 1.0, float("nan"), 2.0
    tokens, shares = K.sample_rows(x, t, u, k, p, q * 0.3, backend="auto")
    for i in range(64):
        token, share = orc.sample(x[i].double().numpy(), *(float(v[i]) for v in (t, u, k, p, q * 0.3)))
        assert tokens[i] == token, i
        assert (np.isnan(share) and shares[i].isnan()) or abs(shares[i].item() - share) <= abs(share) * U + 1e-11


def test_backend_switch_refuses_and_falls_back():
    x = torch.randn(3, 16)
    w, s = K.torch_quantize_rows(torch.randn(8, 16))
    with pytest.raises(RuntimeError, match="HIP GEMM backend is unavailable"):
        K.int8_linear(x, w, s, backend="hip")
    with pytest.raises(RuntimeError, match="HIP GEMM backend is unavailable"):
        K.int8_silu_mul_linear(x, w, s, backend="hip")
    with pytest.raises(RuntimeError, match="HIP GEMM backend is unavailable"):
        K.int8_add_rmsnorm_linear(x, x, torch.zeros(16), 1e-6, w, s, backend="hip")
    with pytest.raises(RuntimeError, match="HIP GEMM backend is unavailable"):
        K.sample_rows(x, torch.ones(3), torch.ones(3), backend="hip")
    assert torch.equal(K.int8_linear(x, w, s, backend="auto"), K.int8_linear(x, w, s, backend="torch"))


def int8_error(x, w):
    """How far a product of rows in 8 bits may be from the exact one: half a step of each factor."""
    sx, sw = x.double().abs().amax(-1, keepdim=True) / 127, w.double().abs().amax(-1) / 127
    k = x.shape[-1]
    return ((sx / 2) * w.double().abs().sum(-1) + (sw / 2) * x.double().abs().sum(-1, keepdim=True)
            + k * sx * sw / 4) * (1 + 1e-5)


def test_layers_in_8_bits():
    g = torch.Generator().manual_seed(3)
    layer = Lyr.ColumnParallelLinear(48, 40, bias=True)
    w, b, x = torch.randn(40, 48, generator=g), torch.randn(40, generator=g), torch.randn(5, 48, generator=g)
    layer.weight.weight_loader(layer.weight, w)
    layer.bias.weight_loader(layer.bias, b)
    layer.gemm_backend = "auto"
    layer.quantize_int8()
    layer.quantize_int8()
    assert layer.weight is None and layer.weight_codes.dtype == torch.int8 and layer.is_int8
    assert set(layer.state_dict()) == {"bias", "weight_codes", "weight_scales"}
    exact = F.linear(x.double(), w.double(), b.double())
    assert bool(((layer(x).double() - exact).abs() <= int8_error(x, w) + 1e-4).all())

    row = Lyr.RowParallelLinear(32, 24)
    wr = torch.randn(24, 32, generator=g)
    row.weight.weight_loader(row.weight, wr)
    row.gemm_backend = "torch"
    row.quantize_int8()
    y, gate = torch.randn(6, 4, 8, generator=g), torch.randn(6, 4, 8, generator=g)
    gated = (y * torch.sigmoid(gate)).reshape(6, 32)
    assert bool(((row.forward_gated(y, gate).double() - F.linear(gated.double(), wr.double())).abs()
                 <= int8_error(gated, wr) + 1e-4).all())

    gdn = Lyr.GdnInputProjection(32, 2, 4, 8, 8)
    torch.nn.init.normal_(gdn.weight)
    gdn.gemm_backend = "torch"
    z = torch.randn(3, 32, generator=g)
    before = torch.cat(gdn(z), -1)
    bound = int8_error(z, gdn.weight.detach())
    Lyr.quantize_int8(gdn)
    for contiguous in (False, True):
        parts = gdn(z, contiguous)
        assert all(p.is_contiguous() for p in parts) or not contiguous
        assert bool(((torch.cat(parts, -1) - before).abs() <= bound + 1e-4).all())


@torch.no_grad()
def test_step_in_8_bits_on_the_torch_backend():
    """Norm, MLP, LM head and draw, as a decode step runs them."""
    g = torch.Generator().manual_seed(4)
    mlp, norm, head = Lyr.Qwen35MLP(32, 48), Lyr.Qwen35RMSNorm(32), Lyr.ParallelLMHead(200, 32)
    for p in (*mlp.parameters(), *head.parameters()):
        p.data = torch.randn(p.shape, generator=g) * 0.2
    h, r = torch.randn(6, 32, generator=g), torch.randn(6, 32, generator=g)
    mlp.gemm_backend = head.gemm_backend = "torch"
    exact, res = mlp.forward_add_norm(h, r, norm)
    for layer in (mlp, head):
        Lyr.quantize_int8(layer)
    out, res8 = mlp.forward_add_norm(h, r, norm)
    assert torch.equal(res, res8)
    # A code is off by a step / sqrt(12) rms, a step being the row's largest value / 127, here 3 rms or less: 0.7% of the
    # rms; two factors a product, two products and the SiLU between them make 2% of what is random, and no more than 5%.
    assert (out - exact).norm() < 0.05 * exact.norm()
    t, u = torch.full((6,), 0.8), torch.rand(6, generator=g)
    k = torch.full((6,), 20, dtype=torch.int32)
    tokens, shares = head.draw(out, t, u, k)
    logits = head(out)
    assert all(orc.sample(logits[i].double().numpy(), 0.8, float(u[i]), 20)[0] == tokens[i] for i in range(6))
    assert bool((shares <= 0).all())
    for call in (lambda: head.greedy(out), lambda: head.sample(out, t, 0, 0)):
        with pytest.raises(RuntimeError, match="8 bits"):
            call()


def test_torch_sample_logits_at_infinite_temperatures():
    """Every finite logit weighs 1; below an infinite one nothing has weight."""
    inf = float("inf")
    x = torch.randn(6, 40, generator=torch.Generator().manual_seed(5))
    x[1, ::3] = -inf
    x[2] = -inf
    x[3, 7], x[3, 20], x[3, 30] = inf, inf, -inf
    x[4] = inf
    t, u = torch.full((6,), inf), torch.linspace(0, 0.99, 6)
    for p, q in ((None, None), (0.5, None), (None, 1.0), (0.5, 0.5), (None, 2.0)):
        tokens, shares = K.torch_sample_logits(x, t, u, None, *(None if v is None else torch.full((6,), v) for v in (p, q)))
        for i in range(6):
            token, share = orc.sample(x[i].double().numpy(), inf, float(u[i]), None, p, q)
            assert tokens[i] == token and abs(shares[i].item() - share) <= abs(share) * U + 1e-11, (i, p, q)


NO_BACKWARD = {
    "int8_linear": lambda x, r, n, w, s: [K.int8_linear(x, w, s, backend="torch")],
    "int8_silu_mul_linear": lambda x, r, n, w, s: [K.int8_silu_mul_linear(x, w, s, backend="torch")],
    "int8_add_rmsnorm_linear": lambda x, r, n, w, s: K.int8_add_rmsnorm_linear(x, r, n, 1e-6, w, s, backend="torch"),
}


@pytest.mark.parametrize("name", NO_BACKWARD)
def test_the_torch_backend_has_no_backward_either(name):
    """What is differentiable of a row in 8 bits is its scale alone: refused, as the ops refuse it."""
    g = torch.Generator().manual_seed(6)
    x, r, n = torch.randn(3, 16, generator=g), torch.randn(3, 16, generator=g), torch.randn(16, generator=g)
    w, s = K.torch_quantize_rows(torch.randn(8, 16, generator=g))
    want = NO_BACKWARD[name](x, r, n, w, s)
    assert not any(y.requires_grad for y in want)
    for leaf in (x, n) if "norm" in name else (x,):
        leaf.requires_grad_()
        with torch.no_grad():
            assert not any(y.requires_grad for y in NO_BACKWARD[name](x, r, n, w, s))
        for i, y in enumerate(want):
            out = NO_BACKWARD[name](x, r, n, w, s)[i]
            assert torch.equal(out, y) and out.requires_grad
            with pytest.raises(RuntimeError, match=f"{name} has no backward"):
                out.sum().backward()
        assert leaf.grad is None
        leaf.requires_grad_(False)


LAYERS = {
    "column": lambda: Lyr.ColumnParallelLinear(48, 40, bias=True),
    "merged": lambda: Lyr.MergedColumnParallelLinear(48, [24, 16]),
    "row": lambda: Lyr.RowParallelLinear(48, 40),
    "gdn": lambda: Lyr.GdnInputProjection(48, 2, 4, 8, 8),
    "head": lambda: Lyr.ParallelLMHead(200, 48),
    "mlp": lambda: Lyr.Qwen35MLP(48, 32),
}


def _made(name, seed, int8):
    layer = LAYERS[name]()
    g = torch.Generator().manual_seed(seed)
    for p in layer.parameters():
        p.data = torch.randn(p.shape, generator=g)
    for part in layer.modules():
        if hasattr(part, "gemm_backend"):
            part.gemm_backend = "torch"
    return Lyr.quantize_int8(layer) if int8 else layer


def _same(x, y):
    return all(torch.equal(a, b) for a, b in zip(*(v if isinstance(v, tuple) else (v,) for v in (x, y))))


@torch.no_grad()
@pytest.mark.parametrize("strict", [True, False])
@pytest.mark.parametrize("assign", [False, True])
@pytest.mark.parametrize("name", LAYERS)
def test_a_state_dict_in_8_bits_is_loaded(name, assign, strict):
    """Into a 16-bit layer, which keeps its weight in 8 bits from then on, and into one in 8 bits."""
    x = torch.randn(5, 48, generator=torch.Generator().manual_seed(9))
    saved = _made(name, 1, True)
    want, state = saved(x), {k: v.clone() for k, v in saved.state_dict().items()}
    for int8 in (False, True):
        layer = _made(name, 2, int8)
        out = layer.load_state_dict(state, strict=strict, assign=assign)
        assert not out.missing_keys and not out.unexpected_keys
        assert all(part.is_int8 for part in layer.modules() if isinstance(part, Lyr.Int8Weight))
        assert _same(layer(x), want)
        again = layer.state_dict()
        assert set(again) == set(state) and all(again[k].dtype == state[k].dtype for k in state)


@pytest.mark.parametrize("strict", [True, False])
def test_state_dicts_that_do_not_fit_are_refused(strict):
    layer, full = _made("row", 3, False), _made("row", 4, True)
    short = {"weight_codes": full.weight_codes[:39], "weight_scales": full.weight_scales[:39]}
    with pytest.raises(RuntimeError, match="size mismatch for weight_codes"):
        layer.load_state_dict(short, strict=strict)
    assert not layer.is_int8 and layer.weight is not None
    with pytest.raises(RuntimeError, match="keeps its weight in 8 bits"):
        full.load_state_dict(layer.state_dict(), strict=strict)
    assert full.is_int8
    with pytest.raises(RuntimeError, match="size mismatch"):
        full.load_state_dict(short, strict=strict)
    if strict:
        with pytest.raises(RuntimeError, match="weight_codes"):
            layer.load_state_dict({"weight_codes": full.weight_codes})


@torch.no_grad()
@pytest.mark.parametrize("bias", [False, True])
def test_every_linear_layer_goes_to_8_bits(bias):
    """GemmLinear, the drop-in for nn.Linear, among them: its rows go through the 8-bit product, and its state dict loads."""
    g = torch.Generator().manual_seed(8)
    model = torch.nn.ModuleDict({"plain": Lyr.GemmLinear(48, 40, bias=bias), "row": Lyr.RowParallelLinear(40, 48)})
    plain = model["plain"]
    plain.gemm_backend = "auto"
    for p in model.parameters():
        p.data = torch.randn(p.shape, generator=g)
    x, w, b = torch.randn(5, 48, generator=g), plain.weight.clone(), plain.bias
    exact = F.linear(x.double(), w.double(), None if b is None else b.double())
    assert Lyr.quantize_int8(model) is model
    assert plain.is_int8 and plain.weight is None and model["row"].is_int8
    assert bool(((plain(x).double() - exact).abs() <= int8_error(x, w) + 1e-4).all())
    fresh = Lyr.GemmLinear(48, 40, bias=bias)
    fresh.load_state_dict(plain.state_dict())
    assert fresh.is_int8 and torch.equal(fresh(x), plain(x))


@torch.no_grad()
@pytest.mark.parametrize("backend", ["torch", "auto"])
@pytest.mark.parametrize("shapes", [((4, 8), (4, 8)), ((32,), (32,)), ((32,), (4, 8)), ((4, 8), (32,))])
def test_gated_rows_in_8_bits(backend, shapes):
    """The heads and their gate in either layout, without rows too."""
    g = torch.Generator().manual_seed(12)
    row = Lyr.RowParallelLinear(32, 24)
    row.weight.data = torch.randn(24, 32, generator=g)
    row.gemm_backend = backend
    row.quantize_int8()
    for m in (0, 1, 5):
        x, gate = (torch.randn(m, *s, generator=g) for s in shapes)
        want = row((x.reshape(m, 32) * torch.sigmoid(gate.reshape(m, 32))))
        assert torch.equal(row.forward_gated(x, gate), want) and want.shape == (m, 24)


@torch.no_grad()
@pytest.mark.parametrize("backend", ["torch", "auto"])
def test_scales_of_a_converted_module_are_refused(backend):
    """As on the HIP backend: scales rounded to 16 bits are not used in silence."""
    mlp, norm = _made("mlp", 1, True).to(BF16), Lyr.Qwen35RMSNorm(48).to(BF16)
    mlp.gemm_backend = backend
    x = torch.zeros(2, 48, dtype=BF16)
    for call in (lambda: mlp(x), lambda: mlp.forward_add_norm(x, x, norm), lambda: mlp.down_proj(x[:, :32])):
        with pytest.raises(RuntimeError, match="w must be int8 and w_scales float32"):
            call()
