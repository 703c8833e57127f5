"""A decode step and a prompt in 8 bits through the layers: norm, MLP, LM head and draw on the GPU kernels, against the
same arithmetic in torch operations and against the oracle's sampler."""
from __future__ import annotations

import pytest
import torch

from oracle import int8_oracle as orc

pytestmark = pytest.mark.gpu

DEV, BF16 = "cuda", torch.bfloat16
HIDDEN, INNER, VOCAB = 256, 688, 5003


def build(pkg, seed=0):
    L = pkg.layers
    g = torch.Generator().manual_seed(seed)
    parts = torch.nn.ModuleDict({"norm": L.Qwen35RMSNorm(HIDDEN), "mlp": L.Qwen35MLP(HIDDEN, INNER),
                                 "head": L.ParallelLMHead(VOCAB, HIDDEN), "o_proj": L.RowParallelLinear(512, HIDDEN)})
    for p in parts.parameters():
        p.data = torch.randn(p.shape, generator=g) * 0.1
    return L.quantize_int8(parts.to(BF16).to(DEV))


def backend(parts, name):
    for part in ("mlp", "head", "o_proj"):
        parts[part].gemm_backend = name


@torch.no_grad()
@pytest.mark.parametrize("rows", [1, 7, 40, 300])
def test_step_in_8_bits(pkg, rows):
    parts = build(pkg)
    g = torch.Generator().manual_seed(rows)
    h, r = (torch.randn(rows, HIDDEN, generator=g).to(BF16).to(DEV) for _ in range(2))
    heads, gate = (torch.randn(rows, 4, 128, generator=g).to(BF16).to(DEV) for _ in range(2))
    t, u = (0.6 + 0.5 * torch.rand(rows, generator=g)).to(DEV), torch.rand(rows, generator=g).to(DEV)
    k = torch.full((rows,), 30, dtype=torch.int32, device=DEV)
    p = torch.full((rows,), 0.95, device=DEV)

    def step(given=None):
        """The stages' outputs; each takes the one before it, or that of ``given``."""
        before = [None] * 4 if given is None else given
        a = parts["o_proj"].forward_gated(heads, gate)
        out, res = parts["mlp"].forward_add_norm((a if given is None else before[0]) + h, r, parts["norm"])
        plain = parts["mlp"](out if given is None else before[1])
        logits = parts["head"](out if given is None else before[1])
        return a, out, res, plain, logits

    backend(parts, "hip")
    hip = step()
    again = step()
    assert all(torch.equal(x, y) for x, y in zip(hip, again))
    tokens, shares = parts["head"].draw(hip[1], t, u, k, p)
    backend(parts, "torch")
    # Codes and sums are the same but where a rounding to 16 bits, or the norm's
    # last bits, fall to the other side: then an element is a step (2^-8 of it)
    # or a code (1 / 127 of a row's largest value, a third of which is the rms)
    # off.  Were each off by as much at random, outputs were off by 1%.
    for x, y in zip(hip, step(hip)):
        assert x.dtype == y.dtype and x.shape == y.shape
        assert (x.float() - y.float()).norm() <= 0.01 * y.float().norm()
    logits = hip[4].double().cpu().numpy()
    for i in range(rows):
        token, share = orc.sample(logits[i], float(t[i]), float(u[i]), 30, float(p[i]))
        assert tokens[i] == token and abs(shares[i].item() - share) <= abs(share) * 2.0 ** -24 + 1e-11


@torch.no_grad()
def test_step_in_8_bits_is_captured(pkg):
    parts = build(pkg, 1)
    backend(parts, "hip")
    rows = 16
    static = [torch.zeros(rows, HIDDEN, dtype=BF16, device=DEV), torch.zeros(rows, HIDDEN, dtype=BF16, device=DEV),
              torch.ones(rows, device=DEV), torch.zeros(rows, device=DEV)]

    def step(h, r, t, u):
        out, res = parts["mlp"].forward_add_norm(h, r, parts["norm"])
        return out, res, *parts["head"].draw(out, t, u)

    step(*static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        new = [torch.randn(rows, HIDDEN, generator=g).to(BF16), torch.randn(rows, HIDDEN, generator=g).to(BF16),
               0.5 + torch.rand(rows, generator=g), torch.rand(rows, generator=g)]
        for dst, src in zip(static, new):
            dst.copy_(src)
        graph.replay()
        want = step(*[x.to(DEV) for x in new])
        assert all(torch.equal(x, y) for x, y in zip(out, want))


@torch.no_grad()
def test_float_scales_are_refused_once_converted(pkg):
    """A module converted after its weights went to 8 bits has 16-bit scales: refused, not used."""
    parts = build(pkg, 2)
    mlp = parts["mlp"].to(BF16)
    mlp.gemm_backend = "hip"
    with pytest.raises(RuntimeError, match="float32"):
        mlp(torch.zeros(2, HIDDEN, dtype=BF16, device=DEV))


@torch.no_grad()
@pytest.mark.parametrize("name", ["hip", "auto"])
def test_gated_rows_in_8_bits(pkg, name):
    """On the gate's kernel, and without rows."""
    layer = build(pkg, 3)["o_proj"]
    layer.gemm_backend = name
    g = torch.Generator().manual_seed(4)
    for m in (0, 1, 5):
        x, gate = (torch.randn(m, 4, 128, generator=g).to(BF16).to(DEV) for _ in range(2))
        out = layer.forward_gated(x, gate)
        assert out.shape == (m, HIDDEN) and out.dtype == BF16
        if m:
            assert torch.equal(out, layer(pkg.kernels.sigmoid_gate(x, gate)))
