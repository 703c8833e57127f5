"""GPU tests: the 8-bit ops and the sampler take inputs that require gradients and refuse the backward, by name, in either
registration."""
from __future__ import annotations

import importlib

import pytest
import torch

from conftest import PKG

pytestmark = pytest.mark.gpu

I8 = importlib.import_module("inference_systems_amd.kernels.int8")
SAMPLING = importlib.import_module("inference_systems_amd.kernels.sampling")
K = PKG.kernels
BF16 = torch.bfloat16
NAMES = ("quantize_rows", "add_rmsnorm_quantize", "gemm_int8", "gemm_int8_silu_mul", "sample_logits")


def _op(name, registration):
    """As registered, or through torch.library.custom_op, the other registration."""
    if registration == "library":
        return getattr(torch.ops.nanovllm, name)
    if not hasattr(torch.ops.nanovllm_int8_backward_test, name):
        source = SAMPLING if name == "sample_logits" else I8
        torch.library.custom_op(f"nanovllm_int8_backward_test::{name}", getattr(source, f"_{name}_op"), mutates_args=())
    return getattr(torch.ops.nanovllm_int8_backward_test, name)


def _inputs(name):
    """(tensors and plain values of a call, places of those that have a gradient to ask for)."""
    g = torch.Generator().manual_seed(1)
    row = lambda *s: torch.randn(s, generator=g).cuda()  # noqa: E731
    if name == "quantize_rows":
        return [row(5, 48)], [0]
    if name == "add_rmsnorm_quantize":
        return [row(5, 48).to(BF16), row(5, 48).to(BF16), row(48).to(BF16), 1e-6], [0, 1, 2]
    if name == "sample_logits":
        return [row(5, 300), torch.ones(5).cuda(), torch.rand(5, generator=g).cuda()], [0, 1]
    a, sa = K.quantize_rows(row(5, 48))
    w, sw = K.quantize_rows(row(8, 48))
    return [a, sa, w, sw, torch.float32], [1, 3]


@pytest.mark.parametrize("registration", ["library", "custom_op"])
@pytest.mark.parametrize("name", NAMES)
def test_a_backward_is_refused(name, registration):
    op = _op(name, registration)
    inputs, places = _inputs(name)
    outs = lambda given: [y for y in (lambda r: r if isinstance(r, tuple) else (r,))(op(*given))]  # noqa: E731
    want = outs(inputs)
    for place in places:
        given = list(inputs)
        given[place] = inputs[place].clone().requires_grad_()
        got = outs(given)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        asked = [y for y in got if y.is_floating_point()]
        assert asked and all(y.requires_grad for y in asked)
        for y in asked:
            with pytest.raises(RuntimeError, match=name):
                y.float().sum().backward(retain_graph=True)
        assert given[place].grad is None


@pytest.mark.parametrize("name", ["int8_linear", "int8_silu_mul_linear", "int8_add_rmsnorm_linear"])
def test_the_linears_refuse_it(name):
    g = torch.Generator().manual_seed(2)
    x, r, n = (torch.randn(*s, generator=g).to(BF16).cuda() for s in ((5, 64), (5, 64), (64,)))
    w, s = K.quantize_rows(torch.randn(16, 64, generator=g).cuda())
    x.requires_grad_()
    if name == "int8_add_rmsnorm_linear":
        outs = K.int8_add_rmsnorm_linear(x, r, n, 1e-6, w, s, backend="hip")
    else:
        outs = [getattr(K, name)(x, w, s, backend="hip")]
    for y in outs:
        assert y.requires_grad
        with pytest.raises(RuntimeError, match="nanovllm::|not implemented"):
            y.float().sum().backward(retain_graph=True)
    assert x.grad is None
