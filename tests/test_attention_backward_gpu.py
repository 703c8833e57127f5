"""GPU tests: the attention ops take inputs that require gradients, leave the
cache out of the graph, and refuse the backward, by name, in either
registration."""
from __future__ import annotations

import importlib

import pytest
import torch

from conftest import PKG

pytestmark = pytest.mark.gpu

A = importlib.import_module("inference_systems_amd.kernels.attention")
K = PKG.kernels
BF16 = torch.bfloat16
WRITTEN = {"rope_append": ("k_cache", "v_cache", "k_scales", "v_scales")}


def _ops(registration):
    """The four ops: as registered, or through torch.library.custom_op, the other registration."""
    names = ("rope_append", "kv_gather", "attention_prompt", "attention_paged")
    if registration == "library":
        return {n: getattr(torch.ops.nanovllm, n) for n in names}
    made = {}
    for n in names:
        where = f"nanovllm_backward_test::{n}"
        if not hasattr(getattr(torch.ops, "nanovllm_backward_test"), n):
            torch.library.custom_op(where, getattr(A, f"_{n}_op"), mutates_args=WRITTEN.get(n, ()))
        made[n] = getattr(torch.ops.nanovllm_backward_test, n)
    return made


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("registration", ["library", "custom_op"])
def test_a_backward_is_refused(registration, bits):
    print("backward", registration, bits, flush=True)
    ops, gen = _ops(registration), torch.Generator().manual_seed(bits)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    rows = [torch.randn((20, h, 64), generator=gen).to(BF16).cuda() for h in (4, 2, 2)]
    at, slots = torch.arange(20, device="cuda"), torch.arange(20, dtype=torch.int32, device="cuda")
    table, cu = K.rope_table(20, 64, device="cuda"), i32([0, 20])

    def run(q, k, v):
        cache = K.new_kv_cache(2, 16, 2, 64, bits=bits, device="cuda")
        q1, k1 = ops["rope_append"](q, k, v, at, table, slots, *cache)
        o1 = ops["attention_prompt"](q1, k1, v, cu, cu, 0.125)
        o2 = ops["attention_paged"](q1[-1:], cache.k, cache.v, i32([[0, 1]]), i32([20]), 0.125, cache.k_scales,
                                    cache.v_scales)
        o3, o4 = ops["kv_gather"](cache.k, cache.v, slots, cache.k_scales, cache.v_scales, BF16)
        return (q1, k1, o1, o2, o3, o4), cache

    want, _ = run(*rows)
    leaves = [x.clone().requires_grad_() for x in rows]
    got, cache = run(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # Queries and keys carry the refusal on; what is cached is data.
    assert not any(t is not None and t.requires_grad for t in cache)
    for out, op in zip(got[:4], ("rope_append", "rope_append", "attention_prompt", "attention_paged")):
        assert out.requires_grad
        with pytest.raises(RuntimeError, match=op):
            out.float().sum().backward(retain_graph=True)
    assert all(x.grad is None for x in leaves)
