"""CPU tests of the attention ops: registration, fake shapes, refusals, the
plain torch backend against the oracle, and the layer on it."""
from __future__ import annotations

import importlib
import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from conftest import PKG, ROOT
from oracle import attention_oracle as orc

A = importlib.import_module("inference_systems_amd.kernels.attention")
G = importlib.import_module("inference_systems_amd.kernels.gemm")
K = PKG.kernels
BF16, F16 = torch.bfloat16, torch.float16
OPS = ("rope_append", "kv_gather", "attention_prompt", "attention_paged")

PROBE = r"""
import json, sys
sys.path.insert(0, {root!r})
import torch
import __graft_entry__ as g
K = g.load_package().kernels
said = []
x, i = torch.zeros(4, 2, 64).half(), torch.zeros(4, dtype=torch.int32)
cache = K.new_kv_cache(2, 16, 2, 64, dtype=torch.float16)
for call in (lambda: K.rope_append(x, x, x, i.long(), K.rope_table(4, 64), i, *cache[:2]),
             lambda: K.kv_gather(cache.k, cache.v, i),
             lambda: K.attention_prompt(x, x, x, i, i, 0.1),
             lambda: K.attention_paged(x, cache.k, cache.v, i[:, None], i, 0.1)):
    try:
        call()
    except RuntimeError as exc:
        said.append(str(exc).splitlines()[0])
print(json.dumps({{"schemas": [str(getattr(torch.ops.nanovllm, op).default._schema) for op in {ops!r}],
                  "said": said}}))
"""


def test_registrations_share_schema_and_messages():
    got = []
    for choice in ("torch_library", "custom_op"):
        env = dict(os.environ)
        env.pop("NANOVLLM_GEMM_LIB", None)
        env[G.OPS_ENV] = choice
        proc = subprocess.run([sys.executable, "-c", PROBE.format(root=str(ROOT), ops=OPS)], env=env,
                              capture_output=True, text=True, timeout=300)
        assert proc.returncode == 0, proc.stderr[-2000:]
        got.append(json.loads(proc.stdout.strip().splitlines()[-1]))
    assert got[0] == got[1]
    assert got[0]["said"] == [f"nanovllm::{op}: all operands must be CUDA (HIP) tensors" for op in OPS]


def test_fake_shapes():
    x, y = (torch.empty((5, h, 128), dtype=BF16, device="meta") for h in (4, 2))
    i = torch.empty(5, dtype=torch.int32, device="meta")
    c16, c4 = (K.new_kv_cache(3, 16, 2, 128, bits=b, device="meta") for b in (16, 4))
    q, k = torch.ops.nanovllm.rope_append(x, y, y, i.long(), torch.empty((9, 64), device="meta"), i, *c4)
    assert q.shape == x.shape and k.shape == y.shape and q.dtype == BF16
    assert K.kv_gather(c16.k, c16.v, i)[1].shape == (5, 2, 128)
    k, v = K.kv_gather(c4.k, c4.v, i, c4.k_scales, c4.v_scales, F16)
    assert k.shape == v.shape == (5, 2, 128) and k.dtype == F16
    assert K.attention_prompt(x, y, y, i, i, 0.1).shape == x.shape
    assert K.attention_paged(x, c16.k, c16.v, i[:, None], i, 0.1).shape == x.shape


def _append_args(**changes):
    cache = K.new_kv_cache(3, 16, 2, 128)
    a = dict(q=torch.zeros(5, 4, 128, dtype=BF16), k=torch.zeros(5, 2, 128, dtype=BF16),
             v=torch.zeros(5, 2, 128, dtype=BF16), positions=torch.zeros(5, dtype=torch.int64),
             cos_sin=K.rope_table(9, 64), slots=torch.zeros(5, dtype=torch.int32), k_cache=cache.k, v_cache=cache.v)
    a.update(changes)
    return a


def _paged_args(**changes):
    cache = K.new_kv_cache(3, 16, 2, 128)
    a = dict(q=torch.zeros(5, 4, 128, dtype=BF16), k_cache=cache.k, v_cache=cache.v,
             block_tables=torch.zeros((5, 3), dtype=torch.int32), context_lens=torch.zeros(5, dtype=torch.int32),
             scale=0.1)
    a.update(changes)
    return a


def _prompt_args(**changes):
    cu = torch.zeros(3, dtype=torch.int32)
    a = dict(q=torch.zeros(5, 4, 128, dtype=BF16), k=torch.zeros(6, 2, 128, dtype=BF16),
             v=torch.zeros(6, 2, 128, dtype=BF16), cu_seqlens_q=cu, cu_seqlens_k=cu, scale=0.1)
    a.update(changes)
    return a


def _gather_args(**changes):
    cache = K.new_kv_cache(3, 16, 2, 128, bits=4)
    a = dict(k_cache=cache.k, v_cache=cache.v, slots=torch.zeros(5, dtype=torch.int32), k_scales=cache.k_scales,
             v_scales=cache.v_scales, out_dtype=BF16)
    a.update(changes)
    return a


def _z(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


REFUSED = [
    ("rope_append", _append_args, dict(q=_z(5, 4, 128, dtype=torch.float32)), "q must be float16 or bfloat16"),
    ("rope_append", _append_args, dict(q=_z(5, 4, 128, dtype=F16)), "dtype of its operands"),
    ("rope_append", _append_args, dict(q=_z(5, 3, 128)), "multiple of the 2 key-value heads"),
    ("rope_append", _append_args, dict(q=_z(5, 4, 64)), "q must be a (rows, heads, head_dim)"),
    ("rope_append", _append_args, dict(k=_z(5, 1, 128)), "k must be a (rows, heads, head_dim)"),
    ("rope_append", _append_args, dict(v=_z(4, 2, 128)), "v must be a (rows, heads, head_dim)"),
    ("rope_append", _append_args, dict(v=_z(5, 2, 128, dtype=F16)), "v must have the dtype of q"),
    ("rope_append", _append_args, dict(k=_z(5, 128, 2).transpose(1, 2)), "unit stride"),
    ("rope_append", _append_args, dict(k=_z(5, 2 * 128 + 4)[:, :256].view(5, 2, 128)), "multiples of 8"),
    ("rope_append", _append_args, dict(k=_z(5 * 256 + 8)[4:-4].view(5, 2, 128)), "16-byte aligned"),
    ("rope_append", _append_args, dict(positions=_z(5, dtype=torch.int32)), "positions must be torch.int64"),
    ("rope_append", _append_args, dict(slots=_z(5, dtype=torch.int64)), "slots must be torch.int32"),
    ("rope_append", _append_args, dict(slots=_z(4, dtype=torch.int32)), "slots must have shape (5,), got (4,)"),
    ("rope_append", _append_args, dict(slots=_z(10, dtype=torch.int32)[::2]), "slots must be contiguous"),
    ("rope_append", _append_args, dict(cos_sin=_z(9, 64)), "float32 (positions, rotary_dim)"),
    ("rope_append", _append_args, dict(cos_sin=_z(9, 40, dtype=torch.float32)), "rotary_dim (40)"),
    ("rope_append", _append_args, dict(cos_sin=_z(9, 144, dtype=torch.float32)), "rotary_dim (144)"),
    ("rope_append", _append_args, dict(v_cache=_z(3, 16, 2, 64)), "of the same shape"),
    ("rope_append", _append_args, dict(k_cache=_z(3, 16, 2, 96), v_cache=_z(3, 16, 2, 96)), "64, 128 or 256, got 96"),
    ("rope_append", _append_args, dict(k_cache=_z(0, 16, 2, 128), v_cache=_z(0, 16, 2, 128)), "at least one block"),
    ("rope_append", _append_args, dict(k_cache=_z(3, 2, 16, 128).transpose(1, 2)), "contiguous"),
    ("rope_append", _append_args, dict(k_cache=_z(3 * 16 * 256 + 8)[4:-4].view(3, 16, 2, 128)), "16-byte aligned"),
    ("rope_append", _append_args, dict(k_scales=_z(3, 2, 16, 2, 2, dtype=F16)), "given together"),
    ("rope_append", _append_args, dict(k_cache=_z(3, 16, 2, 128, dtype=torch.uint8)), "uint8 with scales"),
    ("kv_gather", _gather_args, dict(out_dtype=None), "out_dtype of a 4-bit cache"),
    ("kv_gather", _gather_args, dict(out_dtype=torch.float32), "out_dtype of a 4-bit cache"),
    ("kv_gather", _gather_args, dict(k_scales=None, v_scales=None), "with scales"),
    ("kv_gather", _gather_args, dict(k_scales=_z(3, 2, 2, 16, 2, dtype=F16)), "k_scales must be (blocks"),
    ("kv_gather", _gather_args, dict(v_scales=_z(3, 2, 16, 2, 2, dtype=F16)), "v_scales must be (blocks"),
    ("kv_gather", _gather_args, dict(v_scales=_z(3, 2, 2, 16, 2)), "must be float16"),
    ("kv_gather", _gather_args, dict(slots=_z(5, 1, dtype=torch.int32)), "one-dimensional"),
    ("attention_prompt", _prompt_args, dict(q=_z(5, 4, 96)), "head_dim of 64, 128 or 256"),
    ("attention_prompt", _prompt_args, dict(q=_z(5, 512)), "head_dim of 64, 128 or 256"),
    ("attention_prompt", _prompt_args, dict(q=_z(5, 4, 128, dtype=torch.float64)), "float16 or bfloat16"),
    ("attention_prompt", _prompt_args, dict(q=_z(5, 5, 128)), "multiple of the 2"),
    ("attention_prompt", _prompt_args, dict(q=_z(5, 0, 128)), "multiple of the 2"),
    ("attention_prompt", _prompt_args, dict(v=_z(5, 2, 128)), "v must be a (rows"),
    ("attention_prompt", _prompt_args, dict(k=_z(6, 2, 128, dtype=F16)), "k must have the dtype of q"),
    ("attention_prompt", _prompt_args, dict(cu_seqlens_q=_z(0, dtype=torch.int32)), "at least one offset"),
    ("attention_prompt", _prompt_args, dict(cu_seqlens_k=_z(4, dtype=torch.int32)), "cu_seqlens_k must have shape (3,)"),
    ("attention_prompt", _prompt_args, dict(cu_seqlens_q=_z(3, dtype=torch.int64)), "must be torch.int32"),
    ("attention_prompt", _prompt_args, dict(scale=0.0), "scale must be positive and finite, got 0"),
    ("attention_prompt", _prompt_args, dict(scale=float("nan")), "scale must be positive and finite, got nan"),
    ("attention_paged", _paged_args, dict(block_tables=_z(4, 3, dtype=torch.int32)), "int32 (batch, blocks)"),
    ("attention_paged", _paged_args, dict(block_tables=_z(5, 3, dtype=torch.int64)), "int32 (batch, blocks)"),
    ("attention_paged", _paged_args, dict(block_tables=_z(3, 5, dtype=torch.int32).T), "unit stride"),
    ("attention_paged", _paged_args, dict(context_lens=_z(5, 1, dtype=torch.int32)), "context_lens must have shape"),
    ("attention_paged", _paged_args, dict(k_cache=_z(3, 24, 2, 128), v_cache=_z(3, 24, 2, 128)), "multiple of 16"),
    ("attention_paged", _paged_args, dict(scale=-0.5), "got -0.5"),
    ("attention_paged", _paged_args, dict(scale=float("inf")), "got inf"),
]


@pytest.mark.parametrize("op,args,changes,message", REFUSED, ids=[f"{r[0]}-{i}" for i, r in enumerate(REFUSED)])
def test_refusals(monkeypatch, op, args, changes, message):
    """The contract's reasons, on CPU operands (the check of the device left out)."""
    monkeypatch.setattr(A, "_device_reason", lambda *t: None)
    reason = getattr(A, f"{op}_contract_reason")
    assert reason(**args()) is None
    assert message in reason(**args(**changes))


@pytest.mark.gpu
@pytest.mark.parametrize("op,args,changes,message", REFUSED, ids=[f"{r[0]}-{i}" for i, r in enumerate(REFUSED)])
def test_refusals_of_the_ops(op, args, changes, message):
    """The op refuses the same calls in the same words; nothing is launched."""
    print("refusal", op, message, flush=True)
    base = torch.empty(0, device="cuda")

    def put(t):
        if not isinstance(t, torch.Tensor):
            return t
        # The same strides and offset on the GPU.
        whole = torch.empty(t.untyped_storage().nbytes(), dtype=torch.uint8, device=base.device)
        return whole.view(t.dtype).as_strided(t.shape, t.stride(), t.storage_offset())

    call = {k: put(v) for k, v in args(**changes).items()}
    reason = getattr(A, f"{op}_contract_reason")(**call)
    assert message in reason
    with pytest.raises(RuntimeError) as said:
        getattr(K, op)(**call)
    assert f"nanovllm::{op}: {reason}" in str(said.value)
    if op == "rope_append":
        call = {"k_scales": None, "v_scales": None} | call
    with pytest.raises(RuntimeError) as said:
        getattr(A, f"_{op}_op")(**call)
    assert f"nanovllm::{op}: {reason}" in str(said.value)


@pytest.mark.gpu
def test_registration_through_ctypes_gives_the_same_results():
    print("ctypes", flush=True)
    gen = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn((150, h, 128), generator=gen).to(BF16).cuda() for h in (4, 2, 2))
    for bits in (16, 4):
        caches = [K.new_kv_cache(12, 16, 2, 128, bits=bits, device="cuda") for _ in range(2)]
        at = torch.arange(150, device="cuda")
        table, slots = K.rope_table(150, 64, device="cuda"), torch.arange(150, dtype=torch.int32, device="cuda")
        cu = torch.tensor([0, 150], dtype=torch.int32, device="cuda")
        pages = torch.arange(12, dtype=torch.int32, device="cuda")[None]
        results = []
        for cache, (append, gather, prompt, paged) in zip(caches, (
                (K.rope_append, K.kv_gather, K.attention_prompt, K.attention_paged),
                tuple(getattr(A, f"_{op}_op") for op in OPS))):
            a, b = append(q, k, v, at, table, slots, *tuple(cache))
            c, d = gather(cache.k, cache.v, slots, cache.k_scales, cache.v_scales, BF16)
            e = prompt(a, b, v, cu, cu, 0.1)
            f = paged(a[-1:], cache.k, cache.v, pages, cu[1:], 0.1, cache.k_scales, cache.v_scales)
            results.append((a, b, c, d, e, f))
        assert all(torch.equal(x, y) for x, y in zip(*results))


# ---------------------------------------------------------------------------
# The plain torch backend
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_torch_backend_codes_rows_as_the_oracle(dim):
    gen = torch.Generator().manual_seed(dim)
    cache = K.new_kv_cache(3, 16, 2, dim, bits=4)
    k, v = (torch.randn((20, 2, dim), generator=gen).to(BF16) for _ in range(2))
    table, positions = K.rope_table(50, 32), torch.arange(20)
    slots = torch.randperm(48, generator=gen)[:20].to(torch.int32)
    slots[3], slots[7] = -1, 48
    _, turned = K.rope_append_kv(k, k, v, positions, table, slots, cache, backend="torch")
    assert torch.equal(turned, orc.rotate(k, positions.tolist(), table))
    want = [np.zeros(t.shape, t.numpy().dtype) for t in cache]
    for t, s in enumerate(slots.tolist()):
        for h in range(2):
            if 0 <= s < 48:
                orc.write_row(want, s, h, turned[t, h].float().numpy(), v[t, h].float().numpy())
    assert all(np.array_equal(a.numpy(), b) for a, b in zip(cache, want))
    got = K.gather_kv(cache, slots, F16, backend="torch")
    for t, s in enumerate(slots.tolist()):
        for h in range(2):
            rows = orc.read_row(want, s, h)[:2] if 0 <= s < 48 else (np.zeros(dim), np.zeros(dim))
            assert all(torch.equal(g[t, h], torch.from_numpy(r).float().half()) for g, r in zip(got, rows))


@pytest.mark.parametrize("causal", [True, False])
def test_torch_backend_attends_as_the_oracle(causal):
    gen = torch.Generator().manual_seed(1)
    lq, lk = [3, 0, 9, 5], [7, 2, 4, 0]
    q, k, v = (torch.randn((n, h, 64), generator=gen).to(F16) for n, h in ((17, 4), (13, 2), (13, 2)))
    cu = [torch.tensor([0] + list(np.cumsum(x)), dtype=torch.int32) for x in (lq, lk)]
    got = K.prompt_attention(q, k, v, *cu, 0.125, causal, backend="torch")
    a = c = 0
    for n, m in zip(lq, lk):
        qs, ks, vs = q[a:a + n].double(), k[c:c + m].double(), v[c:c + m].double()
        out, w, big = orc.attend(qs, ks, vs, 0.125, m - n if causal else None)
        tol = orc.tolerance(out, torch.einsum("hij,jhd->ihd", w, vs.abs().repeat_interleave(2, 1)), big, F16, 64,
                            p_half_step=2.0 ** -24)
        assert ((got[a:a + n].double() - out).abs() <= tol).all()
        a, c = a + n, c + m


@pytest.mark.parametrize("bits", [16, 4])
def test_layer_decodes_what_it_prefilled(bits):
    """On the torch backend: a prompt in one piece, and in a piece, a chunk and single tokens, give the same states
    (what a 4-bit cache loses aside)."""
    gen = torch.Generator().manual_seed(2)
    layer = PKG.layers.Qwen35Attention(64, 4, 2, 64)
    for p in layer.parameters():
        p.requires_grad_(False)
        p.copy_(torch.randn(p.shape, generator=gen) * 0.1)
    layer.gemm_backend = "torch"
    x, table = torch.randn((40, 64), generator=gen), K.rope_table(64, 32)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    at, slots = torch.arange(40), torch.randperm(48, generator=gen)[:48].to(torch.int32)
    pages = torch.arange(3, dtype=torch.int32).flip(0)[None]
    slots = pages[0][at // 16] * 16 + (at % 16).to(torch.int32)
    cache = K.new_kv_cache(3, 16, 2, 64, bits=bits, dtype=torch.float32)
    whole = layer(x, at, table, cache, slots, cu_seqlens=i32([0, 40]))
    cache = K.new_kv_cache(3, 16, 2, 64, bits=bits, dtype=torch.float32)
    parts = [layer(x[:25], at[:25], table, cache, slots[:25], cu_seqlens=i32([0, 25])),
             layer(x[25:36], at[25:36], table, cache, slots[25:36], cu_seqlens=i32([0, 11]),
                   cu_seqlens_k=i32([0, 36]), context_slots=slots[:36])]
    for t in range(36, 40):
        parts.append(layer(x[t:t + 1], at[t:t + 1], table, cache, slots[t:t + 1], block_tables=pages,
                           context_lens=i32([t + 1])))
    got = torch.cat(parts)
    # fp32 throughout; a 4-bit element is off by up to half of a fifteenth of its group's range.
    assert float((got - whole).norm() / whole.norm()) < (1e-5 if bits == 16 else 0.2)
    with pytest.raises(ValueError, match="block_tables"):
        layer(x, at, table, cache, slots)
    with pytest.raises(ValueError, match="context_slots"):
        layer(x, at, table, cache, slots, cu_seqlens=i32([0, 40]), cu_seqlens_k=i32([0, 40]))


def test_ops_have_no_backward():
    q = torch.zeros((2, 2, 64), dtype=BF16, requires_grad=True)
    cu = torch.tensor([0, 2], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="HIP"):
        K.prompt_attention(q, q, q, cu, cu, 0.1, backend="hip")


def test_new_kv_cache_checks_its_sizes():
    with pytest.raises(ValueError, match="16 or 4 bits"):
        K.new_kv_cache(1, 16, 1, 64, bits=8)
    with pytest.raises(ValueError, match="multiple of 16"):
        K.new_kv_cache(1, 24, 1, 64, bits=4)
    with pytest.raises(ValueError, match="one of 64"):
        K.new_kv_cache(1, 16, 1, 96, bits=4)
