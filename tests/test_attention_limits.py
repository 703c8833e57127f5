"""How large a call of the attention operators may be: what the kernels count in
32 bits is refused on the host, by the C ABI and by the ops' contracts."""
from __future__ import annotations

import ctypes
import importlib

import pytest
import torch

from conftest import PKG

L = PKG._lib
P = 1 << 20        # a device pointer that is never followed


def _cache(block_size=16, kv_heads=1, head_dim=64, bits=16):
    page = block_size * kv_heads * head_dim * 2 if bits == 16 else block_size * kv_heads * head_dim // 2
    scales = block_size * kv_heads * head_dim // 64 * 4 if bits == 4 else 0
    scale_ptr = P if bits == 4 else None
    return ctypes.byref(L.KvCacheStruct(P, P, scale_ptr, scale_ptr, 4, block_size, kv_heads, head_dim, page, page, scales,
                                        scales, bits, L.BF16))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("block_size", [16, 48, 256, 1024])
def test_paged_tables_end_where_the_kernel_counts_to(lib, block_size, bits):
    """The kernel counts tokens in 32 bits and looks up to 2 x 128 + 16 of them past a sequence's end: a table holds at
    most 2^31 - 1024.  (A table may name a page many times, so that needs no cache of the size.)"""
    cache, most = _cache(block_size=block_size, bits=bits), (2 ** 31 - 1024) // block_size
    assert most * block_size + 2 * 128 + 16 < 2 ** 31 - 128
    assert L.attention_paged_workspace_bytes(cache, 1, 1, most) > 0
    for blocks in {most + 1, max(most + 1, (2 ** 31 - 1) // block_size)}:
        assert L.attention_paged_workspace_bytes(cache, 1, 1, blocks) == L.EINVAL
        assert "2^31 - 1024" in L.last_error()
        assert lib.nanovllm_attention_paged(P, cache, P, P, P, 1, 1, blocks, blocks, 0, 0, 0.1, L.BF16, P, 1 << 40,
                                            None) == L.EINVAL
        assert "2^31 - 1024" in L.last_error()


# ---------------------------------------------------------------------------
# The ops' contracts name these limits, so that the backend "auto" falls back
# ---------------------------------------------------------------------------
A = importlib.import_module("inference_systems_amd.kernels.attention")
K = PKG.kernels
BF16 = torch.bfloat16


def _z(shape, dtype=BF16, device="cpu"):
    return torch.zeros(shape, dtype=dtype, device=device)


def _far_rows(rows, heads, dim, stride, device):
    """[rows, heads, dim] whose rows are `stride` elements apart."""
    whole = torch.zeros((rows - 1) * stride + heads * dim, dtype=BF16, device=device)
    return whole.as_strided((rows, heads, dim), (stride, dim, 1))


def _append_call(device, tokens=3, heads=4, dim=128, **changes):
    cache = K.new_kv_cache(3, 16, 2, dim, device=device)
    a = dict(q=_z((1, heads, dim), device=device).expand(tokens, -1, -1),
             k=_z((1, 2, dim), device=device).expand(tokens, -1, -1),
             v=_z((1, 2, dim), device=device).expand(tokens, -1, -1),
             positions=_z(tokens, torch.int64, device), cos_sin=_z((9, 64), torch.float32, device),
             slots=_z(tokens, torch.int32, device), k_cache=cache.k, v_cache=cache.v, k_scales=None, v_scales=None)
    return a | changes


def _gather_call(device, rows=3, **changes):
    cache = K.new_kv_cache(3, 16, 2, 256, device=device)
    return dict(k_cache=cache.k, v_cache=cache.v, slots=_z(rows, torch.int32, device)) | changes


def _prompt_call(device, batch=2, **changes):
    cu = _z(batch + 1, torch.int32, device)
    return dict(q=_z((3, 4, 128), device=device), k=_z((3, 2, 128), device=device), v=_z((3, 2, 128), device=device),
                cu_seqlens_q=cu, cu_seqlens_k=cu, scale=0.1) | changes


def _paged_call(device, batch=3, blocks=3, **changes):
    cache = K.new_kv_cache(3, 16, 2, 128, device=device)
    return dict(q=_z((1, 4, 128), device=device).expand(batch, -1, -1), k_cache=cache.k, v_cache=cache.v,
                block_tables=_z((batch, blocks), torch.int32, device), context_lens=_z(batch, torch.int32, device),
                scale=0.1) | changes


def _big_page(device):
    """One block of a little over 2 GiB (never touched)."""
    return torch.empty((1, 2 ** 22 + 16, 1, 256), dtype=BF16, device=device)


FAR = 2 ** 24
LIMITS = [
    ("rope_append", lambda d: _append_call(d, q=_far_rows(3, 4, 128, FAR, d)), "row stride of q must be below 2^24"),
    ("rope_append", lambda d: _append_call(d, k=_far_rows(3, 2, 128, FAR + 8, d)), "row stride of k must be below 2^24"),
    ("rope_append", lambda d: _append_call(d, v=_far_rows(3, 2, 128, FAR, d)), "row stride of v must be below 2^24"),
    ("rope_append", lambda d: _append_call(d, tokens=2 ** 27), "too many tokens and heads"),
    ("rope_append", lambda d: _append_call(d, tokens=2 ** 28), "tokens times heads below 2^31"),
    ("rope_append", lambda d: _append_call(d, k_cache=_z((1, 16, 2, 128), device=d).expand(3, -1, -1, -1)),
     "not smaller than a page"),
    ("kv_gather", lambda d: _gather_call(d, rows=2 ** 26), "too many rows and heads"),
    ("kv_gather", lambda d: _gather_call(d, v_cache=_z((1, 16, 2, 256), device=d).expand(3, -1, -1, -1)),
     "not smaller than a page"),
    ("kv_gather", lambda d: _gather_call(d, k_cache=_big_page(d), v_cache=_big_page(d)), "smaller than 2 GiB"),
    ("attention_prompt", lambda d: _prompt_call(d, q=_far_rows(3, 4, 128, FAR, d)), "row stride of q"),
    ("attention_prompt", lambda d: _prompt_call(d, v=_far_rows(3, 2, 128, FAR, d)), "row stride of v"),
    ("attention_prompt", lambda d: _prompt_call(d, batch=2 ** 22), "too many sequences, rows and heads"),
    ("attention_paged", lambda d: _paged_call(d, q=_far_rows(3, 4, 128, FAR, d)), "row stride of q"),
    ("attention_paged", lambda d: _paged_call(d, block_tables=_z((1, 3), torch.int32, d).expand(3, -1)),
     "rows of block_tables must not overlap"),
    ("attention_paged", lambda d: _paged_call(d, batch=2 ** 23, blocks=1), "batch, heads and table are too large"),
    ("attention_paged", lambda d: _paged_call(d, k_cache=_z((1, 16, 2, 128), device=d).expand(3, -1, -1, -1)),
     "not smaller than a page"),
]
LIMIT_IDS = [f"{op}-{message.replace(' ', '_')}-{i}" for i, (op, _, message) in enumerate(LIMITS)]


@pytest.mark.parametrize("op,call,message", LIMITS, ids=LIMIT_IDS)
def test_contracts_name_the_limits(monkeypatch, op, call, message):
    monkeypatch.setattr(A, "_device_reason", lambda *t: None)
    assert message in getattr(A, f"{op}_contract_reason")(**call("cpu"))


@pytest.mark.gpu
@pytest.mark.parametrize("op,call,message", LIMITS, ids=LIMIT_IDS)
def test_ops_refuse_in_the_contracts_words(op, call, message):
    print("limit", op, message, flush=True)
    args = call("cuda")
    reason = getattr(A, f"{op}_contract_reason")(**args)
    assert message in reason
    for run in (getattr(K, op), getattr(A, f"_{op}_op")):
        with pytest.raises(RuntimeError) as said:
            run(**args)
        assert f"nanovllm::{op}: {reason}" in str(said.value)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["rope_append", "kv_gather", "big page", "attention_prompt", "attention_paged", "table"])
def test_auto_falls_back(which):
    """Behind the limits the backend "auto" computes what "torch" does; "hip" raises."""
    print("auto", which, flush=True)
    gen, dev = torch.Generator().manual_seed(3), "cuda"
    random = lambda *shape: torch.randn(shape, generator=gen).to(BF16).to(dev)  # noqa: E731
    cache = K.KVCache(random(3, 16, 2, 128), random(3, 16, 2, 128))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    q, k = random(2, 4, 128), random(2, 2, 128)
    far = _far_rows(2, 4, 128, FAR, dev)
    far.copy_(q)
    table, at = K.rope_table(9, 64, device=dev), torch.arange(2, device=dev)

    def append(backend, q=far):
        mine = K.KVCache(cache.k.clone(), cache.v.clone())
        return *K.rope_append_kv(q, k, k, at, table, i32([4, 20]), mine, backend=backend), *mine[:2]

    def gather(backend):
        same = cache.k[:1].expand(3, -1, -1, -1)
        return K.gather_kv(K.KVCache(same, same), i32([3, 40, -1]), backend=backend)

    def big(backend):
        page = _big_page(dev)
        page[0, :4], page[0, -4:] = random(4, 1, 256), 1.0
        return K.gather_kv(K.KVCache(page, page), i32([2, 2 ** 22 + 15]), backend=backend)

    def prompt(backend):
        return (K.prompt_attention(far, k, k, i32([0, 2]), i32([0, 2]), 0.1, backend=backend),)

    def paged(backend, q=far, tables=i32([[0, 1], [2, 0]])):
        return (K.paged_attention(q, cache, tables, i32([20, 7]), 0.1, backend=backend),)

    run = {"rope_append": append, "kv_gather": gather, "big page": big, "attention_prompt": prompt,
           "attention_paged": paged, "table": lambda b: paged(b, q, i32([[2, 1]]).expand(2, -1))}[which]
    seed = gen.get_state()
    want = run("torch")
    gen.set_state(seed)
    assert all(torch.equal(a, b) for a, b in zip(run("auto"), want))
    with pytest.raises(RuntimeError, match="unavailable"):
        run("hip")
