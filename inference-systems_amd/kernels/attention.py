"""The operators between the projections of a Qwen3.5 gated-attention layer,
as PyTorch custom ops (nanovllm/models/qwen3_5.py:81-96,
nanovllm/layers/attention.py, nanovllm/layers/rotary_embedding.py).

    rope_append(q[T, H, D], k[T, KV, D], v[T, KV, D], positions[T], cos_sin,
                slots[T], k_cache, v_cache, k_scales=None, v_scales=None)
            -> (q rotated, k rotated)
        Rotates the first R channels of queries and keys (fp32, rounded once;
        row p of ``cos_sin`` [P, R] holds cosines and sines of position p) and
        writes keys and values to their slots of a paged cache, in place.  A
        negative slot, or one behind the cache, takes none (padding); the
        slots of one call are distinct.  A position outside the table turns
        by NaN.

    kv_gather(k_cache, v_cache, slots[N], k_scales=None, v_scales=None,
              out_dtype=None) -> (k[N, KV, D], v[N, KV, D])
        Cached rows as packed keys and values, zeros for a slot outside the
        cache.  With it a chunk of a prompt attends to its cached prefix.

    attention_prompt(q[Tq, H, D], k[Tk, KV, D], v, cu_seqlens_q, cu_seqlens_k,
                     scale, causal=True) -> out[Tq, H, D]
        Attention of packed sequences: int32 offsets of their rows, from 0 and
        not decreasing.  Query i of a sequence sees keys up to
        i + (its keys - its queries).  A row with no key to see is 0, and so
        are rows behind the last sequence.

    attention_paged(q[B, H, D], k_cache, v_cache, block_tables[B, N],
                    context_lens[B], scale, k_scales=None, v_scales=None)
            -> out[B, H, D]
        One query token per sequence over its first context_lens[b] cached
        tokens.  A page number outside the cache, or a length behind the
        table, makes a sequence's output NaN.

Scores, softmax statistics and sums are held in 32 bits.  Weights are rounded
to q's type before they multiply the values (their total is of the rounded
ones); next to 4-bit values weights, weights times scales and the middle of a
group are rounded to float16.  Errors are up to 1.5 times those of a softmax
that stays in 32 bits.

Types: float16 or bfloat16, D of 64, 128 or 256, H a multiple of KV.  q, k and
v may be strided views (a column range of one projection) with unit stride in
the last dimension, and strides that are multiples of 8, that of rows below
2^24.  ``positions`` is int64, the other index tensors int32,
``cos_sin`` float32.  A block table holds at most 2^31 - 1024 tokens.

A paged cache (``new_kv_cache``) holds 16-bit elements, [blocks, block_size,
KV, D] for keys and for values, or 4-bit codes with a float16 scale and minimum
per token and 64 channels (k_scales, v_scales given); an element of the latter
stands for code * scale + minimum.  include/nanovllm_attention.h gives the
layout.  A block may be a slice of a larger allocation (any stride between
blocks).

Same conventions as ``nanovllm::gemm``.  The ops have no backward.
``rope_append_kv``, ``gather_kv``, ``prompt_attention`` and ``paged_attention``
add the ``torch | hip | auto`` switch, with plain torch as the ``torch`` backend.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from .. import _lib
from .gemm import _CODE, default_backend, register_op, run_hip, validate_gemm_backend

_HALF = (torch.float16, torch.bfloat16)
HEAD_DIMS = (64, 128, 256)
GROUP = 64       # channels that share a 4-bit scale and minimum
ROW_STRIDES = 1 << 24      # row strides of operands, in elements, are below this


class KVCache(NamedTuple):
    """A layer's paged cache; the scales are None in 16 bits."""

    k: torch.Tensor
    v: torch.Tensor
    k_scales: Optional[torch.Tensor] = None
    v_scales: Optional[torch.Tensor] = None


def new_kv_cache(num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int, *, bits: int = 16,
                 dtype: torch.dtype = torch.bfloat16, device=None) -> KVCache:
    """A zeroed cache of 16-bit elements of ``dtype``, or of 4-bit codes."""
    if bits == 16:
        shape = (num_blocks, block_size, num_kv_heads, head_dim)
        return KVCache(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))
    if bits != 4:
        raise ValueError(f"a cache holds 16 or 4 bits, got {bits}")
    if block_size % 16 or head_dim % GROUP:
        raise ValueError("a 4-bit cache needs a block_size that is a multiple of 16 and a head_dim that is one of 64")
    codes = (num_blocks, num_kv_heads, block_size, head_dim // 2)
    groups = head_dim // GROUP
    return KVCache(torch.zeros(codes, dtype=torch.uint8, device=device),
                   torch.zeros(codes, dtype=torch.uint8, device=device),
                   torch.zeros((num_blocks, num_kv_heads, block_size, groups, 2), dtype=torch.float16, device=device),
                   torch.zeros((num_blocks, num_kv_heads, groups, block_size, 2), dtype=torch.float16, device=device))


def rope_table(positions: int, rotary_dim: int, theta: float = 10000.0, device=None) -> torch.Tensor:
    """[positions, rotary_dim] float32 cosines and sines, the angles taken in float64."""
    rate = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * rate
    return torch.cat((angle.cos(), angle.sin()), -1).float()


# ---------------------------------------------------------------------------
# Contracts
# ---------------------------------------------------------------------------
def _blocks_contiguous(t: torch.Tensor) -> bool:
    """Every block (dimension 0) is contiguous."""
    expected = 1
    for size, stride in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
        if size != 1 and stride != expected:
            return False
        expected *= size
    return True


def _block_bytes(t: torch.Tensor) -> int:
    """Bytes between blocks."""
    elements = t.stride(0) if t.shape[0] > 1 else t.numel()
    return elements * t.element_size()


def _cache_reason(k_cache, v_cache, k_scales, v_scales, dtype) -> Optional[str]:
    """Why the ops cannot take this cache next to operands of ``dtype`` (None: any)."""
    if (k_scales is None) != (v_scales is None):
        return "k_scales and v_scales must be given together"
    if k_scales is None:
        if k_cache.dtype not in _HALF or v_cache.dtype != k_cache.dtype:
            return "k_cache and v_cache must be float16 or bfloat16 of the same dtype, or uint8 with scales"
        if dtype is not None and k_cache.dtype != dtype:
            return "a 16-bit cache must have the dtype of its operands"
        if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
            return "k_cache and v_cache must be (blocks, block_size, kv_heads, head_dim) tensors of the same shape"
        blocks, size, heads, dim = k_cache.shape
        tensors = (k_cache, v_cache)
    else:
        if k_cache.dtype != torch.uint8 or v_cache.dtype != torch.uint8:
            return "k_cache and v_cache must be uint8 with scales"
        if k_scales.dtype != torch.float16 or v_scales.dtype != torch.float16:
            return "k_scales and v_scales must be float16"
        if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
            return "k_cache and v_cache must be (blocks, kv_heads, block_size, head_dim / 2) tensors of the same shape"
        blocks, heads, size, dim = k_cache.shape
        dim *= 2
        groups = dim // GROUP
        if tuple(k_scales.shape) != (blocks, heads, size, groups, 2):
            return "k_scales must be (blocks, kv_heads, block_size, head_dim / 64, 2)"
        if tuple(v_scales.shape) != (blocks, heads, groups, size, 2):
            return "v_scales must be (blocks, kv_heads, head_dim / 64, block_size, 2)"
        tensors = (k_cache, v_cache, k_scales, v_scales)
    if dim not in HEAD_DIMS:
        return f"head_dim must be 64, 128 or 256, got {dim}"
    if blocks < 1 or size < 1 or heads < 1:
        return "a cache must have at least one block, token and head"
    if k_scales is not None and size % 16:
        return "block_size of a 4-bit cache must be a multiple of 16"
    if not all(_blocks_contiguous(t) for t in tensors):
        return "the blocks of a cache must be contiguous"
    if any(t.data_ptr() % 16 or _block_bytes(t) % 16 for t in tensors):
        return "the blocks of a cache must be 16-byte aligned"
    return None


def _geometry(k_cache, k_scales):
    """(blocks, block_size, kv_heads, head_dim)."""
    if k_scales is None:
        return tuple(k_cache.shape)
    blocks, heads, size, half = k_cache.shape
    return blocks, size, heads, 2 * half


def _rows_reason(name: str, t: torch.Tensor, dtype, heads: Optional[int], dim: int, rows: Optional[int] = None):
    """Why ``t`` is no [rows, heads, dim] operand."""
    if t.dtype != dtype:
        return f"{name} must have the dtype of q"
    if t.dim() != 3 or t.shape[2] != dim or (heads is not None and t.shape[1] != heads) or (
            rows is not None and t.shape[0] != rows):
        return f"{name} must be a (rows, heads, head_dim) tensor that fits the others, got {tuple(t.shape)}"
    if t.stride(2) != 1:
        return f"{name} must have unit stride in its last dimension"
    if any(x % 8 for x in _strides(t)):
        return f"the strides of {name} must be multiples of 8"
    if _strides(t)[0] >= ROW_STRIDES:
        return f"the row stride of {name} must be below 2^24"
    if t.numel() and t.data_ptr() % 16:
        return f"{name} must be 16-byte aligned"
    return None


def _strides(t: torch.Tensor):
    """Element strides of rows and heads; 0 where there is but one."""
    return tuple(t.stride(i) if t.shape[i] > 1 else 0 for i in range(2))


def _index_reason(name: str, t: torch.Tensor, dtype, shape) -> Optional[str]:
    if t.dtype != dtype:
        return f"{name} must be {dtype}"
    if tuple(t.shape) != tuple(shape):
        return f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}"
    if not t.is_contiguous():
        return f"{name} must be contiguous"
    return None


def _device_reason(*tensors) -> Optional[str]:
    tensors = [t for t in tensors if t is not None]
    if not all(t.is_cuda for t in tensors):
        return "all operands must be CUDA (HIP) tensors"
    if len({t.device for t in tensors}) != 1:
        return "all operands must be on the same device"
    return None


def _heads_reason(q, kv_heads: int) -> Optional[str]:
    if q.shape[1] < 1 or q.shape[1] % kv_heads:
        return f"the heads of q ({q.shape[1]}) must be a positive multiple of the {kv_heads} key-value heads"
    return None


def _sizes_reason(op: str, rc: int) -> Optional[str]:
    """The library's words for sizes it refuses (``rc`` of its check or workspace function)."""
    return None if rc >= 0 else _lib.last_error().removeprefix(f"{op}: ")


def rope_append_contract_reason(q, k, v, positions, cos_sin, slots, k_cache, v_cache, k_scales=None,
                                v_scales=None) -> Optional[str]:
    """Why rope_append cannot take these inputs, or None if it can."""
    reason = _device_reason(q, k, v, positions, cos_sin, slots, k_cache, v_cache, k_scales, v_scales)
    if reason is None and q.dtype not in _HALF:
        reason = "q must be float16 or bfloat16"
    reason = reason or _cache_reason(k_cache, v_cache, k_scales, v_scales, q.dtype)
    if reason is not None:
        return reason
    _, _, heads, dim = _geometry(k_cache, k_scales)
    reason = (_rows_reason("q", q, q.dtype, None, dim) or _heads_reason(q, heads)
              or _rows_reason("k", k, q.dtype, heads, dim, q.shape[0])
              or _rows_reason("v", v, q.dtype, heads, dim, q.shape[0])
              or _index_reason("positions", positions, torch.int64, (q.shape[0],))
              or _index_reason("slots", slots, torch.int32, (q.shape[0],)))
    if reason is not None:
        return reason
    if cos_sin.dtype != torch.float32 or cos_sin.dim() != 2 or not cos_sin.is_contiguous() or cos_sin.shape[0] < 1:
        return "cos_sin must be a contiguous float32 (positions, rotary_dim) tensor"
    rotary = cos_sin.shape[1]
    if rotary < 16 or rotary % 16 or rotary > dim:
        return f"rotary_dim ({rotary}) must be a multiple of 16 from 16 to head_dim ({dim})"
    cache = _cache_struct(k_cache, v_cache, k_scales, v_scales, q.dtype)
    return _sizes_reason("rope_append", _lib.rope_append_check(cache, q.shape[0], q.shape[1]))


def kv_gather_contract_reason(k_cache, v_cache, slots, k_scales=None, v_scales=None,
                              out_dtype: Optional[torch.dtype] = None) -> Optional[str]:
    """Why kv_gather cannot take these inputs, or None if it can."""
    reason = (_device_reason(k_cache, v_cache, slots, k_scales, v_scales)
              or _cache_reason(k_cache, v_cache, k_scales, v_scales, None))
    if reason is not None:
        return reason
    if k_scales is None and out_dtype not in (None, k_cache.dtype):
        return "out_dtype of a 16-bit cache must be its dtype"
    if k_scales is not None and out_dtype not in _HALF:
        return "out_dtype of a 4-bit cache must be float16 or bfloat16"
    if slots.dim() != 1:
        return "slots must be one-dimensional"
    reason = _index_reason("slots", slots, torch.int32, slots.shape)
    if reason is not None:
        return reason
    cache = _cache_struct(k_cache, v_cache, k_scales, v_scales, k_cache.dtype if out_dtype is None else out_dtype)
    return _sizes_reason("kv_gather", _lib.kv_gather_check(cache, slots.shape[0]))


def attention_prompt_contract_reason(q, k, v, cu_seqlens_q, cu_seqlens_k, scale, causal=True) -> Optional[str]:
    """Why attention_prompt cannot take these inputs, or None if it can."""
    reason = _device_reason(q, k, v, cu_seqlens_q, cu_seqlens_k)
    if reason is not None:
        return reason
    if q.dtype not in _HALF:
        return "q must be float16 or bfloat16"
    if q.dim() != 3 or k.dim() != 3 or q.shape[2] not in HEAD_DIMS:
        return "q and k must be (rows, heads, head_dim) tensors with a head_dim of 64, 128 or 256"
    if k.shape[1] < 1:
        return "k must have at least one head"
    reason = (_rows_reason("q", q, q.dtype, None, q.shape[2]) or _heads_reason(q, k.shape[1])
              or _rows_reason("k", k, q.dtype, None, q.shape[2])
              or _rows_reason("v", v, q.dtype, k.shape[1], q.shape[2], k.shape[0]))
    if reason is not None:
        return reason
    if cu_seqlens_q.dim() != 1 or cu_seqlens_q.shape[0] < 1:
        return "cu_seqlens_q must be one-dimensional with at least one offset"
    reason = (_index_reason("cu_seqlens_q", cu_seqlens_q, torch.int32, cu_seqlens_q.shape)
              or _index_reason("cu_seqlens_k", cu_seqlens_k, torch.int32, cu_seqlens_q.shape)
              or _scale_reason(scale))
    return reason or _sizes_reason("attention_prompt", _lib.attention_prompt_workspace_bytes(
        *_prompt_sizes(q, k, cu_seqlens_q), _CODE[q.dtype]))


def _prompt_sizes(q, k, cu_seqlens_q):
    """(batch, q_rows, k_rows, heads, kv_heads, head_dim)."""
    return cu_seqlens_q.shape[0] - 1, q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2]


def _scale_reason(scale: float) -> Optional[str]:
    if not 1e-37 < scale < 1e38:
        return f"scale must be positive and finite, got {scale:g}"
    return None


def attention_paged_contract_reason(q, k_cache, v_cache, block_tables, context_lens, scale, k_scales=None,
                                    v_scales=None) -> Optional[str]:
    """Why attention_paged cannot take these inputs, or None if it can."""
    reason = _device_reason(q, k_cache, v_cache, block_tables, context_lens, k_scales, v_scales)
    if reason is None and q.dtype not in _HALF:
        reason = "q must be float16 or bfloat16"
    reason = reason or _cache_reason(k_cache, v_cache, k_scales, v_scales, q.dtype)
    if reason is not None:
        return reason
    _, size, heads, dim = _geometry(k_cache, k_scales)
    reason = _rows_reason("q", q, q.dtype, None, dim) or _heads_reason(q, heads)
    if reason is not None:
        return reason
    if size % 16:
        return f"block_size ({size}) must be a multiple of 16"
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.shape[0] != q.shape[0]:
        return "block_tables must be an int32 (batch, blocks) tensor"
    if block_tables.shape[1] > 1 and block_tables.stride(1) != 1:
        return "block_tables must have unit stride in its last dimension"
    if _table_stride(block_tables) < block_tables.shape[1]:
        return "the rows of block_tables must not overlap"
    reason = _index_reason("context_lens", context_lens, torch.int32, (q.shape[0],)) or _scale_reason(scale)
    if reason is not None:
        return reason
    cache = _cache_struct(k_cache, v_cache, k_scales, v_scales, q.dtype)
    return _sizes_reason("attention_paged", _lib.attention_paged_workspace_bytes(cache, *q.shape[:2],
                                                                                 block_tables.shape[1]))


def _table_stride(block_tables) -> int:
    """Entries between rows of a block table."""
    batch, blocks = block_tables.shape
    return block_tables.stride(0) if batch > 1 and blocks else blocks


# ---------------------------------------------------------------------------
# Launches
# ---------------------------------------------------------------------------
def _cache_struct(k_cache, v_cache, k_scales, v_scales, dtype):
    blocks, size, heads, dim = _geometry(k_cache, k_scales)
    scales = [t.data_ptr() if t is not None else None for t in (k_scales, v_scales)]
    strides = [_block_bytes(t) if t is not None else 0 for t in (k_cache, v_cache, k_scales, v_scales)]
    return ctypes.byref(_lib.KvCacheStruct(k_cache.data_ptr(), v_cache.data_ptr(), *scales, blocks, size, heads, dim,
                                           *strides, 16 if k_scales is None else 4, _CODE[dtype]))


def _refuse(op: str, reason: Optional[str]) -> None:
    if reason is not None:
        raise RuntimeError(f"nanovllm::{op}: {reason}")


def _rope_append_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                    slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    k_scales: Optional[torch.Tensor],
                    v_scales: Optional[torch.Tensor]) -> tuple[torch.Tensor, torch.Tensor]:
    # No defaults: a custom_op's written operands are all passed.
    _refuse("rope_append", rope_append_contract_reason(q, k, v, positions, cos_sin, slots, k_cache, v_cache, k_scales,
                                                       v_scales))
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    if q.shape[0]:
        with torch.cuda.device(q.device):
            _lib.rope_append_raw(q.data_ptr(), k.data_ptr(), v.data_ptr(), positions.data_ptr(), cos_sin.data_ptr(),
                                 slots.data_ptr(), q_out.data_ptr(), k_out.data_ptr(),
                                 _cache_struct(k_cache, v_cache, k_scales, v_scales, q.dtype), q.shape[0], q.shape[1],
                                 *_strides(q), *_strides(k), *_strides(v), cos_sin.shape[0], cos_sin.shape[1],
                                 torch.cuda.current_stream(q.device).cuda_stream)
    return q_out, k_out


def _rope_append_fake(q, k, v, positions, cos_sin, slots, k_cache, v_cache, k_scales=None, v_scales=None):
    torch._check(q.dim() == 3 and k.dim() == 3)
    return q.new_empty(q.shape), k.new_empty(k.shape)


def _kv_gather_op(k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
                  k_scales: Optional[torch.Tensor] = None, v_scales: Optional[torch.Tensor] = None,
                  out_dtype: Optional[torch.dtype] = None) -> tuple[torch.Tensor, torch.Tensor]:
    _refuse("kv_gather", kv_gather_contract_reason(k_cache, v_cache, slots, k_scales, v_scales, out_dtype))
    dtype = k_cache.dtype if out_dtype is None else out_dtype
    _, _, heads, dim = _geometry(k_cache, k_scales)
    k, v = (torch.empty((slots.shape[0], heads, dim), dtype=dtype, device=slots.device) for _ in range(2))
    if slots.shape[0]:
        with torch.cuda.device(slots.device):
            _lib.kv_gather_raw(_cache_struct(k_cache, v_cache, k_scales, v_scales, dtype), slots.data_ptr(),
                               slots.shape[0], k.data_ptr(), v.data_ptr(), _CODE[dtype],
                               torch.cuda.current_stream(slots.device).cuda_stream)
    return k, v


def _kv_gather_fake(k_cache, v_cache, slots, k_scales=None, v_scales=None, out_dtype=None):
    torch._check(k_cache.dim() == 4 and slots.dim() == 1)
    dtype = k_cache.dtype if out_dtype is None else out_dtype
    _, _, heads, dim = _geometry(k_cache, k_scales)
    return tuple(k_cache.new_empty((slots.shape[0], heads, dim), dtype=dtype) for _ in range(2))


def _attention_prompt_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                         cu_seqlens_k: torch.Tensor, scale: float, causal: bool = True) -> torch.Tensor:
    _refuse("attention_prompt", attention_prompt_contract_reason(q, k, v, cu_seqlens_q, cu_seqlens_k, scale, causal))
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if q.shape[0]:
        sizes = _prompt_sizes(q, k, cu_seqlens_q)
        need = _lib.attention_prompt_workspace_bytes(*sizes, _CODE[q.dtype])
        _lib.check(need if need < 0 else _lib.OK, "nanovllm_attention_prompt_workspace_bytes")
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=q.device)
        with torch.cuda.device(q.device):
            _lib.attention_prompt_raw(q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_seqlens_q.data_ptr(),
                                      cu_seqlens_k.data_ptr(), out.data_ptr(), *sizes, *_strides(q), *_strides(k),
                                      *_strides(v), float(scale), causal, _CODE[q.dtype], workspace.data_ptr(), need,
                                      torch.cuda.current_stream(q.device).cuda_stream)
    return out


def _attention_prompt_fake(q, k, v, cu_seqlens_q, cu_seqlens_k, scale, causal=True):
    torch._check(q.dim() == 3 and k.dim() == 3)
    return q.new_empty(q.shape)


def _attention_paged_op(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                        context_lens: torch.Tensor, scale: float, k_scales: Optional[torch.Tensor] = None,
                        v_scales: Optional[torch.Tensor] = None) -> torch.Tensor:
    _refuse("attention_paged", attention_paged_contract_reason(q, k_cache, v_cache, block_tables, context_lens, scale,
                                                               k_scales, v_scales))
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    batch, heads, _ = q.shape
    if batch:
        cache = _cache_struct(k_cache, v_cache, k_scales, v_scales, q.dtype)
        blocks = block_tables.shape[1]
        need = _lib.attention_paged_workspace_bytes(cache, batch, heads, blocks)
        _lib.check(need if need < 0 else _lib.OK, "nanovllm_attention_paged_workspace_bytes")
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=q.device)
        with torch.cuda.device(q.device):
            _lib.attention_paged_raw(q.data_ptr(), cache, block_tables.data_ptr(), context_lens.data_ptr(),
                                     out.data_ptr(), batch, heads, blocks, _table_stride(block_tables), *_strides(q),
                                     float(scale), _CODE[q.dtype], workspace.data_ptr(), need,
                                     torch.cuda.current_stream(q.device).cuda_stream)
    return out


def _attention_paged_fake(q, k_cache, v_cache, block_tables, context_lens, scale, k_scales=None, v_scales=None):
    torch._check(q.dim() == 3 and k_cache.dim() == 4)
    return q.new_empty(q.shape)


register_op("rope_append", _rope_append_op, _rope_append_fake, ("k_cache", "v_cache", "k_scales", "v_scales"))
register_op("kv_gather", _kv_gather_op, _kv_gather_fake)
register_op("attention_prompt", _attention_prompt_op, _attention_prompt_fake)
register_op("attention_paged", _attention_paged_op, _attention_paged_fake)


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                k_scales: Optional[torch.Tensor] = None,
                v_scales: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(q rotated, k rotated); the rotated keys and the values go to their slots of the cache."""
    return torch.ops.nanovllm.rope_append(q, k, v, positions, cos_sin, slots, k_cache, v_cache, k_scales, v_scales)


def kv_gather(k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
              k_scales: Optional[torch.Tensor] = None, v_scales: Optional[torch.Tensor] = None,
              out_dtype: Optional[torch.dtype] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows ``slots`` of the cache as packed keys and values."""
    return torch.ops.nanovllm.kv_gather(k_cache, v_cache, slots, k_scales, v_scales, out_dtype)


def attention_prompt(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                     cu_seqlens_k: torch.Tensor, scale: float, causal: bool = True) -> torch.Tensor:
    """softmax(scale q k^T) v of packed sequences with grouped heads."""
    return torch.ops.nanovllm.attention_prompt(q, k, v, cu_seqlens_q, cu_seqlens_k, float(scale), bool(causal))


def attention_paged(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                    context_lens: torch.Tensor, scale: float, k_scales: Optional[torch.Tensor] = None,
                    v_scales: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale q k^T) v of one token per sequence over its pages."""
    return torch.ops.nanovllm.attention_paged(q, k_cache, v_cache, block_tables, context_lens, float(scale), k_scales,
                                              v_scales)


# ---------------------------------------------------------------------------
# Backend switch and the plain compositions
# ---------------------------------------------------------------------------
_KEY_SHIFT = [4 * (j // 2) + 16 * (j % 2) for j in range(8)]     # of channel j in a key's word


def _take_turns(words: torch.Tensor, groups: int) -> torch.Tensor:
    """Words of a row in channel order -> as a 4-bit cache holds them, those
    of two groups two by two."""
    pairs = words.shape[-1] // groups // 2
    return words.unflatten(-1, (-1, min(2, groups), pairs, 2)).transpose(-3, -2).flatten(-4)


def _channel_order(words: torch.Tensor, groups: int) -> torch.Tensor:
    pairs = words.shape[-1] // groups // 2
    return words.unflatten(-1, (-1, pairs, min(2, groups), 2)).transpose(-3, -2).flatten(-4)


def _quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes [T, heads, dim] and float16 (scale, minimum) [T, heads, dim / 64, 2] of rows."""
    g = x.float().clamp(-65504.0, 65504.0).unflatten(-1, (-1, GROUP))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s, m = ((high - low) / 15).half(), low.half()
    # Code 15 stays in float16's range: the scale below one that was rounded up past it.
    s = torch.where(15 * s.float() + m.float() > 65504.0, (s.view(torch.int16) - 1).view(torch.float16), s)
    codes = ((g - m.float()) / s.float()).round().clamp(0, 15)
    codes = torch.where(s > 0, codes, 0.0).to(torch.int32)
    return codes.flatten(-2), torch.cat((s, m), -1)


def _torch_store(cache: KVCache, slots: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
    blocks, size, heads, dim = _geometry(cache.k, cache.k_scales)
    kept = (slots >= 0) & (slots < blocks * size)
    slots, k, v = slots[kept].long(), k[kept], v[kept]
    block, row = slots // size, slots % size
    if cache.k_scales is None:
        cache.k[block, row], cache.v[block, row] = k, v
        return
    codes, scales = _quantise(k)
    shift = torch.tensor(_KEY_SHIFT, device=k.device)
    words = _take_turns((codes.long().unflatten(-1, (-1, 8)) << shift).sum(-1), dim // GROUP)
    byte = (words[..., None] >> (8 * torch.arange(4, device=k.device))) & 255
    cache.k[block, :, row] = byte.flatten(-2).to(torch.uint8)
    cache.k_scales[block, :, row] = scales
    codes, scales = _quantise(v)
    pair = codes.unflatten(-1, (-1, 2))
    byte = _take_turns(pair[..., 0] | pair[..., 1] << 4, dim // GROUP).to(torch.uint8)
    cache.v.view(blocks, heads, size // 4, dim // 2, 4)[block, :, row // 4, :, row % 4] = byte
    cache.v_scales[block, :, :, row] = scales


def _torch_rows(cache: KVCache, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """fp32 rows [..., kv_heads, dim] of valid slots."""
    blocks, size, heads, dim = _geometry(cache.k, cache.k_scales)
    slots = slots.long()
    block, row = slots // size, slots % size
    if cache.k_scales is None:
        return cache.k[block, row].float(), cache.v[block, row].float()
    byte = cache.k[block, :, row].to(torch.int64).unflatten(-1, (-1, 4))
    word = (byte << (8 * torch.arange(4, device=byte.device))).sum(-1)
    word = _channel_order(word, dim // GROUP)
    k = ((word[..., None] >> torch.tensor(_KEY_SHIFT, device=word.device)) & 15).flatten(-2)
    byte = cache.v.view(blocks, heads, size // 4, dim // 2, 4)[block, :, row // 4, :, row % 4]
    byte = _channel_order(byte, dim // GROUP)
    v = torch.stack((byte & 15, byte >> 4), -1).flatten(-2)
    pairs = (cache.k_scales[block, :, row].float(), cache.v_scales[block, :, :, row].float())
    k, v = ((c.float().unflatten(-1, (-1, GROUP)) * p[..., :1] + p[..., 1:]).flatten(-2)
            for c, p in zip((k, v), pairs))
    return k, v


def _torch_rope_append(q, k, v, positions, cos_sin, slots, k_cache, v_cache, k_scales=None, v_scales=None):
    half = cos_sin.shape[1] // 2
    known = (positions >= 0) & (positions < cos_sin.shape[0])
    turn = torch.where(known[:, None], cos_sin[positions.clamp(0, cos_sin.shape[0] - 1)], torch.nan)[:, None]
    cos, sin = turn[..., :half], turn[..., half:]

    def rotate(x):
        x1, x2, rest = x[..., :half].float(), x[..., half:2 * half].float(), x[..., 2 * half:].float()
        return torch.cat((x1 * cos - x2 * sin, x2 * cos + x1 * sin, rest), -1).to(x.dtype)

    q, k = rotate(q), rotate(k)
    _torch_store(KVCache(k_cache, v_cache, k_scales, v_scales), slots, k, v)
    return q, k


def _torch_kv_gather(k_cache, v_cache, slots, k_scales=None, v_scales=None, out_dtype=None):
    blocks, size, _, _ = _geometry(k_cache, k_scales)
    dtype = k_cache.dtype if out_dtype is None else out_dtype
    there = (slots >= 0) & (slots < blocks * size)
    rows = _torch_rows(KVCache(k_cache, v_cache, k_scales, v_scales), torch.where(there, slots, 0))
    return tuple(torch.where(there[:, None, None], x, 0.0).to(dtype) for x in rows)


def _torch_attend(q, k, v, scale, first):
    """fp32 q [m, heads, dim] over k, v [n, kv_heads, dim]; row i sees keys up to first + i (None: all)."""
    group = q.shape[1] // k.shape[1]
    k, v = (x.repeat_interleave(group, 1).transpose(0, 1).contiguous() for x in (k, v))
    m, n = q.shape[0], k.shape[1]
    last = torch.full((m,), n - 1, device=q.device) if first is None else first + torch.arange(m, device=q.device)
    hidden = torch.arange(n, device=q.device) > last[:, None]
    s = torch.matmul(q.transpose(0, 1).contiguous(), k.transpose(1, 2).contiguous()) * scale
    s = s.masked_fill(hidden, -torch.inf)
    top = s.amax(-1, keepdim=True) if n else s.new_zeros((*s.shape[:2], 1))
    p = torch.exp(s - torch.where(top == -torch.inf, 0.0, top))
    # Values that are not finite only reach the rows that see them (a product would: 0 x infinity).
    finite = torch.isfinite(v)
    o = torch.matmul(p, torch.where(finite, v, 0.0))
    for j in (~finite).any(-1).any(0).nonzero().flatten().tolist():
        rows = slice(0 if first is None else max(0, j - first), None)
        o[:, rows] += p[:, rows, j:j + 1] * torch.where(finite[:, j], 0.0, v[:, j])[:, None]
    # A row that sees no key is 0; one whose every score is -infinity is 0 / 0.
    return (o / torch.where(hidden.all(-1)[:, None], 1.0, p.sum(-1, keepdim=True))).transpose(0, 1)


def _torch_attention_prompt(q, k, v, cu_seqlens_q, cu_seqlens_k, scale, causal=True):
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    cu_q, cu_k = cu_seqlens_q.tolist(), cu_seqlens_k.tolist()
    for q0, q1, k0, k1 in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
        first = (k1 - k0) - (q1 - q0) if causal else None
        out[q0:q1] = _torch_attend(q[q0:q1].float(), k[k0:k1].float(), v[k0:k1].float(), scale, first).to(q.dtype)
    return out


def _torch_attention_paged(q, k_cache, v_cache, block_tables, context_lens, scale, k_scales=None, v_scales=None):
    cache = KVCache(k_cache, v_cache, k_scales, v_scales)
    blocks, size, _, _ = _geometry(k_cache, k_scales)
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    for b, n in enumerate(context_lens.tolist()):
        pages = block_tables[b, :-(-max(n, 0) // size)].long()
        if n > block_tables.shape[1] * size or ((pages < 0) | (pages >= blocks)).any():
            out[b] = torch.nan
            continue
        at = torch.arange(max(n, 0), device=q.device)
        k, v = _torch_rows(cache, pages[at // size] * size + at % size)
        out[b] = _torch_attend(q[b:b + 1].float(), k, v, scale, None)[0].to(q.dtype)
    return out


def _switch(op, plain, reason, backend: Optional[str], *args):
    backend = validate_gemm_backend(backend) if backend is not None else default_backend()
    if backend == "hip":
        return run_hip(op, reason, *args)
    if backend == "auto" and all(t.is_cuda for t in args if isinstance(t, torch.Tensor)):
        # The op checks its contract itself, before it launches or writes anything.
        try:
            return op(*args)
        except RuntimeError:
            if reason(*args) is None:
                raise
    return plain(*args)


def rope_append_kv(q, k, v, positions, cos_sin, slots, cache: KVCache, *, backend: Optional[str] = None):
    """rope_append with the backend switch of ``linear``."""
    return _switch(rope_append, _torch_rope_append, rope_append_contract_reason, backend, q, k, v, positions, cos_sin,
                   slots, *cache)


def gather_kv(cache: KVCache, slots, out_dtype: Optional[torch.dtype] = None, *, backend: Optional[str] = None):
    """kv_gather with the backend switch of ``linear``."""
    return _switch(kv_gather, _torch_kv_gather, kv_gather_contract_reason, backend, cache.k, cache.v, slots,
                   cache.k_scales, cache.v_scales, out_dtype)


def prompt_attention(q, k, v, cu_seqlens_q, cu_seqlens_k, scale: float, causal: bool = True, *,
                     backend: Optional[str] = None):
    """attention_prompt with the backend switch of ``linear``."""
    return _switch(attention_prompt, _torch_attention_prompt, attention_prompt_contract_reason, backend, q, k, v,
                   cu_seqlens_q, cu_seqlens_k, scale, causal)


def paged_attention(q, cache: KVCache, block_tables, context_lens, scale: float, *, backend: Optional[str] = None):
    """attention_paged with the backend switch of ``linear``."""
    return _switch(attention_paged, _torch_attention_paged, attention_paged_contract_reason, backend, q, cache.k,
                   cache.v, block_tables, context_lens, scale, cache.k_scales, cache.v_scales)
