"""Qwen3.5's gated attention with the paged-cache and attention ops.

Same submodules and weight layout as the reference's layer
(nanovllm/models/qwen3_5.py:40-96): ``q_proj`` gives a query and an output gate
per head, queries and keys are normalised per head, the first ``rotary_dim``
channels are rotated, and the attention output is gated in front of ``o_proj``.
Between the projections this layer runs the four ops of kernels/attention.py;
the reference calls its rotary embedding, store_kvcache and flash attention
there (nanovllm/layers/attention.py).

``forward`` takes what the reference keeps in its context: where the new tokens
go (``slots``) and one of

  decode   one token per sequence: ``block_tables`` and ``context_lens`` (this
           token counted)
  prompt   ``cu_seqlens``: packed prompts
  chunk    ``cu_seqlens`` of the new tokens with ``cu_seqlens_k`` and
           ``context_slots``, the slots of every token of each sequence (the
           cached prefix and the new ones): what the chunk attends to is read
           back from the cache
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from ..kernels import KVCache, gather_kv, paged_attention, prompt_attention, rope_append_kv
from .linear import ColumnParallelLinear, RowParallelLinear, _tp_rank_size, divide
from .norm import Qwen35RMSNorm


class Qwen35Attention(nn.Module):

    def __init__(self, hidden_size: int, num_heads: int, num_kv_heads: int, head_dim: int,
                 rms_norm_eps: float = 1e-6):
        super().__init__()
        _, tp_size = _tp_rank_size()
        self.num_heads = divide(num_heads, tp_size)
        self.num_kv_heads = divide(num_kv_heads, tp_size)
        self.head_dim = head_dim
        self.scale = head_dim ** -0.5
        self.q_proj = ColumnParallelLinear(hidden_size, num_heads * head_dim * 2)
        self.k_proj = ColumnParallelLinear(hidden_size, num_kv_heads * head_dim)
        self.v_proj = ColumnParallelLinear(hidden_size, num_kv_heads * head_dim)
        self.o_proj = RowParallelLinear(num_heads * head_dim, hidden_size)
        self.q_norm = Qwen35RMSNorm(head_dim, rms_norm_eps)
        self.k_norm = Qwen35RMSNorm(head_dim, rms_norm_eps)
        self._gemm_backend: Optional[str] = None

    @property
    def gemm_backend(self) -> Optional[str]:
        return self._gemm_backend

    @gemm_backend.setter
    def gemm_backend(self, value: Optional[str]) -> None:
        """Backend of the projections and the ops (None: NANOVLLM_GEMM_BACKEND)."""
        self._gemm_backend = value
        for proj in (self.q_proj, self.k_proj, self.v_proj, self.o_proj):
            proj.gemm_backend = value

    def forward(self, hidden: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, cache: KVCache,
                slots: torch.Tensor, *, block_tables: Optional[torch.Tensor] = None,
                context_lens: Optional[torch.Tensor] = None, cu_seqlens: Optional[torch.Tensor] = None,
                cu_seqlens_k: Optional[torch.Tensor] = None,
                context_slots: Optional[torch.Tensor] = None) -> torch.Tensor:
        if (block_tables is None) != (context_lens is None) or (block_tables is None) == (cu_seqlens is None):
            raise ValueError("pass block_tables and context_lens (decode) or cu_seqlens (prompts)")
        if (cu_seqlens_k is None) != (context_slots is None) or (cu_seqlens is None and cu_seqlens_k is not None):
            raise ValueError("cu_seqlens_k and context_slots go together, with cu_seqlens")
        backend = self._gemm_backend
        q, gate = self.q_proj(hidden).view(-1, self.num_heads, 2 * self.head_dim).chunk(2, dim=-1)
        q = self.q_norm(q)
        k = self.k_norm(self.k_proj(hidden).view(-1, self.num_kv_heads, self.head_dim))
        v = self.v_proj(hidden).view(-1, self.num_kv_heads, self.head_dim)
        q, k = rope_append_kv(q, k, v, positions, cos_sin, slots, cache, backend=backend)
        if block_tables is not None:
            out = paged_attention(q, cache, block_tables, context_lens, self.scale, backend=backend)
        elif context_slots is not None:
            k, v = gather_kv(cache, context_slots, q.dtype, backend=backend)
            out = prompt_attention(q, k, v, cu_seqlens, cu_seqlens_k, self.scale, backend=backend)
        else:
            out = prompt_attention(q, k, v, cu_seqlens, cu_seqlens, self.scale, backend=backend)
        return self.o_proj.forward_gated(out, gate)
