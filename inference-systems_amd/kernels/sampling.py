"""The sampler on logits, as a PyTorch custom op (beside Sampler.forward,
nanovllm/layers/sampler.py:8-21, which knows the temperature alone).

    sample_logits(logits[..., V], temperatures[...], uniforms[...], top_k=None,
                  top_p=None, min_p=None) -> (tokens int64 [...], logprobs [...])
        A token a row by temperature, top-k, top-p and min-p from a given random
        number u in [0, 1).  Tokens are ordered by logit, the largest first and
        the first index first among equals, and weigh exp((l - max l) / T)
        (one below 2^-63 may count as 0).  Kept are the first top_k of them (all where it
        is 0 or less), of these the shortest run from the front whose weights
        reach the share top_p of theirs (all where it is 1 or more), and of
        these the ones of a weight of at least min_p (all where it is 0 or
        less); the first is always kept.  The token is the first, by index, at
        which the running sum of the kept weights is above u times their total;
        logprobs is the natural logarithm of its share of that total.  Rows with
        T <= 1e-10 take the largest logit, the first of equals, logprob 0.

        logits: float32, float16 or bfloat16, contiguous or a 2-D view with rows
        of unit stride.  temperatures, uniforms, top_p, min_p: float32; top_k:
        int32; one entry a row.  A row whose largest logit is an infinity draws
        among its holders; one with a NaN takes its first NaN, logprob NaN.

The result depends on the inputs alone: weights are good to 2^-32 of themselves
(2^-25 where T is above 2^100), and no sum depends on the order in which
workgroups run.  ``sample_rows`` adds the ``torch | hip | auto`` switch.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from .gemm import _CODE, default_backend, register_op, run_hip, validate_gemm_backend
from .int8 import _row_stride, _rows_reason

_FLOAT = (torch.float32, torch.float16, torch.bfloat16)
GREEDY_TEMPERATURE = 1e-10
MAX_VOCAB = 1 << 23
MAX_SAMPLE_ROWS = 1 << 20


def sample_logits_contract_reason(logits: torch.Tensor, temperatures: torch.Tensor, uniforms: torch.Tensor,
                                  top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
                                  min_p: Optional[torch.Tensor] = None) -> Optional[str]:
    """Why sample_logits cannot take these inputs, or None if it can."""
    given = [("temperatures", temperatures, torch.float32), ("uniforms", uniforms, torch.float32)]
    given += [(name, t, dtype) for name, t, dtype in
              (("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32))
              if t is not None]
    if not (logits.is_cuda and all(t.is_cuda for _, t, _ in given)):
        return "logits and the rows' parameters must be CUDA (HIP) tensors"
    if any(t.device != logits.device for _, t, _ in given):
        return "logits and the rows' parameters must be on the same device"
    if logits.dtype not in _FLOAT:
        return "logits must be float32, float16 or bfloat16"
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= MAX_VOCAB:
        return f"logits must have rows of 1 to {MAX_VOCAB} entries, got shape {tuple(logits.shape)}"
    reason = _rows_reason("logits", logits)
    if reason is not None:
        return reason
    if logits.numel() // logits.shape[-1] > MAX_SAMPLE_ROWS:
        return "logits must have at most 2^20 rows"
    for name, t, dtype in given:
        if t.dtype != dtype:
            return f"{name} must be {dtype}"
        if t.shape != logits.shape[:-1] or not t.is_contiguous():
            return f"{name} must be a contiguous {tuple(logits.shape[:-1])} tensor, got shape {tuple(t.shape)}"
    return None


def _sample_logits_op(logits: torch.Tensor, temperatures: torch.Tensor, uniforms: torch.Tensor,
                      top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
                      min_p: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    reason = sample_logits_contract_reason(logits, temperatures, uniforms, top_k, top_p, min_p)
    if reason is not None:
        raise RuntimeError(f"nanovllm::sample_logits: {reason}")
    vocab = logits.shape[-1]
    m = logits.numel() // vocab
    tokens = torch.empty(logits.shape[:-1], dtype=torch.int64, device=logits.device)
    logprobs = torch.empty(logits.shape[:-1], dtype=torch.float32, device=logits.device)
    if m:
        need = _lib.sample_logits_workspace_bytes(m, vocab, _CODE[logits.dtype])
        _lib.check(need if need < 0 else _lib.OK, "nanovllm_sample_logits_workspace_bytes")
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=logits.device)
        with torch.cuda.device(logits.device):
            _lib.sample_logits_raw(logits.data_ptr(), temperatures.data_ptr(), uniforms.data_ptr(),
                                   *(None if t is None else t.data_ptr() for t in (top_k, top_p, min_p)),
                                   tokens.data_ptr(), logprobs.data_ptr(), m, vocab, _row_stride(logits),
                                   _CODE[logits.dtype], workspace.data_ptr(), need,
                                   torch.cuda.current_stream(logits.device).cuda_stream)
    return tokens, logprobs


def _sample_logits_fake(logits, temperatures, uniforms, top_k=None, top_p=None, min_p=None):
    torch._check(logits.dim() >= 1)
    return (logits.new_empty(logits.shape[:-1], dtype=torch.int64),
            logits.new_empty(logits.shape[:-1], dtype=torch.float32))


register_op("sample_logits", _sample_logits_op, _sample_logits_fake)


def sample_logits(logits: torch.Tensor, temperatures: torch.Tensor, uniforms: torch.Tensor,
                  top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
                  min_p: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(token ids, log-probabilities among the kept tokens) of the rows of logits."""
    return torch.ops.nanovllm.sample_logits(logits, temperatures, uniforms, top_k, top_p, min_p)


def torch_sample_logits(logits: torch.Tensor, temperatures: torch.Tensor, uniforms: torch.Tensor,
                        top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
                        min_p: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """sample_logits in torch operations, on finite and infinite logits: a sort a row, weights in 64 bits."""
    shape, vocab = logits.shape[:-1], logits.shape[-1]
    x = logits.reshape(-1, vocab).float()
    t = temperatures.reshape(-1, 1)
    greedy = ~(t > GREEDY_TEMPERATURE)
    # NaN sorts first, as it does in torch.argmax.
    ordered, index = torch.sort(x, dim=1, descending=True, stable=True)
    top = ordered[:, :1].double()
    weight = torch.where(ordered.double() == top, 1.0,
                         ((ordered.double() - top) / torch.where(greedy, 1.0, t).double()).exp())
    # Below an infinite logit nothing has weight, nor has -inf below a finite one (at T = inf both are NaN so far).
    weight = torch.where((ordered.double() < top) & (top.isinf() | ordered.isinf()), 0.0, weight)
    rank = torch.arange(vocab, device=logits.device)
    kept = torch.ones_like(weight, dtype=torch.bool)
    if top_k is not None:
        k = top_k.reshape(-1, 1)
        kept &= (rank < k) | (k <= 0)
    if top_p is not None:
        p = top_p.reshape(-1, 1).double()
        some = torch.where(kept, weight, 0.0)
        kept &= (some.cumsum(1) - some < p * some.sum(1, keepdim=True)) | ~(p < 1)
    if min_p is not None:
        p = min_p.reshape(-1, 1).double()
        kept &= (weight >= p) | ~(p > 0)
    kept[:, 0] = True
    by_index = torch.zeros_like(weight).scatter_(1, index, torch.where(kept, weight, 0.0))
    running = by_index.cumsum(1)
    total = running[:, -1:]
    u = uniforms.reshape(-1, 1).double()
    # From 1 on no running sum is above it, whose last bits may pass the total's.
    target = torch.where(u >= 1, float("inf"), torch.where(u > 0, u, 0.0)) * total
    above = (running > target) & (by_index > 0)
    last = vocab - 1 - (by_index > 0).flip(1).to(torch.int8).argmax(1, keepdim=True)
    token = torch.where(above.any(1, keepdim=True), above.to(torch.int8).argmax(1, keepdim=True), last)
    share = (by_index.gather(1, token) / total).log().float()
    bad = ordered[:, :1].isnan()
    token = torch.where(greedy | bad, index[:, :1], token)
    share = torch.where(bad, float("nan"), torch.where(greedy, 0.0, share))
    return token.reshape(shape), share.reshape(shape)


def sample_rows(logits: torch.Tensor, temperatures: torch.Tensor, uniforms: torch.Tensor,
                top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
                min_p: Optional[torch.Tensor] = None, *, backend: Optional[str] = None
                ) -> tuple[torch.Tensor, torch.Tensor]:
    """sample_logits with the backend switch of ``linear``."""
    backend = validate_gemm_backend(backend) if backend is not None else default_backend()
    args = (logits, temperatures, uniforms, top_k, top_p, min_p)
    if backend == "hip" or (backend == "auto" and sample_logits_contract_reason(*args) is None):
        return run_hip(sample_logits, sample_logits_contract_reason, *args)
    return torch_sample_logits(*args)
