"""Products in 8 bits, as PyTorch custom ops: rows in 8-bit integers with a
scale each, and the GEMM of such rows with such weights (beside the F.linear
call sites of nanovllm/layers/linear.py:51, 73, 153 and embed_head.py:61).

    quantize_rows(x[..., K]) -> (codes int8 [..., K], scales float32 [...])
        A row x in 8 bits: scale s = max |x| / 127 (float32), codes
        clamp(rint(x / s), -127, 127) of the exact quotient; a code stands for
        code * s.  x is float32, float16 or bfloat16, contiguous or a 2-D view
        with rows of unit stride.  A row of zeros has scale 0; one with a NaN
        or an infinity scale NaN and codes 0.  A weight [N, K] goes through it
        once: its scales are then those of the output channels.

    add_rmsnorm_quantize(h[M, K], residual[M, K], norm_weight[K], eps)
            -> (codes [M, K], scales [M], residual_out [M, K])
        Qwen3_5RMSNorm(h, residual) (nanovllm/layers/layernorm.py:131-142) with
        the normalised rows in 8 bits, taken from float32.

    gemm_int8(a[..., K], a_scales[...], w[N, K], w_scales[N], out_dtype=None)
            -> out[..., N]
        a_scales[i] * w_scales[j] * sum_k a[i, k] w[j, k]: the sum in int32
        (exact; K is below 131072), the scales in float32, rounded once to
        out_dtype (bfloat16 if None; float16, float32).

    gemm_int8_silu_mul(a, a_scales, w[2N, K], w_scales[2N], out_dtype=None)
            -> out[..., N]
        silu(gate) * up of the same product on w = [w_gate; w_up].

Same conventions as ``nanovllm::gemm``: ``nanovllm`` namespace, fixed
RuntimeError messages, fake implementations, launch on the current stream, no
fallback inside the op.  ``int8_linear``, ``int8_silu_mul_linear`` and
``int8_add_rmsnorm_linear`` add the ``torch | hip | auto`` switch with the same
arithmetic in torch operations as the ``torch`` backend.  None of these has a
backward: asking for one raises, on either backend.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F

from .. import _lib
from .gemm import _CODE, default_backend, register_op, run_hip, validate_gemm_backend

_FLOAT = (torch.float32, torch.float16, torch.bfloat16)
_HALF = (torch.float16, torch.bfloat16)
MAX_K = 131071          # int32 holds the sum of so many products of two codes
MAX_ROWS = 1 << 23


def _row_stride(x: torch.Tensor) -> int:
    """Elements between rows of a contiguous tensor or a 2-D view."""
    k = x.shape[-1]
    return x.stride(0) if x.dim() == 2 and x.shape[0] > 1 and not x.is_contiguous() else k


def _rows_reason(name: str, x: torch.Tensor) -> Optional[str]:
    """Why ``x`` is no set of rows, or None if it is."""
    if x.dim() < 1:
        return f"{name} must have at least one dimension"
    if x.shape[-1] == 0:
        return "K must be positive"
    if not x.is_contiguous():
        if x.dim() != 2 or (x.shape[1] > 1 and x.stride(1) != 1):
            return f"{name} must be contiguous, or 2-D with unit stride in its last dimension"
        if x.shape[0] > 1 and x.stride(0) < x.shape[1]:
            return f"the rows of {name} must not overlap"
    if x.numel() // x.shape[-1] > MAX_ROWS:
        return f"{name} must have at most 2^23 rows"
    return None


def quantize_rows_contract_reason(x: torch.Tensor) -> Optional[str]:
    """Why quantize_rows cannot take this input, or None if it can."""
    if not x.is_cuda:
        return "x must be a CUDA (HIP) tensor"
    if x.dtype not in _FLOAT:
        return "x must be float32, float16 or bfloat16"
    return _rows_reason("x", x)


def _quantize_rows_op(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    reason = quantize_rows_contract_reason(x)
    if reason is not None:
        raise RuntimeError(f"nanovllm::quantize_rows: {reason}")
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scales = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    if x.numel():
        k = x.shape[-1]
        with torch.cuda.device(x.device):
            _lib.quantize_rows_raw(x.data_ptr(), codes.data_ptr(), scales.data_ptr(), x.numel() // k, k,
                                   _row_stride(x), _CODE[x.dtype], torch.cuda.current_stream(x.device).cuda_stream)
    return codes, scales


def _quantize_rows_fake(x):
    torch._check(x.dim() >= 1)
    return (x.new_empty(x.shape, dtype=torch.int8), x.new_empty(x.shape[:-1], dtype=torch.float32))


register_op("quantize_rows", _quantize_rows_op, _quantize_rows_fake)


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows in 8 bits: (codes int8, scales float32)."""
    return torch.ops.nanovllm.quantize_rows(x)


def add_rmsnorm_quantize_contract_reason(h: torch.Tensor, residual: torch.Tensor, norm_weight: torch.Tensor,
                                         eps: float) -> Optional[str]:
    """Why add_rmsnorm_quantize cannot take these inputs, or None if it can."""
    tensors = (h, residual, norm_weight)
    if not all(t.is_cuda for t in tensors):
        return "h, residual and norm_weight must be CUDA (HIP) tensors"
    if len({t.device for t in tensors}) != 1:
        return "h, residual and norm_weight must be on the same device"
    if h.dtype not in _HALF:
        return "h must be float16 or bfloat16"
    if any(t.dtype != h.dtype for t in tensors):
        return "h, residual and norm_weight must have the same dtype"
    if h.dim() != 2 or residual.shape != h.shape:
        return "h and residual must be (M, K) tensors of the same shape"
    reason = _rows_reason("h", h) or _rows_reason("residual", residual)
    if reason is not None:
        return reason
    if norm_weight.dim() != 1 or norm_weight.shape[0] != h.shape[1] or not norm_weight.is_contiguous():
        return f"norm_weight must be a contiguous (K,) tensor (K = {h.shape[1]})"
    if not 0.0 <= eps < 3.0e38:
        return "eps must be finite and not negative"
    return None


def _add_rmsnorm_quantize_op(h: torch.Tensor, residual: torch.Tensor, norm_weight: torch.Tensor,
                             eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    reason = add_rmsnorm_quantize_contract_reason(h, residual, norm_weight, eps)
    if reason is not None:
        raise RuntimeError(f"nanovllm::add_rmsnorm_quantize: {reason}")
    m, k = h.shape
    codes = torch.empty((m, k), dtype=torch.int8, device=h.device)
    scales = torch.empty((m,), dtype=torch.float32, device=h.device)
    residual_out = torch.empty((m, k), dtype=h.dtype, device=h.device)
    if m:
        with torch.cuda.device(h.device):
            _lib.add_rmsnorm_quantize_raw(h.data_ptr(), residual.data_ptr(), norm_weight.data_ptr(), float(eps),
                                          codes.data_ptr(), scales.data_ptr(), residual_out.data_ptr(), m, k,
                                          _row_stride(h), _row_stride(residual), _CODE[h.dtype],
                                          torch.cuda.current_stream(h.device).cuda_stream)
    return codes, scales, residual_out


def _add_rmsnorm_quantize_fake(h, residual, norm_weight, eps):
    torch._check(h.dim() == 2)
    return (h.new_empty(h.shape, dtype=torch.int8), h.new_empty(h.shape[:1], dtype=torch.float32),
            h.new_empty(h.shape))


register_op("add_rmsnorm_quantize", _add_rmsnorm_quantize_op, _add_rmsnorm_quantize_fake)


def add_rmsnorm_quantize(h: torch.Tensor, residual: torch.Tensor, norm_weight: torch.Tensor,
                         eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(RMSNorm(h + residual) in 8 bits: codes and scales, round(h + residual))."""
    return torch.ops.nanovllm.add_rmsnorm_quantize(h, residual, norm_weight, float(eps))


def gemm_int8_contract_reason(a: torch.Tensor, a_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
                              out_dtype: Optional[torch.dtype] = None, silu_mul: bool = False) -> Optional[str]:
    """Why the 8-bit GEMM cannot take these inputs, or None if it can."""
    tensors = (a, a_scales, w, w_scales)
    if not all(t.is_cuda for t in tensors):
        return "a, w and their scales must be CUDA (HIP) tensors"
    if len({t.device for t in tensors}) != 1:
        return "a, w and their scales must be on the same device"
    if a.dtype != torch.int8 or w.dtype != torch.int8:
        return "a and w must be int8"
    if a_scales.dtype != torch.float32 or w_scales.dtype != torch.float32:
        return "a_scales and w_scales must be float32"
    if out_dtype is not None and out_dtype not in _FLOAT:
        return f"out_dtype {out_dtype} is not supported: float32, float16 or bfloat16"
    if w.dim() != 2:
        return "w must be 2-D"
    if a.dim() < 1 or a.shape[-1] != w.shape[1]:
        return f"a must have rows of w.size(1) ({w.shape[1]}) codes, got shape {tuple(a.shape)}"
    k = w.shape[1]
    if k < 1 or k > MAX_K:
        return f"K ({k}) must be from 1 to {MAX_K}"
    if silu_mul and w.shape[0] % 2:
        return f"w must hold gate and up halves of equal height (got {w.shape[0]} rows)"
    if not a.is_contiguous() or not w.is_contiguous():
        return "a and w must be contiguous"
    if a_scales.shape != a.shape[:-1] or not a_scales.is_contiguous():
        return f"a_scales must be a contiguous {tuple(a.shape[:-1])} tensor, got shape {tuple(a_scales.shape)}"
    if w_scales.shape != w.shape[:1] or not w_scales.is_contiguous():
        return f"w_scales must be a contiguous {tuple(w.shape[:1])} tensor, got shape {tuple(w_scales.shape)}"
    return None


def _launch_gemm_int8(op, a, a_scales, w, w_scales, out_dtype, silu_mul):
    reason = gemm_int8_contract_reason(a, a_scales, w, w_scales, out_dtype, silu_mul)
    if reason is not None:
        raise RuntimeError(f"nanovllm::{op}: {reason}")
    out_dtype = torch.bfloat16 if out_dtype is None else out_dtype
    k = w.shape[1]
    n = w.shape[0] // 2 if silu_mul else w.shape[0]
    m = a.numel() // k
    out = torch.empty((*a.shape[:-1], n), dtype=out_dtype, device=a.device)
    if m and n:
        with torch.cuda.device(a.device):
            _lib.gemm_int8_raw(a.data_ptr(), a_scales.data_ptr(), w.data_ptr(), w_scales.data_ptr(), out.data_ptr(),
                               m, n, k, k, k, n, silu_mul, _CODE[out_dtype],
                               torch.cuda.current_stream(a.device).cuda_stream)
    return out


def _gemm_int8_op(a: torch.Tensor, a_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
                  out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    return _launch_gemm_int8("gemm_int8", a, a_scales, w, w_scales, out_dtype, False)


def _gemm_int8_fake(a, a_scales, w, w_scales, out_dtype=None):
    torch._check(w.dim() == 2)
    torch._check(a.shape[-1] == w.shape[1])
    return a.new_empty((*a.shape[:-1], w.shape[0]), dtype=torch.bfloat16 if out_dtype is None else out_dtype)


register_op("gemm_int8", _gemm_int8_op, _gemm_int8_fake)


def gemm_int8(a: torch.Tensor, a_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
              out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """(a * a_scales) @ (w * w_scales).T of 8-bit codes, the sum exact in int32."""
    return torch.ops.nanovllm.gemm_int8(a, a_scales, w, w_scales, out_dtype)


def _gemm_int8_silu_mul_op(a: torch.Tensor, a_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
                           out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    return _launch_gemm_int8("gemm_int8_silu_mul", a, a_scales, w, w_scales, out_dtype, True)


def _gemm_int8_silu_mul_fake(a, a_scales, w, w_scales, out_dtype=None):
    torch._check(w.dim() == 2)
    torch._check(w.shape[0] % 2 == 0)
    torch._check(a.shape[-1] == w.shape[1])
    return a.new_empty((*a.shape[:-1], w.shape[0] // 2), dtype=torch.bfloat16 if out_dtype is None else out_dtype)


register_op("gemm_int8_silu_mul", _gemm_int8_silu_mul_op, _gemm_int8_silu_mul_fake)


def gemm_int8_silu_mul(a: torch.Tensor, a_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
                       out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """SiluAndMul of the 8-bit GEMM on w = [w_gate; w_up] in one launch."""
    return torch.ops.nanovllm.gemm_int8_silu_mul(a, a_scales, w, w_scales, out_dtype)


# ---------------------------------------------------------------------------
# Backend switch and the same arithmetic in torch operations
# ---------------------------------------------------------------------------
def torch_quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """quantize_rows in torch operations (the quotients in 64 bits; a division by a plain number in 32 is a product with its
    reciprocal on a GPU)."""
    top = x.float().abs().amax(-1)
    good = top < float("inf")      # false for a NaN too
    scale = torch.where(good, (top.double() / 127).float(), float("nan"))
    safe = torch.where(good & (scale > 0), scale, 1.0).double().unsqueeze(-1)
    codes = torch.where((good & (scale > 0)).unsqueeze(-1), (x.double() / safe).round().clamp(-127, 127), 0.0)
    return codes.to(torch.int8), scale


def torch_gemm_int8(a: torch.Tensor, a_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
                    out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """gemm_int8 in torch operations (the sum in 64 bits, which is exact)."""
    y = F.linear(a.double(), w.double()).float() * w_scales * a_scales.unsqueeze(-1)
    return y.to(torch.bfloat16 if out_dtype is None else out_dtype)


def _torch_silu_mul(y: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    gate, up = y.chunk(2, -1)
    return (F.silu(gate) * up).to(dtype)


def _weights_reason(x, w, w_scales, out_dtype, silu_mul) -> Optional[str]:
    """Why the 8-bit GEMM cannot take these weights behind rows like x's, or None if it can."""
    if not (w.is_cuda and w_scales.is_cuda) or not w.device == w_scales.device == x.device:
        return "w and w_scales must be on the device of x"
    if w.dtype != torch.int8 or w_scales.dtype != torch.float32:
        return "w must be int8 and w_scales float32"
    if out_dtype not in _FLOAT:
        return f"out_dtype {out_dtype} is not supported: float32, float16 or bfloat16"
    if w.dim() != 2 or x.shape[-1] != w.shape[1]:
        return f"x must have rows of w.size(1), got shapes {tuple(x.shape)} and {tuple(w.shape)}"
    if w.shape[1] > MAX_K:
        return f"K ({w.shape[1]}) must be from 1 to {MAX_K}"
    if silu_mul and w.shape[0] % 2:
        return f"w must hold gate and up halves of equal height (got {w.shape[0]} rows)"
    if not w.is_contiguous() or w_scales.shape != w.shape[:1] or not w_scales.is_contiguous():
        return "w and w_scales must be contiguous, with a scale for each row of w"
    return None


class _NoBackward(torch.autograd.Function):

    @staticmethod
    def forward(ctx, y, name, *inputs):
        ctx.name = name
        return y.view_as(y)

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError(f"{ctx.name} has no backward: the layers in 8 bits serve")


def _refuse_backward(name: str, y: torch.Tensor, *inputs: torch.Tensor) -> torch.Tensor:
    """y with the ops' refusal of a backward: codes have no gradient, and that of the scales alone is no row's."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in inputs):
        return _NoBackward.apply(y, name, *inputs)
    return y


def _hip(backend: Optional[str], reason) -> bool:
    backend = validate_gemm_backend(backend) if backend is not None else default_backend()
    return backend == "hip" or (backend == "auto" and reason() is None)


def _check_types(name: str, w: torch.Tensor, w_scales: torch.Tensor) -> None:
    """The torch backend takes the ops' types alone: scales rounded to 16 bits, of a module that was converted after its
    weights went to 8 bits, are refused and not used."""
    if w.dtype != torch.int8 or w_scales.dtype != torch.float32:
        raise RuntimeError(f"{name}: w must be int8 and w_scales float32, got {w.dtype} and {w_scales.dtype}")


def _int8_linear(x, w, w_scales, out_dtype, backend, silu_mul):
    out_dtype = x.dtype if out_dtype is None else out_dtype

    def reason(x, w, w_scales):
        return quantize_rows_contract_reason(x) or _weights_reason(x, w, w_scales, out_dtype, silu_mul)

    def op(x, w, w_scales):
        return (gemm_int8_silu_mul if silu_mul else gemm_int8)(*quantize_rows(x), w, w_scales, out_dtype)

    if _hip(backend, lambda: reason(x, w, w_scales)):
        return run_hip(op, reason, x, w, w_scales)
    name = "int8_silu_mul_linear" if silu_mul else "int8_linear"
    _check_types(name, w, w_scales)
    with torch.no_grad():
        if silu_mul:
            y = _torch_silu_mul(torch_gemm_int8(*torch_quantize_rows(x), w, w_scales, torch.float32), out_dtype)
        else:
            y = torch_gemm_int8(*torch_quantize_rows(x), w, w_scales, out_dtype)
    return _refuse_backward(name, y, x, w_scales)


def int8_linear(x: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, *, out_dtype: Optional[torch.dtype] = None,
                backend: Optional[str] = None) -> torch.Tensor:
    """x times 8-bit weights: quantize_rows and gemm_int8, with the backend
    switch of ``linear``; the output has the dtype of x unless one is named."""
    return _int8_linear(x, w, w_scales, out_dtype, backend, False)


def int8_silu_mul_linear(x: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, *,
                         out_dtype: Optional[torch.dtype] = None, backend: Optional[str] = None) -> torch.Tensor:
    """SiluAndMul of x times 8-bit [gate; up] weights, with the backend switch."""
    return _int8_linear(x, w, w_scales, out_dtype, backend, True)


def int8_add_rmsnorm_linear(h: torch.Tensor, residual: torch.Tensor, norm_weight: torch.Tensor, eps: float,
                            w: torch.Tensor, w_scales: torch.Tensor, *, silu_mul: bool = False,
                            backend: Optional[str] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(8-bit projection of RMSNorm(h + residual) [then SiluAndMul], new
    residual) with the backend switch: add_rmsnorm_quantize, then the GEMM."""

    def reason(h, residual, norm_weight, w, w_scales):
        return (add_rmsnorm_quantize_contract_reason(h, residual, norm_weight, eps)
                or _weights_reason(h, w, w_scales, h.dtype, silu_mul))

    def op(h, residual, norm_weight, w, w_scales):
        codes, scales, new_residual = add_rmsnorm_quantize(h, residual, norm_weight, eps)
        product = gemm_int8_silu_mul if silu_mul else gemm_int8
        return product(codes, scales, w, w_scales, h.dtype), new_residual

    args = (h, residual, norm_weight, w, w_scales)
    if _hip(backend, lambda: reason(*args)):
        return run_hip(op, reason, *args)
    _check_types("int8_add_rmsnorm_linear", w, w_scales)
    with torch.no_grad():
        summed = h.float() + residual.float()
        normed = summed * torch.rsqrt(summed.pow(2).mean(-1, keepdim=True) + eps) * (1.0 + norm_weight.float())
        y = torch_gemm_int8(*torch_quantize_rows(normed), w, w_scales, torch.float32)
        y = _torch_silu_mul(y, h.dtype) if silu_mul else y.to(h.dtype)
    given = (h, residual, norm_weight, w_scales)
    return (_refuse_backward("int8_add_rmsnorm_linear", y, *given),
            _refuse_backward("int8_add_rmsnorm_linear", summed.to(h.dtype), *given))
