"""The operators of an 8-bit serving step, from the residual stream to the token, as cases that can be timed.

  rows    ``kernels.quantize_rows``: rows in 8 bits, a scale a row
  norm    ``kernels.add_rmsnorm_quantize``: residual add and zero-centred RMS norm, the normalised rows in 8 bits
  gemm    ``kernels.gemm_int8``: product of 8-bit rows with 8-bit weights, scales by row and by output channel
  silu    ``kernels.gemm_int8_silu_mul``: the same on [gate; up] weights, SiLU(gate) * up
  sample  ``kernels.sample_logits``: a token a row by temperature, top-k, top-p and min-p, from a given random number

``own`` false: elementary torch operations in 32 bits, rounded once at the end; in 64 bits where a quotient is rounded to
a code or a sum is compared with a border.  ``own`` true: the library's calls.

A case is a dict of plain values:

  op      "rows", "norm", "gemm", "silu", "sample"
  dtype   "rows", "norm": type of the rows; "gemm", "silu": type of the output; "sample": type of the logits
          ("bf16", "f16", "f32")
  m       rows
  k       length of a row ("rows", "norm", "gemm", "silu")
  n       output channels ("gemm", "silu")
  vocab   logits of a row ("sample")
  peak    "sample": how far the likeliest tokens stand above the others; 0: none does
  top_k   "sample": typical number of tokens kept (each row has its own); 0: off
  top_p, min_p   "sample": typical values, a row has its own; 0: off

A row x in 8 bits: scale s = max |x| / 127 (in float32), codes round(x / s), to even on a tie; it stands for code * s.
"sample": the tokens of a row, the largest logit first and the lowest index first among equals, have weights
exp((l - max l) / T).  Kept are the first top_k of them, of these the shortest run from the front that holds at least
the share top_p of their weight, and of these the tokens whose weight is at least min_p times the largest.  The token
is the first, by index, at which the running sum of the kept weights is above u times their total; beside it comes the
logarithm of its share of that total.  A temperature up to 1e-10 takes the largest logit, the first of equals, and 0.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
GREEDY = 1e-10


def _kernels():
    import __graft_entry__
    return __graft_entry__.load_package().kernels


def listed():
    return [
        # The input of a projection in a decode step: latency counts.
        {"name": "rows 8x1024", "op": "rows", "dtype": "bf16", "m": 8, "k": 1024},
        # The hidden rows of an MLP over a batch of prompts.
        {"name": "rows 8192x3584 f16", "op": "rows", "dtype": "f16", "m": 8192, "k": 3584},
        # The norm before a projection, one sequence.
        {"name": "norm 1x1024", "op": "norm", "dtype": "bf16", "m": 1, "k": 1024},
        # The same over packed prompts.
        {"name": "norm 4100x1024", "op": "norm", "dtype": "bf16", "m": 4100, "k": 1024},
        # Decode projection of a batch of 8.
        {"name": "gemm 8x6144x1024", "op": "gemm", "dtype": "bf16", "m": 8, "n": 6144, "k": 1024},
        # Odd sizes: rows that are no whole 16-byte chunks.
        {"name": "gemm 333x2501x1003 f16", "op": "gemm", "dtype": "f16", "m": 333, "n": 2501, "k": 1003},
        # The LM head of a decode batch, logits in 32 bits.
        {"name": "gemm 32x151936x1024 f32", "op": "gemm", "dtype": "f32", "m": 32, "n": 151936, "k": 1024},
        # A projection over packed prompts of a larger model: the largest product.
        {"name": "gemm 8192x8192x4096", "op": "gemm", "dtype": "bf16", "m": 8192, "n": 8192, "k": 4096},
        # Gate and up projection, decode batch.
        {"name": "silu 16x3584x1024", "op": "silu", "dtype": "bf16", "m": 16, "n": 3584, "k": 1024},
        # Gate and up projection of a prompt.
        {"name": "silu 2048x3584x1024", "op": "silu", "dtype": "bf16", "m": 2048, "n": 3584, "k": 1024},
        # One sequence's next token, the usual filters.
        {"name": "sample 1x151936", "op": "sample", "dtype": "bf16", "m": 1, "vocab": 151936, "peak": 12.0,
         "top_k": 50, "top_p": 0.9, "min_p": 0.0},
        # The next tokens of a large batch, logits in 32 bits, no limit on the count.
        {"name": "sample 256x151936 f32", "op": "sample", "dtype": "f32", "m": 256, "vocab": 151936, "peak": 8.0,
         "top_k": 0, "top_p": 0.95, "min_p": 0.02},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rows", "norm", "gemm", "gemm", "silu", "sample", "sample"])
    if op in ("rows", "norm"):
        k = rng.choice([_log(rng, 16, 16000), 8 * _log(rng, 2, 2000)])
        return {"op": op, "dtype": rng.choice(["bf16", "f16", "f32"] if op == "rows" else ["bf16", "f16"]),
                "m": max(1, min(_log(rng, 1, 16000), int(2.9e7) // k)), "k": k}
    if op == "sample":
        vocab = _log(rng, 500, 262144)
        return {"op": op, "dtype": rng.choice(["bf16", "f16", "f32"]),
                "m": max(1, min(_log(rng, 1, 512), int(3.8e7) // vocab)), "vocab": vocab,
                "peak": rng.choice([0.0, rng.uniform(4.0, 14.0), rng.uniform(4.0, 14.0)]),
                "top_k": rng.choice([0, _log(rng, 1, 2000)]), "top_p": rng.choice([0.0, rng.uniform(0.3, 0.99)]),
                "min_p": rng.choice([0.0, rng.uniform(0.005, 0.3)])}
    while True:
        case = {"op": op, "dtype": rng.choice(["bf16", "f16", "f32"]), "m": _log(rng, 1, 8192),
                "n": rng.choice([_log(rng, 8, 100000), 16 * _log(rng, 1, 8000)]),
                "k": rng.choice([_log(rng, 16, 8192), 16 * _log(rng, 1, 512), 16 * _log(rng, 1, 512)])}
        done = work(case)
        if done["flops"] <= 5.0e11 and done["bytes"] <= 3.0e8:
            return case


# ---------------------------------------------------------------------------
# Inputs: activations are standard normal with a few large channels, as behind
# a norm; weights are normal; logits are normal, a few tokens a row above them.
# ---------------------------------------------------------------------------
class _Inputs:
    def __init__(self, seed):
        self.gen = torch.Generator(device=DEV).manual_seed(int(seed))

    def normal(self, *shape):
        return torch.randn(shape, generator=self.gen, device=DEV)

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.gen, device=DEV)

    def activations(self, m, k):
        channel = torch.where(self.uniform(k) < 0.01, 8.0, 1.0)
        return self.normal(m, k) * channel

    def codes(self, x):
        """Rows in 8 bits, in the form in which the product takes them."""
        scale = x.abs().amax(-1).clamp_min(1e-20) / 127
        return (x / scale[:, None]).round().to(torch.int8), scale


def prepare(case, seed):
    inp, op, m = _Inputs(seed), case["op"], case["m"]
    state = {"case": case}
    if op == "rows":
        return state | {"x": inp.activations(m, case["k"]).to(DTYPES[case["dtype"]])}
    if op == "norm":
        dtype, k = DTYPES[case["dtype"]], case["k"]
        return state | {"h": inp.activations(m, k).to(dtype), "residual": (3 * inp.normal(m, k)).to(dtype),
                        "weight": (0.2 * inp.normal(k)).to(dtype)}
    if op == "sample":
        vocab = case["vocab"]
        logits = 2.0 * inp.normal(m, vocab)
        if case["peak"]:
            at = torch.randint(0, vocab, (m, 24), generator=inp.gen, device=DEV)
            logits.scatter_add_(1, at, case["peak"] * inp.uniform(m, 24))
        state |= {"logits": logits.to(DTYPES[case["dtype"]]), "u": inp.uniform(m)}
        temperature = 0.6 + 0.7 * inp.uniform(m)
        if m > 3:
            temperature[m // 2] = 0.0      # a greedy row in the batch
        state["temperature"] = temperature
        state["top_k"] = (torch.randint(1, 2 * case["top_k"] + 1, (m,), generator=inp.gen, device=DEV,
                                        dtype=torch.int32) if case["top_k"] else None)
        state["top_p"] = (1 - (1 - case["top_p"]) * 2 * inp.uniform(m)).clamp(0.05, 0.999) if case["top_p"] else None
        state["min_p"] = 2 * case["min_p"] * inp.uniform(m) if case["min_p"] else None
        return state
    a, a_scales = inp.codes(inp.activations(m, case["k"]))
    w, w_scales = inp.codes(0.02 * inp.normal(case["n"] * (2 if op == "silu" else 1), case["k"]))
    return state | {"a": a, "a_scales": a_scales, "w": w, "w_scales": w_scales}


# ---------------------------------------------------------------------------
# The plain forms.
# ---------------------------------------------------------------------------
def _quantise(x):
    """Rows x in 32 bits: (codes as 32-bit numbers, scales)."""
    scale = x.abs().amax(-1) / 127
    # In 64 bits: a quotient next to a half must fall to the right side.
    codes = (x.double() / torch.where(scale == 0, 1.0, scale).double()[:, None]).round().clamp(-127, 127)
    return codes.float(), scale


def _product(state):
    p = torch.matmul(state["a"].float(), state["w"].float().T)
    return p * state["a_scales"][:, None] * state["w_scales"]


def _sample(logits, temperature, u, top_k, top_p, min_p):
    vocab = logits.shape[1]
    # The order of the tokens: descending, the lowest index first among equals.
    ordered, index = torch.sort(logits.float(), dim=1, descending=True, stable=True)
    greedy = temperature <= GREEDY
    t = torch.where(greedy, 1.0, temperature).double()[:, None]
    weight = ((ordered.double() - ordered[:, :1].double()) / t).exp()
    rank = torch.arange(vocab, device=DEV)
    kept = torch.ones_like(weight, dtype=torch.bool)
    if top_k is not None:
        kept &= rank < top_k[:, None]
    if top_p is not None:
        some = torch.where(kept, weight, 0.0)
        before = some.cumsum(1) - some
        kept &= (before < top_p.double()[:, None] * some.sum(1, keepdim=True)) | (rank == 0)
    if min_p is not None:
        kept &= weight >= min_p.double()[:, None]
    by_index = torch.zeros_like(weight).scatter_(1, index, torch.where(kept, weight, 0.0))
    running = by_index.cumsum(1)
    token = (running <= u.double()[:, None] * running[:, -1:]).sum(1).clamp(max=vocab - 1)
    share = (by_index.gather(1, token[:, None]) / running[:, -1:])[:, 0]
    return {"tokens": torch.where(greedy, index[:, 0], token),
            "logprobs": torch.where(greedy, 0.0, share.log()).float()}


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    if op == "rows":
        codes, scale = _quantise(state["x"].float())
        return {"values": (codes * scale[:, None]).to(dtype), "scales": scale}
    if op == "norm":
        total = state["h"].float() + state["residual"].float()
        normed = total * (total.square().mean(-1, keepdim=True) + EPS).rsqrt() * (1 + state["weight"].float())
        codes, scale = _quantise(normed)
        return {"values": (codes * scale[:, None]).to(dtype), "scales": scale, "residual": total.to(dtype)}
    if op == "gemm":
        return _product(state).to(dtype)
    if op == "silu":
        gate, up = _product(state).chunk(2, -1)
        return (gate / (1 + (-gate).exp()) * up).to(dtype)
    return _sample(*(state[x] for x in ("logits", "temperature", "u", "top_k", "top_p", "min_p")))


def _values(codes, scales, dtype):
    """What codes stand for."""
    return torch.mul(codes, scales[:, None], out=torch.empty(codes.shape, dtype=dtype, device=codes.device))


def _run_own(case, state):
    ops, op, dtype = _kernels(), case["op"], DTYPES[case["dtype"]]
    if op == "rows":
        codes, scales = ops.quantize_rows(state["x"])
        return {"values": _values(codes, scales, dtype), "scales": scales}
    if op == "norm":
        codes, scales, residual = ops.add_rmsnorm_quantize(state["h"], state["residual"], state["weight"], EPS)
        return {"values": _values(codes, scales, dtype), "scales": scales, "residual": residual}
    if op == "gemm":
        return ops.gemm_int8(state["a"], state["a_scales"], state["w"], state["w_scales"], dtype)
    if op == "silu":
        return ops.gemm_int8_silu_mul(state["a"], state["a_scales"], state["w"], state["w_scales"], dtype)
    tokens, logprobs = ops.sample_logits(state["logits"], state["temperature"], state["u"], state["top_k"],
                                         state["top_p"], state["min_p"])
    return {"tokens": tokens, "logprobs": logprobs}


# ---------------------------------------------------------------------------
# What a pass cannot do without.
# ---------------------------------------------------------------------------
def work(case):
    op, m, size = case["op"], case["m"], 4 if case["dtype"] == "f32" else 2
    if op == "rows":       # the rows read; what they are in 8 bits written
        return {"bytes": m * case["k"] * (size + 1) + 4 * m, "flops": 4 * m * case["k"]}
    if op == "norm":
        return {"bytes": m * case["k"] * (3 * size + 1) + size * case["k"] + 4 * m, "flops": 9 * m * case["k"]}
    if op == "sample":
        given = 8 + 4 * sum(1 for x in ("top_k", "top_p", "min_p") if case[x])
        return {"bytes": m * case["vocab"] * size + m * (given + 12), "flops": 4 * m * case["vocab"]}
    n, k, pair = case["n"], case["k"], 2 if op == "silu" else 1
    return {"bytes": m * k + pair * n * k + size * m * n + 4 * (m + pair * n), "flops": 2 * pair * m * n * k}


# ---------------------------------------------------------------------------
# The definition in 64 bits.
# ---------------------------------------------------------------------------
def _stands_for(x):
    """What rows x (64 bits) are in 8 bits, and their scales (which are kept in 32 bits)."""
    scale = (x.abs().max(-1).values / 127).float().double()
    safe = torch.where(scale > 0, scale, 1.0)[:, None]
    return torch.clip(torch.round(x / safe), -127, 127) * scale[:, None], scale


def _token(logits, t, u, top_k, top_p, min_p):
    """The token of one row and the logarithm of its share (numpy, 64 bits)."""
    if t <= GREEDY:
        return int(np.argmax(logits)), 0.0
    order = np.lexsort((np.arange(logits.size), -logits))
    weight = np.exp((logits[order] - logits[order[0]]) / t)
    last = logits.size if top_k is None else min(int(top_k), logits.size)
    if top_p is not None:
        share = np.cumsum(weight[:last])
        last = min(last, 1 + int(np.searchsorted(share, top_p * share[-1])))
    if min_p is not None:
        last = min(last, max(1, int(np.count_nonzero(weight >= min_p))))
    chosen = np.sort(order[:last])
    share = np.cumsum(np.exp((logits[chosen] - logits[order[0]]) / t))
    token = int(chosen[min(int(np.searchsorted(share, u * share[-1], side="right")), last - 1)])
    return token, float((logits[token] - logits[order[0]]) / t - np.log(share[-1]))


def exact(case, seed):
    state, op = prepare(case, seed), case["op"]
    if op == "rows":
        values, scales = _stands_for(state["x"].double())
        return {"values": values, "scales": scales}
    if op == "norm":
        s = state["h"].double() + state["residual"].double()
        root = torch.sqrt(torch.sum(s * s, -1, keepdim=True) / s.shape[1] + EPS)
        values, scales = _stands_for((1.0 + state["weight"].double()) * s / root)
        return {"values": values, "scales": scales, "residual": s}
    if op == "sample":
        rows = state["logits"].double().cpu().numpy()
        given = [None if state[x] is None else state[x].double().cpu().numpy()
                 for x in ("temperature", "u", "top_k", "top_p", "min_p")]
        found = [_token(row, *(None if g is None else g[i] for g in given)) for i, row in enumerate(rows)]
        return {"tokens": torch.tensor([f[0] for f in found], device=DEV),
                "logprobs": torch.tensor([f[1] for f in found], device=DEV, dtype=torch.float64)}
    a = state["a"].double() * state["a_scales"].double()[:, None]
    w = state["w"].double() * state["w_scales"].double()[:, None]
    if op == "gemm":
        return a @ w.T.contiguous()
    gate, up = (a @ half.T.contiguous() for half in w.chunk(2))
    return gate * torch.sigmoid(gate) * up
