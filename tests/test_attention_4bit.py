"""A 4-bit cache byte for byte."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import PKG
from oracle import attention_oracle as orc

K = PKG.kernels
BF16, F16 = torch.bfloat16, torch.float16
IDS = {BF16: "bf16", F16: "f16"}


def _say(*what):
    print(*what, flush=True)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _numpy(cache):
    return [t.cpu().numpy().copy() for t in cache]


def _still(device):
    """A table that turns by nothing."""
    return torch.cat((torch.ones(1, 16), torch.zeros(1, 16)), 1).to(device)


def _append(k, v, slots, cache, backend):
    at = torch.zeros(k.shape[0], dtype=torch.int64, device=k.device)
    K.rope_append_kv(k, k, v, at, _still(k.device), slots, cache, backend=backend)


# ---------------------------------------------------------------------------
# rope_append: every byte
# ---------------------------------------------------------------------------
def _noisy(cache, gen):
    """Contents that no call may change: any codes, scales with NaN among them."""
    out = []
    for t in cache:
        if t.dtype == torch.uint8:
            out.append(torch.randint(0, 256, t.shape, generator=gen, dtype=torch.uint8))
        else:
            x = torch.randn(t.shape, generator=gen).to(t.dtype)
            out.append(torch.where(torch.rand(t.shape, generator=gen) < 0.3, torch.nan, x))
    return out


def _slots(kind, tokens, capacity, gen):
    if kind == "random":
        return torch.randperm(capacity, generator=gen)[:tokens]
    slots = torch.arange(tokens) + (0 if kind == "aligned" else 3)
    if tokens > 9:
        slots[tokens // 2], slots[tokens // 2 + 4] = -1, capacity + 7
    return slots


def _append_and_compare(device, backend, dtype, dim, kv, size, tokens, kind):
    gen = _gen(tokens * dim + kv)
    blocks = -(-60 // size)
    k, v = (torch.randn((tokens, kv, dim), generator=gen).to(dtype) for _ in range(2))
    if tokens > 5:
        v[3, 0, dim // 2], v[5] = torch.nan, 2.0
    table, positions = K.rope_table(500, 32), torch.randint(0, 500, (tokens,), generator=gen)
    if tokens > 2:
        positions[1], positions[2] = 500, -1       # outside the table: NaN in the group that turns
    slots = _slots(kind, tokens, blocks * size, gen)
    want = _noisy(K.new_kv_cache(blocks, size, kv, dim, bits=4), gen)
    cache = K.KVCache(*[t.to(device) for t in want])
    want = [t.numpy() for t in want]
    K.rope_append_kv(k.to(device), k.to(device), v.to(device), positions.to(device), table.to(device),
                     slots.to(torch.int32).to(device), cache, backend=backend)
    turned = orc.rotate(k, positions.tolist(), table)
    for t, s in enumerate(slots.tolist()):
        for h in range(kv):
            if 0 <= s < blocks * size:
                orc.write_row(want, s, h, turned[t, h].float().numpy(), v[t, h].float().numpy())
    got = _numpy(cache)
    for name, a, b in zip(("k", "v"), got, want):
        assert np.array_equal(a, b), name      # codes of a group with a NaN are 0
    for name, a, b in zip(("k_scales", "v_scales"), got[2:], want[2:]):
        same = (a.view(np.uint16) == b.view(np.uint16)) | (np.isnan(a) & np.isnan(b))
        assert same.all(), name


APPENDED = [(tokens, kind) for tokens in (1, 7, 41) for kind in ("aligned", "shifted", "random")]


@pytest.mark.parametrize("dim,kv,size", [(64, 3, 16), (128, 2, 48)])
@pytest.mark.parametrize("tokens,kind", APPENDED)
def test_torch_backend_leaves_every_other_byte(dim, kv, size, tokens, kind):
    _append_and_compare("cpu", "torch", BF16, dim, kv, size, tokens, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("dim,kv,size", [(64, 3, 16), (128, 2, 48), (256, 1, 16), (128, 5, 256)])
@pytest.mark.parametrize("tokens,kind", APPENDED)
def test_append_leaves_every_other_byte(dtype, dim, kv, size, tokens, kind):
    """Written rows by the oracle, every other byte as it was: words that four tokens share among them."""
    _say("every byte", dtype, dim, kv, size, tokens, kind)
    _append_and_compare("cuda:0", "hip", dtype, dim, kv, size, tokens, kind)
