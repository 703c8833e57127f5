"""CPU tests of how large a call of the attention operators may be: what the
kernels count in 32 bits is refused on the host.  No test here launches a
kernel."""
from __future__ import annotations

import ctypes

import pytest

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
