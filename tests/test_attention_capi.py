"""CPU tests of the attention operators' C ABI: every argument is checked on
the host before anything is launched, plainly and under the host sanitizers.
No test here launches a kernel."""
from __future__ import annotations

import ctypes
import os
import subprocess
import sys

import pytest

from conftest import PKG, ROOT

L = PKG._lib
P = 1 << 20        # a device pointer that is never followed


def _cache(**changes):
    bits, dim = changes.get("bits", 16), changes.get("head_dim", 128)
    size, heads = changes.get("block_size", 16), changes.get("kv_heads", 2)
    page = size * heads * dim * 2 if bits == 16 else size * heads * dim // 2
    scales = size * heads * dim // 64 * 4 if bits == 4 else 0
    fields = dict(k=P, v=P, k_scales=P if bits == 4 else None, v_scales=P if bits == 4 else None, num_blocks=4,
                  block_size=size, kv_heads=heads, head_dim=dim, k_stride=page, v_stride=page, k_scales_stride=scales,
                  v_scales_stride=scales, bits=bits, dtype=L.BF16)
    fields.update(changes)
    return ctypes.byref(L.KvCacheStruct(**fields))


def _append(cache=None, **changes):
    a = dict(q=P, k=P, v=P, positions=P, cos_sin=P, slots=P, q_out=P, k_out=P, cache=cache or _cache(), tokens=3,
             heads=4, q_row=512, q_head=128, k_row=256, k_head=128, v_row=256, v_head=128, positions_max=10, rotary=64)
    a.update(changes)
    return L.load().nanovllm_rope_append(*a.values(), None)


def _prompt(**changes):
    a = dict(q=P, k=P, v=P, cu_q=P, cu_k=P, out=P, batch=1, q_rows=3, k_rows=3, heads=4, kv_heads=2, head_dim=128,
             q_row=512, q_head=128, k_row=256, k_head=128, v_row=256, v_head=128, scale=0.1, causal=1, dtype=L.BF16,
             workspace=P, workspace_bytes=1 << 30)
    a.update(changes)
    return L.load().nanovllm_attention_prompt(*a.values(), None)


def _paged(cache=None, **changes):
    a = dict(q=P, cache=cache or _cache(), tables=P, lens=P, out=P, batch=2, heads=4, table_blocks=20, table_stride=20,
             q_row=512, q_head=128, scale=0.1, dtype=L.BF16, workspace=P, workspace_bytes=1 << 30)
    a.update(changes)
    return L.load().nanovllm_attention_paged(*a.values(), None)


def _gather(cache=None, **changes):
    a = dict(cache=cache or _cache(), slots=P, rows=3, k_out=P, v_out=P, dtype=L.BF16)
    a.update(changes)
    return L.load().nanovllm_kv_gather(*a.values(), None)


BAD_CACHES = [
    (dict(bits=8), L.EUNSUPPORTED, "16 or 4 bits"),
    (dict(dtype=L.F32), L.EUNSUPPORTED, "f16 or bf16"),
    (dict(head_dim=96), L.EUNSUPPORTED, "head_dim"),
    (dict(num_blocks=0), L.EINVAL, "slots"),
    (dict(num_blocks=2 ** 28), L.EINVAL, "slots"),
    (dict(num_blocks=2 ** 62), L.EINVAL, "slots"),
    (dict(block_size=0), L.EINVAL, "slots"),
    (dict(kv_heads=0), L.EINVAL, "kv_heads"),
    (dict(bits=4, block_size=24), L.EUNSUPPORTED, "multiple of 16"),
    (dict(k_stride=16 * 2 * 128 * 2 - 16), L.EINVAL, "strides"),
    (dict(v_stride=16 * 2 * 128 * 2 + 8), L.EINVAL, "strides"),
    (dict(bits=4, v_scales_stride=0), L.EINVAL, "strides"),
    (dict(k_stride=2 ** 36), L.EUNSUPPORTED, "64 GiB"),
    (dict(bits=4, v_scales_stride=2 ** 40), L.EUNSUPPORTED, "64 GiB"),
    (dict(k=None), L.EINVAL, "non-null"),
    (dict(v=P + 8), L.EINVAL, "16-byte aligned"),
    (dict(bits=4, k_scales=None), L.EINVAL, "non-null"),
]


@pytest.mark.parametrize("fields,code,message", BAD_CACHES, ids=lambda x: str(x))
def test_bad_caches_are_refused(lib, fields, code, message):
    for call in (_append, _gather, _paged):
        assert call(_cache(**fields)) == code
        assert message in L.last_error()


@pytest.mark.parametrize("call,changes,code,message", [
    (_append, dict(cache=None), None, None),
    (_append, dict(tokens=-1), L.EINVAL, "tokens"),
    (_append, dict(tokens=2 ** 31), L.EINVAL, "tokens"),
    (_append, dict(tokens=2 ** 29), L.EINVAL, "2^31"),
    (_append, dict(heads=3), L.EINVAL, "multiple of kv_heads"),
    (_append, dict(heads=0), L.EINVAL, "multiple of kv_heads"),
    (_append, dict(q_row=4), L.EINVAL, "strides of q"),
    (_append, dict(k_head=-8), L.EINVAL, "strides of k"),
    (_append, dict(v_row=12), L.EINVAL, "strides of v"),
    (_append, dict(q_row=2 ** 24), L.EUNSUPPORTED, "2^24"),
    (_append, dict(tokens=2 ** 27), L.EUNSUPPORTED, "too many"),
    (_append, dict(rotary=0), L.EINVAL, "rotary"),
    (_append, dict(rotary=24), L.EINVAL, "rotary"),
    (_append, dict(rotary=144), L.EINVAL, "rotary"),
    (_append, dict(positions_max=0), L.EINVAL, "positions_max"),
    (_append, dict(slots=None), L.EINVAL, "non-null"),
    (_append, dict(q=P + 2), L.EINVAL, "aligned"),
    (_append, dict(tokens=0, q=None), L.OK, ""),
    (_gather, dict(rows=-1), L.EINVAL, "rows"),
    (_gather, dict(rows=2 ** 30), L.EINVAL, "2^31"),
    (_gather, dict(rows=2 ** 28), L.EUNSUPPORTED, "too many"),
    (_gather, dict(dtype=L.F16), L.EUNSUPPORTED, "own dtype"),
    (_gather, dict(slots=None), L.EINVAL, "non-null"),
    (_gather, dict(rows=0, k_out=None), L.OK, ""),
    (_prompt, dict(dtype=L.F32), L.EUNSUPPORTED, "f16 or bf16"),
    (_prompt, dict(head_dim=80), L.EUNSUPPORTED, "head_dim"),
    (_prompt, dict(kv_heads=3), L.EINVAL, "multiple"),
    (_prompt, dict(scale=0.0), L.EINVAL, "scale"),
    (_prompt, dict(scale=float("nan")), L.EINVAL, "scale"),
    (_prompt, dict(scale=float("inf")), L.EINVAL, "scale"),
    (_prompt, dict(scale=3e38), L.EINVAL, "scale"),
    (_prompt, dict(scale=-1.0), L.EINVAL, "scale"),
    (_prompt, dict(batch=-1), L.EINVAL, "batch"),
    (_prompt, dict(q_rows=2 ** 31), L.EINVAL, "rows"),
    (_prompt, dict(k_rows=5000, workspace=None), L.EINVAL, "workspace"),
    (_prompt, dict(k_rows=5000, workspace_bytes=100), L.EINVAL, "workspace"),
    (_prompt, dict(k_row=2 ** 24), L.EUNSUPPORTED, "2^24"),
    (_prompt, dict(batch=2 ** 22), L.EUNSUPPORTED, "too many"),
    (_prompt, dict(k=None), L.EINVAL, "non-null"),
    (_prompt, dict(k_row=3), L.EINVAL, "strides of k"),
    (_prompt, dict(q_rows=0, q=None, out=None), L.OK, ""),
    (_paged, dict(cache=_cache(block_size=24)), L.EUNSUPPORTED, "multiple of 16"),
    (_paged, dict(batch=-1), L.EINVAL, "batch"),
    (_paged, dict(batch=2 ** 31), L.EINVAL, "batch"),
    (_paged, dict(table_blocks=2 ** 28), L.EINVAL, "2^31"),
    (_paged, dict(batch=2 ** 23, table_blocks=1, table_stride=1), L.EUNSUPPORTED, "too large"),
    (_paged, dict(batch=2 ** 20, table_blocks=2 ** 20, table_stride=2 ** 20), L.EUNSUPPORTED, "too large"),
    (_paged, dict(table_stride=19), L.EINVAL, "table_stride"),
    (_paged, dict(workspace=None), L.EINVAL, "workspace"),
    (_paged, dict(workspace_bytes=16), L.EINVAL, "workspace"),
    (_paged, dict(dtype=L.F16), L.EUNSUPPORTED, "dtype"),
    (_paged, dict(scale=0.0), L.EINVAL, "scale"),
    (_paged, dict(lens=None), L.EINVAL, "non-null"),
    (_paged, dict(batch=0, q=None, out=None), L.OK, ""),
], ids=lambda x: getattr(x, "__name__", str(x)))
def test_bad_arguments_are_refused(lib, call, changes, code, message):
    if code is None:       # no cache at all
        assert L.load().nanovllm_rope_append(*[P] * 8, None, *[0] * 10, None) == L.EINVAL
        assert "cache" in L.last_error()
        return
    assert call(**changes) == code
    assert message in L.last_error()


def test_paged_workspace(lib):
    need = L.attention_paged_workspace_bytes
    # A table of one unit of tokens leaves nothing to join.
    assert need(_cache(), 8, 4, 8) == 0
    one = need(_cache(), 1, 4, 16)
    assert one > 0 and one % 16 == 0
    # Bounded by the grid, whatever the batch and the table.
    assert need(_cache(), 1000, 4, 1000) == need(_cache(), 4000, 4, 9000)
    assert need(_cache(bits=4), 1, 4, 16) == one
    assert need(_cache(head_dim=96), 1, 4, 16) == L.EUNSUPPORTED and "head_dim" in L.last_error()


def test_prompt_workspace(lib):
    need = L.attention_prompt_workspace_bytes
    assert need(1, 0, 0, 4, 2, 128, L.BF16) == 0
    small = need(1, 5, 2000, 1, 1, 128, L.BF16)
    assert 0 < small < need(1, 500, 3000, 4, 2, 128, L.BF16)
    # Bounded by the grid, whatever the keys; none where every workgroup has a block of its own: few keys, many blocks.
    assert need(1, 500, 500, 4, 2, 128, L.BF16) == need(3, 900, 900, 4, 2, 64, L.BF16) == 0
    assert need(1, 512, 10 ** 4, 32, 8, 128, L.BF16) == need(1, 600, 10 ** 9, 32, 8, 128, L.BF16) < 1 << 27
    assert need(9, 10 ** 7, 10 ** 9, 64, 8, 128, L.BF16) == 0
    assert need(1, 5, 5, 3, 2, 128, L.BF16) == L.EINVAL and "multiple" in L.last_error()


CHILD = r"""
import sys
import pytest
sys.path.insert(0, {root!r})
rc = pytest.main(["-q", "-p", "no:cacheprovider", "-k", "not sanitized", {tests!r}])
sys.exit(int(rc))
"""


def test_attention_capi_sanitized(tmp_path):
    """The tests above against a library whose host code carries AddressSanitizer and UndefinedBehaviorSanitizer."""
    import importlib
    build = importlib.import_module("inference_systems_amd.build")
    try:
        runtime = build.sanitizer_runtime()
        build.hipcc()
    except RuntimeError as exc:
        pytest.skip(str(exc))
    library = build.build(sanitize=True, out=tmp_path / "libnanovllm_gemm.so")
    env = dict(os.environ, LD_PRELOAD=str(runtime), ASAN_OPTIONS="detect_leaks=0:halt_on_error=1",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1", NANOVLLM_GEMM_LIB=str(library))
    proc = subprocess.run([sys.executable, "-c", CHILD.format(root=str(ROOT), tests=__file__)], env=env,
                          capture_output=True, text=True, timeout=600, cwd=str(tmp_path))
    out = proc.stdout + proc.stderr
    assert proc.returncode == 0 and "passed" in proc.stdout, out[-4000:]
    assert "AddressSanitizer" not in out and "runtime error:" not in out, out[-4000:]
