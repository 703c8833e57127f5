"""CPU tests of the C ABI of the 8-bit products and of the sampler: every argument is checked on the host before
anything is launched, plainly and under the host sanitizers.  No test here launches a kernel."""
from __future__ import annotations

import importlib
import os
import subprocess
import sys

import pytest

from conftest import PKG, ROOT

L = PKG._lib
P = 1 << 20        # a device pointer that is never followed


def _rows(**changes):
    a = dict(x=P, codes=P, scales=P, m=3, k=10, ldx=10, dtype=L.BF16)
    a.update(changes)
    return L.load().nanovllm_quantize_rows(*a.values(), None)


def _norm(**changes):
    a = dict(h=P, r=P, w=P, eps=1e-6, codes=P, scales=P, residual_out=P, m=3, k=10, ldh=10, ldr=10, dtype=L.BF16)
    a.update(changes)
    return L.load().nanovllm_add_rmsnorm_quantize(*a.values(), None)


def _gemm(**changes):
    a = dict(a=P, a_scales=P, w=P, w_scales=P, c=P, m=3, n=5, k=32, lda=32, ldw=32, ldc=5, silu_mul=0,
             dtype_out=L.BF16)
    a.update(changes)
    return L.load().nanovllm_gemm_int8(*a.values(), None)


def _sample(**changes):
    a = dict(logits=P, temperatures=P, uniforms=P, top_k=None, top_p=None, min_p=None, tokens=P, logprobs=P, m=3,
             vocab=100, ld=100, dtype=L.F32, workspace=P, workspace_bytes=1 << 40)
    a.update(changes)
    return L.load().nanovllm_sample_logits(*a.values(), None)


BAD = [
    (_rows, dict(dtype=3), L.EUNSUPPORTED, "dtype"),
    (_rows, dict(m=-1), L.EINVAL, "m (-1)"),
    (_rows, dict(m=2 ** 23 + 1), L.EINVAL, "2^23"),
    (_rows, dict(k=0), L.EINVAL, "k (0)"),
    (_rows, dict(k=2 ** 31, ldx=2 ** 31), L.EINVAL, "2^30"),
    (_rows, dict(ldx=9), L.EINVAL, "ldx (9)"),
    (_rows, dict(ldx=2 ** 41), L.EINVAL, "2^40"),
    (_rows, dict(x=None), L.EINVAL, "x must be non-null"),
    (_rows, dict(x=P + 1), L.EINVAL, "aligned"),
    (_rows, dict(x=P + 2, dtype=L.F32), L.EINVAL, "aligned"),
    (_rows, dict(codes=None), L.EINVAL, "codes"),
    (_rows, dict(scales=P + 2), L.EINVAL, "scales"),
    (_norm, dict(dtype=L.F32), L.EUNSUPPORTED, "f16 or bf16"),
    (_norm, dict(eps=-1.0), L.EINVAL, "eps"),
    (_norm, dict(eps=float("nan")), L.EINVAL, "eps"),
    (_norm, dict(eps=float("inf")), L.EINVAL, "eps"),
    (_norm, dict(m=-2), L.EINVAL, "m (-2)"),
    (_norm, dict(k=0), L.EINVAL, "k (0)"),
    (_norm, dict(ldh=3), L.EINVAL, "ldh"),
    (_norm, dict(ldr=3), L.EINVAL, "ldr"),
    (_norm, dict(w=None), L.EINVAL, "non-null"),
    (_norm, dict(residual_out=P + 1), L.EINVAL, "aligned"),
    (_norm, dict(scales=None), L.EINVAL, "scales"),
    (_gemm, dict(dtype_out=3), L.EUNSUPPORTED, "dtype_out"),
    (_gemm, dict(m=-1), L.EINVAL, "m and n"),
    (_gemm, dict(n=-1), L.EINVAL, "m and n"),
    (_gemm, dict(n=2 ** 30, ldc=2 ** 30), L.EINVAL, "2^30"),
    (_gemm, dict(k=0), L.EINVAL, "k (0)"),
    (_gemm, dict(k=131072, lda=131072, ldw=131072), L.EINVAL, "131071"),
    (_gemm, dict(lda=31), L.EINVAL, "lda"),
    (_gemm, dict(ldw=31), L.EINVAL, "ldw"),
    (_gemm, dict(ldc=4), L.EINVAL, "ldc"),
    (_gemm, dict(a=None), L.EINVAL, "a must"),
    (_gemm, dict(w=None), L.EINVAL, "w must"),
    (_gemm, dict(c=P + 1), L.EINVAL, "c must"),
    (_gemm, dict(a_scales=None), L.EINVAL, "a_scales"),
    (_gemm, dict(w_scales=P + 1), L.EINVAL, "w_scales"),
    (_sample, dict(dtype=5), L.EUNSUPPORTED, "dtype"),
    (_sample, dict(m=-1), L.EINVAL, "m (-1)"),
    (_sample, dict(m=2 ** 20 + 1), L.EINVAL, "2^20"),
    (_sample, dict(vocab=0), L.EINVAL, "vocab (0)"),
    (_sample, dict(vocab=2 ** 23 + 1, ld=2 ** 24), L.EINVAL, "2^23"),
    (_sample, dict(ld=99), L.EINVAL, "ld (99)"),
    (_sample, dict(logits=None), L.EINVAL, "logits"),
    (_sample, dict(logits=P + 2), L.EINVAL, "logits"),
    (_sample, dict(temperatures=None), L.EINVAL, "temperatures"),
    (_sample, dict(uniforms=P + 1), L.EINVAL, "uniforms"),
    (_sample, dict(top_k=P + 1), L.EINVAL, "top_k"),
    (_sample, dict(min_p=P + 2), L.EINVAL, "min_p"),
    (_sample, dict(logprobs=None), L.EINVAL, "logprobs"),
    (_sample, dict(tokens=P + 4), L.EINVAL, "tokens"),
]


@pytest.mark.parametrize("call,changes,code,message", BAD, ids=[f"{c.__name__}-{ch}" for c, ch, _, _ in BAD])
def test_bad_arguments_are_refused(call, changes, code, message):
    assert call(**changes) == code
    assert message in L.last_error()


@pytest.mark.parametrize("call", [_rows, _norm, _gemm, _sample])
def test_empty_calls_launch_nothing(call):
    assert call(m=0) == L.OK
    assert L.last_error() == ""


def test_no_columns_launch_nothing():
    assert _gemm(n=0) == L.OK


def test_sampler_workspace_is_checked():
    need = L.sample_logits_workspace_bytes(3, 100, L.F32)
    assert need >= 0 and L.sample_logits_workspace_bytes(0, 100, L.F32) == 0
    assert L.sample_logits_workspace_bytes(3, 0, L.F32) == L.EINVAL
    if need:
        assert _sample(workspace=None) == L.EINVAL and "workspace" in L.last_error()
        assert _sample(workspace_bytes=need - 1) == L.EINVAL
        assert _sample(workspace=P + 8) == L.EINVAL


K20 = 20000 * 2    # bytes of a row of 20000


@pytest.mark.parametrize("changes", [dict(h=P), dict(r=P), dict(h=P - 2), dict(r=P + 3 * K20 - 2),
                                     dict(h=P - (2 * 20008 + 19999) * 2, ldh=20008), dict(r=P + 40, ldr=2 ** 40)])
def test_the_sum_does_not_replace_its_terms(changes):
    """residual_out in place of h or r, or next to them by an element: rows too long for the registers are read twice."""
    a = dict(h=P + 100 * K20, r=P + 200 * K20, residual_out=P, m=3, k=20000, ldh=20000, ldr=20000)
    assert _norm(**(a | changes)) == L.EINVAL
    assert "must not overlap" in L.last_error()


CHILD = r"""
import sys
import pytest
sys.path.insert(0, {root!r})
rc = pytest.main(["-q", "-p", "no:cacheprovider", "-k", "not sanitized", {tests!r}])
sys.exit(int(rc))
"""


def test_int8_capi_sanitized(tmp_path):
    """The tests above against a library whose host code carries AddressSanitizer and UndefinedBehaviorSanitizer."""
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
