// C ABI of the 8-bit products and of the sampler: argument validation, the
// choice of a GEMM kernel and dispatch to the launchers.  Declarations:
// include/nanovllm_int8.h, include/nanovllm_sampling.h.
#include <hip/hip_runtime.h>

#include <cmath>

#include "int8_common.hpp"

namespace nvg {
namespace {

bool is_half(int dt) { return dt == NANOVLLM_GEMM_F16 || dt == NANOVLLM_GEMM_BF16; }
bool is_float(int dt) { return dt == NANOVLLM_GEMM_F32 || is_half(dt); }
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
int element_bytes(int dt) { return dt == NANOVLLM_GEMM_F32 ? 4 : 2; }

// Rows of k elements; a launch has a workgroup for at most one row.
int check_rows(const char* op, int64_t m, int64_t k) {
    if (m < 0 || m > (int64_t(1) << 23))
        return set_error(NANOVLLM_GEMM_EINVAL, "%s: m (%lld) must be from 0 to 2^23", op, (long long)m);
    if (k < 1 || k > (int64_t(1) << 30))
        return set_error(NANOVLLM_GEMM_EINVAL, "%s: k (%lld) must be from 1 to 2^30", op, (long long)k);
    return NANOVLLM_GEMM_OK;
}

int check_stride(const char* op, const char* name, int64_t ld, int64_t k) {
    if (ld < k || ld > (int64_t(1) << 40))
        return set_error(NANOVLLM_GEMM_EINVAL, "%s: %s (%lld) must be from %lld to 2^40", op, name, (long long)ld,
                         (long long)k);
    return NANOVLLM_GEMM_OK;
}

// Non-null, and aligned to their elements.
int check_pointer(const char* op, const char* name, const void* p, int bytes) {
    if (p == nullptr || reinterpret_cast<uintptr_t>(p) % bytes != 0)
        return set_error(NANOVLLM_GEMM_EINVAL, "%s: %s must be non-null and aligned to its elements", op, name);
    return NANOVLLM_GEMM_OK;
}

// Whether the contiguous [m, k] at `out` shares bytes with the span of m rows of k
// elements at `in`, `ld` apart (positive sizes; all elements of `bytes`).
bool overlaps(const void* out, const void* in, int64_t m, int64_t k, int64_t ld, int bytes) {
    const auto begin = static_cast<__int128>(reinterpret_cast<uintptr_t>(out));
    const auto other = static_cast<__int128>(reinterpret_cast<uintptr_t>(in));
    return begin < other + (static_cast<__int128>(m - 1) * ld + k) * bytes &&
           other < begin + static_cast<__int128>(m) * k * bytes;
}

// Which rows splitk_decode takes, in the units of the bf16 GEMM of the same
// bytes (nanovllm_gemm_select and nanovllm_gemm_silu_mul_select): the weights
// are streamed once up to M = 32, and up to 64 where larger tiles would leave
// CUs idle.
bool decode_rows(int64_t m, int64_t n, int64_t k2, int silu) {
    if (m <= 32) return true;
    if (m > 64) return false;
    if (silu) return 2 * n <= 16384;
    return n <= 4096 || (n <= 10240 && k2 <= 1024);
}

}  // namespace
}  // namespace nvg

extern "C" {

int nanovllm_quantize_rows(const void* x, int8_t* codes, float* scales, int64_t m, int64_t k, int64_t ldx, int dtype,
                           void* stream) {
    using namespace nvg;
    const char* op = "quantize_rows";
    clear_error();
    if (!is_float(dtype))
        return set_error(NANOVLLM_GEMM_EUNSUPPORTED, "%s: dtype must be f32, f16 or bf16, got %d", op, dtype);
    int rc = check_rows(op, m, k);
    if (rc == NANOVLLM_GEMM_OK) rc = check_stride(op, "ldx", ldx, k);
    if (rc != NANOVLLM_GEMM_OK || m == 0) return rc;
    rc = check_pointer(op, "x", x, element_bytes(dtype));
    if (rc == NANOVLLM_GEMM_OK) rc = check_pointer(op, "codes", codes, 1);
    if (rc == NANOVLLM_GEMM_OK) rc = check_pointer(op, "scales", scales, 4);
    if (rc != NANOVLLM_GEMM_OK) return rc;
    return launch_quantize_rows(x, ldx, codes, scales, m, k, dtype, static_cast<hipStream_t>(stream));
}

int nanovllm_add_rmsnorm_quantize(const void* h, const void* r, const void* w, float eps, int8_t* codes, float* scales,
                                  void* residual_out, int64_t m, int64_t k, int64_t ldh, int64_t ldr, int dtype,
                                  void* stream) {
    using namespace nvg;
    const char* op = "add_rmsnorm_quantize";
    clear_error();
    if (!is_half(dtype)) return set_error(NANOVLLM_GEMM_EUNSUPPORTED, "%s: dtype must be f16 or bf16, got %d", op, dtype);
    if (!(eps >= 0.0f) || std::isinf(eps))
        return set_error(NANOVLLM_GEMM_EINVAL, "%s: eps must be finite and not negative", op);
    int rc = check_rows(op, m, k);
    if (rc == NANOVLLM_GEMM_OK) rc = check_stride(op, "ldh", ldh, k);
    if (rc == NANOVLLM_GEMM_OK) rc = check_stride(op, "ldr", ldr, k);
    if (rc != NANOVLLM_GEMM_OK || m == 0) return rc;
    for (const void* p : {h, r, w, static_cast<const void*>(residual_out)})
        if (rc == NANOVLLM_GEMM_OK) rc = check_pointer(op, "h, r, w and residual_out", p, 2);
    if (rc == NANOVLLM_GEMM_OK) rc = check_pointer(op, "codes", codes, 1);
    if (rc == NANOVLLM_GEMM_OK) rc = check_pointer(op, "scales", scales, 4);
    if (rc != NANOVLLM_GEMM_OK) return rc;
    if (overlaps(residual_out, h, m, k, ldh, 2) || overlaps(residual_out, r, m, k, ldr, 2))
        return set_error(NANOVLLM_GEMM_EINVAL, "%s: residual_out must not overlap h or r", op);
    return launch_add_rmsnorm_quantize(h, ldh, r, ldr, w, eps, codes, scales, residual_out, m, k, dtype,
                                       static_cast<hipStream_t>(stream));
}

int nanovllm_gemm_int8(const int8_t* a, const float* a_scales, const int8_t* w, const float* w_scales, void* c,
                       int64_t m, int64_t n, int64_t k, int64_t lda, int64_t ldw, int64_t ldc, int silu_mul,
                       int dtype_out, void* stream) {
    using namespace nvg;
    const char* op = "gemm_int8";
    clear_error();
    if (!is_float(dtype_out))
        return set_error(NANOVLLM_GEMM_EUNSUPPORTED, "%s: dtype_out must be f32, f16 or bf16, got %d", op, dtype_out);
    constexpr int64_t kMost = int64_t(1) << 31;
    if (m < 0 || n < 0 || m >= kMost || n >= kMost / 2)
        return set_error(NANOVLLM_GEMM_EINVAL, "%s: m and n must be non-negative, m below 2^31 and n below 2^30 "
                         "(m=%lld, n=%lld)", op, (long long)m, (long long)n);
    // A sum of 2^17 products of 2^14 each would pass int32.
    if (k < 1 || k >= 131072)
        return set_error(NANOVLLM_GEMM_EINVAL, "%s: k (%lld) must be from 1 to 131071", op, (long long)k);
    int rc = check_stride(op, "lda", lda, k);
    if (rc == NANOVLLM_GEMM_OK) rc = check_stride(op, "ldw", ldw, k);
    if (rc == NANOVLLM_GEMM_OK) rc = check_stride(op, "ldc", ldc, n);
    if (rc != NANOVLLM_GEMM_OK || m == 0 || n == 0) return rc;
    rc = check_pointer(op, "a", a, 1);
    if (rc == NANOVLLM_GEMM_OK) rc = check_pointer(op, "w", w, 1);
    if (rc == NANOVLLM_GEMM_OK) rc = check_pointer(op, "c", c, element_bytes(dtype_out));
    if (rc == NANOVLLM_GEMM_OK) rc = check_pointer(op, "a_scales", a_scales, 4);
    if (rc == NANOVLLM_GEMM_OK) rc = check_pointer(op, "w_scales", w_scales, 4);
    if (rc != NANOVLLM_GEMM_OK) return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (k % 16 || lda % 16 || ldw % 16 || !aligned16(a) || !aligned16(w))
        return launch_int8_any({a, w, a_scales, w_scales, c, m, n, k, lda, ldw, ldc, silu_mul != 0, dtype_out}, s);
    Problem p{};
    p.a = a;
    p.b = w;
    p.c = c;
    p.m = m;
    p.n = n;
    p.k = k / 2;
    p.lda = lda / 2;
    p.ldb = ldw / 2;
    p.ldc = ldc;
    p.b_layout = NANOVLLM_GEMM_B_NK;
    p.dtype_in = kI8;
    p.dtype_out = dtype_out;
    p.epi = silu_mul ? EPI_SILU_MUL : EPI_NONE;
    p.row_scale = a_scales;
    p.col_scale = w_scales;
    return decode_rows(m, n, p.k, silu_mul) ? launch_splitk_decode(p, s) : launch_mfma_staged(p, s);
}

int64_t nanovllm_sample_logits_workspace_bytes(int64_t m, int64_t vocab, int dtype) {
    using namespace nvg;
    const char* op = "sample_logits";
    clear_error();
    if (!is_float(dtype))
        return set_error(NANOVLLM_GEMM_EUNSUPPORTED, "%s: dtype must be f32, f16 or bf16, got %d", op, dtype);
    if (m < 0 || m > (int64_t(1) << 20))
        return set_error(NANOVLLM_GEMM_EINVAL, "%s: m (%lld) must be from 0 to 2^20", op, (long long)m);
    if (vocab < 1 || vocab > (int64_t(1) << 23))
        return set_error(NANOVLLM_GEMM_EINVAL, "%s: vocab (%lld) must be from 1 to 2^23", op, (long long)vocab);
    return m == 0 ? 0 : sample_logits_workspace(m, vocab, dtype);
}

int nanovllm_sample_logits(const void* logits, const float* temperatures, const float* uniforms, const int32_t* top_k,
                           const float* top_p, const float* min_p, int64_t* tokens, float* logprobs, int64_t m,
                           int64_t vocab, int64_t ld, int dtype, void* workspace, int64_t workspace_bytes,
                           void* stream) {
    using namespace nvg;
    const char* op = "sample_logits";
    const int64_t need = nanovllm_sample_logits_workspace_bytes(m, vocab, dtype);
    if (need < 0) return static_cast<int>(need);
    int rc = check_stride(op, "ld", ld, vocab);
    if (rc != NANOVLLM_GEMM_OK || m == 0) return rc;
    rc = check_pointer(op, "logits", logits, element_bytes(dtype));
    for (const void* p : {static_cast<const void*>(temperatures), static_cast<const void*>(uniforms),
                          static_cast<const void*>(logprobs)})
        if (rc == NANOVLLM_GEMM_OK) rc = check_pointer(op, "temperatures, uniforms and logprobs", p, 4);
    if (rc == NANOVLLM_GEMM_OK) rc = check_pointer(op, "tokens", tokens, 8);
    for (const void* p : {static_cast<const void*>(top_k), static_cast<const void*>(top_p),
                          static_cast<const void*>(min_p)})
        if (rc == NANOVLLM_GEMM_OK && p != nullptr) rc = check_pointer(op, "top_k, top_p and min_p", p, 4);
    if (rc != NANOVLLM_GEMM_OK) return rc;
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace)))
        return set_error(NANOVLLM_GEMM_EINVAL, "%s: workspace of %lld bytes (16-byte aligned) needed, got %lld", op,
                         (long long)need, (long long)workspace_bytes);
    return launch_sample_logits({logits, temperatures, uniforms, top_k, top_p, min_p, tokens, logprobs, m, vocab, ld,
                                 dtype, static_cast<char*>(workspace)},
                                static_cast<hipStream_t>(stream));
}

}  // extern "C"
