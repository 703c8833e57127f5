/*
 * nanovllm_int8.h — C ABI of the 8-bit products: rows in 8 bits with a scale
 * each (from plain rows, or behind the residual add and RMSNorm), and the GEMM
 * of such rows with 8-bit weights.  They are part of libnanovllm_gemm.so and
 * follow nanovllm_gemm.h: plain device pointers, sizes and an opaque HIP
 * stream, negative return codes with nanovllm_gemm_last_error(), the dtype and
 * return codes of that header.  Every entry point is asynchronous, allocates
 * nothing and can be captured into a HIP graph.
 *
 * Reference interfaces beside which these stand (paths relative to the
 * reference repo): the F.linear call sites of nanovllm/layers/linear.py:51, 73,
 * 153 and nanovllm/layers/embed_head.py:61, the norm of
 * nanovllm/layers/layernorm.py:131-142 in front of them and SiluAndMul
 * (nanovllm/layers/activation.py:8-11) behind gate_up_proj.
 *
 * A row x in 8 bits: scale s = max |x| / 127 in fp32, codes
 * clamp(rint(x / s), -127, 127), the quotient exact (ties to even); a code
 * stands for code * s.  A row of zeros, or one whose scale rounds to 0, has
 * scale 0 and codes 0.  A row with a NaN or an infinity has scale NaN and codes
 * 0, so every output made of it is NaN.
 */
#ifndef NANOVLLM_INT8_H
#define NANOVLLM_INT8_H

#include "nanovllm_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Rows of x [m, k] (dtype f32, f16 or bf16; element (i, c) at x[i * ldx + c])
 * in 8 bits: codes [m, k] contiguous, scales [m].
 */
int nanovllm_quantize_rows(const void* x, int8_t* codes, float* scales,
                           int64_t m, int64_t k, int64_t ldx, int dtype, void* stream);

/*
 * Residual add and zero-centred RMSNorm with the result in 8 bits: with
 * s = h + r in fp32, residual_out = round(s), and the row
 *     s * (1 + w) * rsqrt(mean(s^2) + eps)
 * in 8 bits as above, from fp32 (it is rounded to no other type; where the sum
 * of squares passes fp32 it is a row of zeros).  h, r, w and
 * residual_out are of dtype (f16 or bf16); h and r have row strides ldh and
 * ldr; codes and residual_out are contiguous [m, k].  residual_out must not
 * overlap the span of h or of r (refused); nor may any output of these entry
 * points overlap an input.
 */
int nanovllm_add_rmsnorm_quantize(const void* h, const void* r, const void* w, float eps,
                                  int8_t* codes, float* scales, void* residual_out,
                                  int64_t m, int64_t k, int64_t ldh, int64_t ldr, int dtype, void* stream);

/*
 * c[i, j] = round(a_scales[i] * w_scales[j] * sum_k a[i, k] * w[j, k]) with a
 * [m, k] and w [n, k] (row strides lda, ldw, in elements) of int8, the sum in
 * int32 (exact: k is below 131072), the scales applied in fp32.  With silu_mul
 * w is [w_gate; w_up], 2n rows, and c[i, j] = round(silu(g) * u) of the scaled
 * gate and up sums.  c is [m, n] of dtype_out (f32, f16 or bf16), row stride
 * ldc.  Rows that are whole aligned 16-byte chunks (k, lda and ldw multiples of
 * 16, a and w 16-byte aligned) take the fast kernels, any others a kernel of
 * their own.
 */
int nanovllm_gemm_int8(const int8_t* a, const float* a_scales, const int8_t* w, const float* w_scales, void* c,
                       int64_t m, int64_t n, int64_t k, int64_t lda, int64_t ldw, int64_t ldc,
                       int silu_mul, int dtype_out, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* NANOVLLM_INT8_H */
