// Launchers of the 8-bit products and of the sampler that capi_int8.cpp
// dispatches to (arguments already validated).
#pragma once

#include "../../include/nanovllm_int8.h"
#include "../../include/nanovllm_sampling.h"
#include "gemm_common.hpp"

namespace nvg {

int launch_quantize_rows(const void* x, int64_t ldx, int8_t* codes, float* scales, int64_t m, int64_t k, int dtype,
                         hipStream_t s);
int launch_add_rmsnorm_quantize(const void* h, int64_t ldh, const void* r, int64_t ldr, const void* w, float eps,
                                int8_t* codes, float* scales, void* res, int64_t m, int64_t k, int dtype,
                                hipStream_t s);

// Rows of any length and alignment (gemm_int8.hip); lda, ldw in bytes.
struct Int8Args {
    const int8_t *a, *w;
    const float *a_scales, *w_scales;
    void* c;
    int64_t m, n, k, lda, ldw, ldc;
    int silu, dtype_out;
};
int launch_int8_any(const Int8Args& p, hipStream_t s);

struct SampleLogitsArgs {
    const void* logits;
    const float *temperatures, *uniforms;
    const int32_t* top_k;
    const float *top_p, *min_p;
    int64_t* tokens;
    float* logprobs;
    int64_t m, vocab, ld;
    int dtype;
    char* workspace;
};
int64_t sample_logits_workspace(int64_t m, int64_t vocab, int dtype);
int launch_sample_logits(const SampleLogitsArgs& p, hipStream_t s);

// Clears the error text of the calling thread.
void clear_error();

}  // namespace nvg
