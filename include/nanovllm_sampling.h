/*
 * nanovllm_sampling.h — C ABI of the sampler on logits: a token a row by
 * temperature, top-k, top-p and min-p from a given random number.  Part of
 * libnanovllm_gemm.so; conventions as in nanovllm_gemm.h.  Asynchronous,
 * allocates nothing, can be captured into a HIP graph.
 *
 * Reference interface beside which it stands: Sampler.forward
 * (nanovllm/layers/sampler.py:8-21), which knows the temperature alone.
 */
#ifndef NANOVLLM_SAMPLING_H
#define NANOVLLM_SAMPLING_H

#include "nanovllm_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Row i of logits [m, vocab] (f32, f16 or bf16, row stride ld) has temperature
 * T = temperatures[i] and random number u = uniforms[i] in [0, 1).
 *
 * T <= 1e-10 (or NaN): tokens[i] is the largest logit, the first of equals, and
 * logprobs[i] 0.  Otherwise the tokens, in the order of their logits from the
 * largest down (the first index first among equals), have weights
 * exp((l - max l) / T); one below 2^-63 may count as 0.  Kept are
 *     the first top_k[i] (all where that is 0 or less),
 *     of these the shortest run from the front whose weights reach the share
 *         top_p[i] of theirs (all where that is 1 or more, or NaN; always the
 *         first),
 *     of these the ones of a weight of at least min_p[i] (all where that is 0
 *         or less, or NaN; always the first).
 * tokens[i] is the first token, by index, at which the running sum of the kept
 * weights is above u times their total; logprobs[i] the natural logarithm of
 * its share of that total.  top_k, top_p and min_p may be null (off).
 *
 * -inf: weight 0.  A row whose largest logit is an infinity draws among the
 * tokens that hold it.  A row with a NaN takes its first NaN, with logprob NaN.
 * u below 0 or NaN counts as 0, u of 1 or more takes the last kept token.
 *
 * Weights are off by less than 2^-32 of themselves (2^-25 where T is above
 * 2^100), their sums are held in 64 bits, and no sum depends on the order in
 * which workgroups run.  Workspace: nanovllm_sample_logits_workspace_bytes()
 * bytes, 16-byte aligned scratch.  vocab is at most 2^23.
 */
int nanovllm_sample_logits(const void* logits, const float* temperatures, const float* uniforms,
                           const int32_t* top_k, const float* top_p, const float* min_p,
                           int64_t* tokens, float* logprobs,
                           int64_t m, int64_t vocab, int64_t ld, int dtype,
                           void* workspace, int64_t workspace_bytes, void* stream);

/* Workspace bytes of nanovllm_sample_logits, or the negative code that it
 * returns for a call of these sizes.  Pure host function. */
int64_t nanovllm_sample_logits_workspace_bytes(int64_t m, int64_t vocab, int dtype);

#ifdef __cplusplus
}
#endif

#endif /* NANOVLLM_SAMPLING_H */
