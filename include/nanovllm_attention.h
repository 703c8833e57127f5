/*
 * nanovllm_attention.h — C ABI of the operators between the projections of a
 * Qwen3.5 gated-attention layer: rotation and cache append, cache reads,
 * attention over packed prompts and attention over a paged cache.  They are
 * part of libnanovllm_gemm.so and follow nanovllm_gemm.h: plain device
 * pointers, sizes and an opaque HIP stream, negative return codes with
 * nanovllm_gemm_last_error(), the dtype and return codes of that header.
 * Every entry point is asynchronous, allocates nothing and can be captured
 * into a HIP graph.
 *
 * Reference interfaces these replace (paths relative to the reference repo):
 *   - nanovllm/layers/rotary_embedding.py, nanovllm/layers/attention.py:10-40
 *     the rotation and the store_kvcache kernel;
 *   - nanovllm/layers/attention.py, the flash-attention calls of
 *     Qwen3_5Attention (nanovllm/models/qwen3_5.py:81-96).
 */
#ifndef NANOVLLM_ATTENTION_H
#define NANOVLLM_ATTENTION_H

#include "nanovllm_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * A paged cache of keys and values.  Slot s is row s % block_size of page
 * s / block_size; there are fewer than 2^31.  Strides between pages are in
 * bytes, a multiple of 16 below 64 GiB, pages smaller than 2 GiB; pointers are
 * 16-byte aligned; head_dim is 64, 128 or 256.
 *
 * bits == 16: a page of k, and of v, is [block_size, kv_heads, head_dim]
 * elements of dtype (the layout of store_kvcache); the scales are null.
 *
 * bits == 4 (block_size a multiple of 16): an element stands for
 * code * scale + minimum, with 4-bit codes and one float16 scale and minimum
 * per token and group of 64 channels.
 *   k         [kv_heads, block_size, head_dim / 2] bytes.  A 32-bit word holds
 *             8 channels, channel j at bits 4 (j / 2) + 16 (j % 2).
 *   v         [kv_heads, block_size / 4, head_dim / 2, 4] bytes.  A 32-bit word
 *             holds 2 channels of 4 tokens, a byte a token, the even channel in
 *             the low 4 bits.
 *   k_scales  [kv_heads, block_size, head_dim / 64, 2] float16
 *   v_scales  [kv_heads, head_dim / 64, block_size, 2] float16
 * The words of a row lie in channel order, except that those of two
 * neighbouring groups take turns two by two: with u = 8 (k) or 32 (v) words a
 * group, words g0.0 g0.1 g1.0 g1.1 g0.2 g0.3 g1.2 g1.3 ... of a block of 128
 * channels.
 */
typedef struct nanovllm_kv_cache {
    void* k;
    void* v;
    void* k_scales;
    void* v_scales;
    int64_t num_blocks;
    int64_t block_size;
    int64_t kv_heads;
    int64_t head_dim;
    int64_t k_stride;
    int64_t v_stride;
    int64_t k_scales_stride;
    int64_t v_scales_stride;
    int bits;
    int dtype;
} nanovllm_kv_cache;

/*
 * Rotates queries and keys and appends keys and values to the cache.  q is
 * [tokens, heads, head_dim], k and v [tokens, kv_heads, head_dim], of dtype,
 * element (t, h, c) at t * row stride + h * head stride + c (strides in
 * elements, multiples of 8, that of rows below 2^24).  With x1, x2 the two halves of the first
 * `rotary` channels (a multiple of 16, at most head_dim),
 *     y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin,
 * in fp32, rounded once; the other channels stay.  Row p of cos_sin
 * [positions_max, rotary] holds the cosines and the sines of position p.
 * q_out [tokens, heads, head_dim] and k_out [tokens, kv_heads, head_dim] are
 * contiguous.  The rotated, rounded keys and the values go to slots[t]; a
 * negative slot, or one behind the cache, takes none (padding), and the slots
 * of one call are distinct.  A position outside the table turns by NaN.
 *
 * 4 bits: a group x of 64 channels of a row, clamped to float16's finite range,
 * is kept as minimum m = f16(min x), scale s = f16((max x - min x) / 15), or
 * the float16 below it where 15 s + m passes 65504, and codes
 * clamp(rint((x - m) / s), 0, 15), 0 where s is 0.  So what a code stands for is
 * in float16's finite range too.  A NaN in the group makes all of it NaN.
 */
int nanovllm_rope_append(const void* q, const void* k, const void* v,
                         const int64_t* positions, const float* cos_sin, const int32_t* slots,
                         void* q_out, void* k_out, const nanovllm_kv_cache* cache,
                         int64_t tokens, int64_t heads,
                         int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head,
                         int64_t v_row, int64_t v_head,
                         int64_t positions_max, int64_t rotary, void* stream);

/* Whether nanovllm_rope_append takes a call of these sizes: OK, or the code it
 * would return.  Pure host function; the cache's pointers are not looked at. */
int nanovllm_rope_append_check(const nanovllm_kv_cache* cache, int64_t tokens, int64_t heads);

/*
 * Rows of the cache as packed keys and values: k_out and v_out [rows,
 * kv_heads, head_dim] of dtype (the cache's in 16 bits) hold row slots[i] of
 * the cache, or zeros where slots[i] is negative or behind the cache.
 */
int nanovllm_kv_gather(const nanovllm_kv_cache* cache, const int32_t* slots, int64_t rows,
                       void* k_out, void* v_out, int dtype, void* stream);

/* Whether nanovllm_kv_gather takes a call of these sizes, as above. */
int nanovllm_kv_gather_check(const nanovllm_kv_cache* cache, int64_t rows);

/*
 * Attention of packed sequences, heads in groups of heads / kv_heads that
 * share keys and values.  Sequence b holds queries cu_q[b] .. cu_q[b + 1] and
 * keys cu_k[b] .. cu_k[b + 1] (batch + 1 offsets each, not decreasing, the
 * first of cu_q 0); its row i attends to key j where causal is 0 or
 * j <= i + (keys - queries), so the last query sees every key.
 * out = softmax(scale q k^T) v; a row with no key to attend to is 0, and so are
 * rows behind the last sequence.  Scores, maxima, totals and sums are fp32; the
 * weights are rounded to dtype before they multiply v (the total is that of the
 * rounded ones), and out is rounded once.  q, k, v as in
 * nanovllm_rope_append; out is [q_rows, heads, head_dim], contiguous.
 * Workspace: nanovllm_attention_prompt_workspace_bytes() bytes, 16-byte
 * aligned scratch.
 */
int nanovllm_attention_prompt(const void* q, const void* k, const void* v,
                              const int32_t* cu_q, const int32_t* cu_k, void* out,
                              int64_t batch, int64_t q_rows, int64_t k_rows,
                              int64_t heads, int64_t kv_heads, int64_t head_dim,
                              int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head,
                              int64_t v_row, int64_t v_head,
                              float scale, int causal, int dtype,
                              void* workspace, int64_t workspace_bytes, void* stream);

/* Workspace bytes of nanovllm_attention_prompt, or the negative code that it
 * returns for a call of these sizes.  Pure host function. */
int64_t nanovllm_attention_prompt_workspace_bytes(int64_t batch, int64_t q_rows, int64_t k_rows, int64_t heads,
                                                  int64_t kv_heads, int64_t head_dim, int dtype);

/*
 * Attention of one query token per sequence over its cached tokens: out[b, h]
 * = softmax(scale q[b, h] k^T) v over the first lens[b] tokens of pages
 * tables[b, 0 .. table_blocks) (row stride table_stride, in entries).  Page
 * sizes are multiples of 16, and a table holds at most 2^31 - 1024 tokens.  No
 * token: 0.  A page number outside the cache, or a length behind the table,
 * makes the sequence's output NaN.  Roundings as above on 16-bit pages; on 4-bit
 * ones weights, weights times scales, and minimum + 7.5 scale are rounded to
 * float16, whatever the dtype of q.  q is [batch, heads, head_dim] with strides
 * as above, out contiguous.  Workspace:
 * nanovllm_attention_paged_workspace_bytes() bytes, 16-byte aligned scratch.
 */
int nanovllm_attention_paged(const void* q, const nanovllm_kv_cache* cache,
                             const int32_t* tables, const int32_t* lens, void* out,
                             int64_t batch, int64_t heads, int64_t table_blocks, int64_t table_stride,
                             int64_t q_row, int64_t q_head, float scale, int dtype,
                             void* workspace, int64_t workspace_bytes, void* stream);

/* Workspace bytes of nanovllm_attention_paged, or the negative code that it
 * returns for a call of these sizes.  Pure host function. */
int64_t nanovllm_attention_paged_workspace_bytes(const nanovllm_kv_cache* cache, int64_t batch, int64_t heads,
                                                 int64_t table_blocks);

#ifdef __cplusplus
}
#endif

#endif /* NANOVLLM_ATTENTION_H */
