// C ABI of the attention operators: argument validation and dispatch to the
// launchers.  Declarations: include/nanovllm_attention.h.
#include <hip/hip_runtime.h>

#include <cmath>

#include "attention_common.hpp"

namespace nvg {
namespace {

bool is_half(int dt) { return dt == NANOVLLM_GEMM_F16 || dt == NANOVLLM_GEMM_BF16; }

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

bool fits32(int64_t x) { return x >= 0 && x <= INT32_MAX; }

int check_dims(const char* op, int64_t heads, int64_t kv_heads, int64_t head_dim, int dtype) {
    if (!is_half(dtype)) return set_error(NANOVLLM_GEMM_EUNSUPPORTED, "%s: dtype must be f16 or bf16, got %d", op, dtype);
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return set_error(NANOVLLM_GEMM_EUNSUPPORTED, "%s: head_dim must be 64, 128 or 256, got %lld", op,
                         (long long)head_dim);
    if (kv_heads < 1 || heads < 1 || heads % kv_heads != 0 || heads > 65536)
        return set_error(NANOVLLM_GEMM_EINVAL, "%s: heads (%lld) must be a positive multiple of kv_heads (%lld)", op,
                         (long long)heads, (long long)kv_heads);
    return NANOVLLM_GEMM_OK;
}

// Element strides of a [rows, heads, head_dim] operand whose rows are read in
// 16-byte chunks.
int check_strides(const char* op, const char* name, int64_t row, int64_t head) {
    if (row % 8 || head % 8 || row < 0 || head < 0)
        return set_error(NANOVLLM_GEMM_EINVAL, "%s: strides of %s (%lld, %lld) must be non-negative multiples of 8", op,
                         name, (long long)row, (long long)head);
    // A tile of 64 rows is addressed with 32 bits.
    if (row >= int64_t(1) << 24)
        return set_error(NANOVLLM_GEMM_EUNSUPPORTED, "%s: the row stride of %s (%lld) must be below 2^24", op, name,
                         (long long)row);
    return NANOVLLM_GEMM_OK;
}

int check_pointers(const char* op, std::initializer_list<const void*> vector, std::initializer_list<const void*> other) {
    for (const void* p : vector)
        if (p == nullptr || !aligned16(p))
            return set_error(NANOVLLM_GEMM_EINVAL, "%s: operands must be non-null and 16-byte aligned", op);
    for (const void* p : other)
        if (p == nullptr) return set_error(NANOVLLM_GEMM_EINVAL, "%s: operands must be non-null", op);
    return NANOVLLM_GEMM_OK;
}

// `op` on this cache: sizes, strides and (where `touched`) pointers.
int check_cache(const char* op, const nanovllm_kv_cache* c, bool touched) {
    if (c == nullptr) return set_error(NANOVLLM_GEMM_EINVAL, "%s: cache must be non-null", op);
    if (c->bits != 16 && c->bits != 4)
        return set_error(NANOVLLM_GEMM_EUNSUPPORTED, "%s: a cache holds 16 or 4 bits, got %d", op, c->bits);
    if (!is_half(c->dtype))
        return set_error(NANOVLLM_GEMM_EUNSUPPORTED, "%s: dtype must be f16 or bf16, got %d", op, c->dtype);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return set_error(NANOVLLM_GEMM_EUNSUPPORTED, "%s: head_dim must be 64, 128 or 256, got %lld", op,
                         (long long)c->head_dim);
    if (c->num_blocks < 1 || c->block_size < 1 || c->kv_heads < 1 || c->kv_heads > 65536 || !fits32(c->num_blocks) ||
        !fits32(c->block_size) || !fits32(c->num_blocks * c->block_size))
        return set_error(NANOVLLM_GEMM_EINVAL,
                         "%s: a cache needs num_blocks, block_size and kv_heads of 1 or more and fewer than 2^31 slots",
                         op);
    if (c->bits == 4 && c->block_size % 16)
        return set_error(NANOVLLM_GEMM_EUNSUPPORTED, "%s: block_size (%lld) of a 4-bit cache must be a multiple of 16",
                         op, (long long)c->block_size);
    const int64_t rows = c->block_size * c->kv_heads;
    const int64_t page = c->bits == 16 ? rows * c->head_dim * 2 : rows * c->head_dim / 2;
    const int64_t scales = rows * (c->head_dim / kGroup) * 4;
    if (page > INT32_MAX) return set_error(NANOVLLM_GEMM_EUNSUPPORTED, "%s: a page must be smaller than 2 GiB", op);
    if (c->k_stride < page || c->v_stride < page || c->k_stride % 16 || c->v_stride % 16 ||
        (c->bits == 4 && (c->k_scales_stride < scales || c->v_scales_stride < scales || c->k_scales_stride % 16 ||
                          c->v_scales_stride % 16)))
        return set_error(NANOVLLM_GEMM_EINVAL,
                         "%s: page strides must be multiples of 16 bytes and not smaller than a page", op);
    // A kernel holds them in 32 bits, in units of 16 bytes.
    constexpr int64_t most = int64_t(16) * UINT32_MAX;
    if (c->k_stride > most || c->v_stride > most || (c->bits == 4 && (c->k_scales_stride > most || c->v_scales_stride > most)))
        return set_error(NANOVLLM_GEMM_EUNSUPPORTED, "%s: page strides must be smaller than 64 GiB", op);
    if (!touched) return NANOVLLM_GEMM_OK;
    const int rc = check_pointers(op, {c->k, c->v}, {});
    if (rc != NANOVLLM_GEMM_OK || c->bits == 16) return rc;
    return check_pointers(op, {c->k_scales, c->v_scales}, {});
}

Cache kernel_cache(const nanovllm_kv_cache& c) {
    return Cache{static_cast<char*>(c.k), static_cast<char*>(c.v), static_cast<char*>(c.k_scales),
                 static_cast<char*>(c.v_scales), c.k_stride, c.v_stride, c.k_scales_stride, c.v_scales_stride,
                 c.num_blocks * c.block_size, static_cast<int32_t>(c.num_blocks), static_cast<int32_t>(c.block_size),
                 static_cast<int32_t>(c.kv_heads)};
}

constexpr float kLog2e = 1.44269504088896340736f;

int check_scale(const char* op, float scale) {
    if (!(scale > 0.0f) || !std::isnormal(scale * kLog2e))
        return set_error(NANOVLLM_GEMM_EINVAL, "%s: scale must be positive, normal and finite", op);
    return NANOVLLM_GEMM_OK;
}

int check_prompt(const char* op, int64_t batch, int64_t q_rows, int64_t k_rows, int64_t heads, int64_t kv_heads,
                 int64_t head_dim, int dtype) {
    const int rc = check_dims(op, heads, kv_heads, head_dim, dtype);
    if (rc != NANOVLLM_GEMM_OK) return rc;
    if (batch < 0 || q_rows < 0 || k_rows < 0 || batch > INT32_MAX / 2 || q_rows > INT32_MAX / 2 || k_rows > INT32_MAX / 2)
        return set_error(NANOVLLM_GEMM_EINVAL, "%s: batch and rows must be non-negative and below 2^30", op);
    if (q_rows > 0 && attention_prompt_groups(batch, q_rows, k_rows, heads, head_dim) > kMostGroups)
        return set_error(NANOVLLM_GEMM_EUNSUPPORTED, "%s: too many sequences, rows and heads", op);
    return NANOVLLM_GEMM_OK;
}

int check_append(const char* op, const nanovllm_kv_cache* cache, int64_t tokens, int64_t heads, bool touched) {
    int rc = check_cache(op, cache, touched);
    if (rc == NANOVLLM_GEMM_OK) rc = check_dims(op, heads, cache->kv_heads, cache->head_dim, cache->dtype);
    if (rc != NANOVLLM_GEMM_OK) return rc;
    if (tokens < 0 || !fits32(tokens) || tokens * (heads + 2 * cache->kv_heads) > INT32_MAX)
        return set_error(NANOVLLM_GEMM_EINVAL, "%s: tokens must be non-negative, and tokens times heads below 2^31", op);
    if (rope_append_groups(tokens, heads, cache->kv_heads, static_cast<int>(cache->head_dim), cache->bits) > kMostGroups)
        return set_error(NANOVLLM_GEMM_EUNSUPPORTED, "%s: too many tokens and heads", op);
    return NANOVLLM_GEMM_OK;
}

int check_gather(const char* op, const nanovllm_kv_cache* cache, int64_t rows, bool touched) {
    const int rc = check_cache(op, cache, touched);
    if (rc != NANOVLLM_GEMM_OK) return rc;
    if (rows < 0 || !fits32(rows) || rows * 2 * cache->kv_heads > INT32_MAX)
        return set_error(NANOVLLM_GEMM_EINVAL, "%s: rows must be non-negative, and rows times heads below 2^31", op);
    if (kv_gather_groups(rows, cache->kv_heads, static_cast<int>(cache->head_dim), cache->bits) > kMostGroups)
        return set_error(NANOVLLM_GEMM_EUNSUPPORTED, "%s: too many rows and heads", op);
    return NANOVLLM_GEMM_OK;
}

int check_paged(const char* op, const nanovllm_kv_cache* cache, int64_t batch, int64_t heads, int64_t table_blocks,
                bool touched) {
    int rc = check_cache(op, cache, touched);
    if (rc == NANOVLLM_GEMM_OK) rc = check_dims(op, heads, cache->kv_heads, cache->head_dim, cache->dtype);
    if (rc != NANOVLLM_GEMM_OK) return rc;
    if (cache->block_size % 16)
        return set_error(NANOVLLM_GEMM_EUNSUPPORTED, "%s: block_size (%lld) must be a multiple of 16", op,
                         (long long)cache->block_size);
    // Tokens are counted in 32 bits, and the kernel looks two units of 128 and half a tile past a sequence's end.
    constexpr int64_t most = INT32_MAX - 1023;
    if (!fits32(batch) || !fits32(table_blocks) || table_blocks * cache->block_size > most)
        return set_error(NANOVLLM_GEMM_EINVAL,
                         "%s: batch and table must be non-negative, and a table hold at most 2^31 - 1024 tokens", op);
    // Units of 128 tokens are counted in 32 bits; the join has a workgroup or more for each pair.
    const int64_t blocks = cache->kv_heads * ((heads / cache->kv_heads + 15) / 16);
    if (batch * blocks > kMostGroups || !fits32(batch * blocks * (table_blocks * cache->block_size / 128 + 8)))
        return set_error(NANOVLLM_GEMM_EUNSUPPORTED, "%s: batch, heads and table are too large", op);
    return NANOVLLM_GEMM_OK;
}

}  // namespace
}  // namespace nvg

extern "C" {

int nanovllm_rope_append(const void* q, const void* k, const void* v, const int64_t* positions, const float* cos_sin,
                         const int32_t* slots, void* q_out, void* k_out, const nanovllm_kv_cache* cache,
                         int64_t tokens, int64_t heads, int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head,
                         int64_t v_row, int64_t v_head, int64_t positions_max, int64_t rotary, void* stream) {
    using namespace nvg;
    const char* op = "rope_append";
    clear_error();
    int rc = check_append(op, cache, tokens, heads, tokens > 0);
    if (rc == NANOVLLM_GEMM_OK) rc = check_strides(op, "q", q_row, q_head);
    if (rc == NANOVLLM_GEMM_OK) rc = check_strides(op, "k", k_row, k_head);
    if (rc == NANOVLLM_GEMM_OK) rc = check_strides(op, "v", v_row, v_head);
    if (rc != NANOVLLM_GEMM_OK) return rc;
    if (rotary < 16 || rotary % 16 || rotary > cache->head_dim)
        return set_error(NANOVLLM_GEMM_EINVAL, "rope_append: rotary (%lld) must be a multiple of 16 from 16 to head_dim",
                         (long long)rotary);
    if (positions_max < 1) return set_error(NANOVLLM_GEMM_EINVAL, "rope_append: positions_max must be positive");
    if (tokens == 0) return NANOVLLM_GEMM_OK;
    rc = check_pointers(op, {q, k, v, q_out, k_out}, {positions, cos_sin, slots});
    if (rc != NANOVLLM_GEMM_OK) return rc;
    const AppendArgs p{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k),
                       static_cast<const uint16_t*>(v), q_row, q_head, k_row, k_head, v_row, v_head, positions,
                       cos_sin, slots, static_cast<uint16_t*>(q_out), static_cast<uint16_t*>(k_out), positions_max,
                       static_cast<int32_t>(tokens), static_cast<int32_t>(heads), static_cast<int32_t>(rotary),
                       kernel_cache(*cache)};
    return launch_rope_append(p, static_cast<int>(cache->head_dim), cache->bits, cache->dtype,
                              static_cast<hipStream_t>(stream));
}

int nanovllm_kv_gather(const nanovllm_kv_cache* cache, const int32_t* slots, int64_t rows, void* k_out, void* v_out,
                       int dtype, void* stream) {
    using namespace nvg;
    const char* op = "kv_gather";
    clear_error();
    int rc = check_gather(op, cache, rows, rows > 0);
    if (rc != NANOVLLM_GEMM_OK) return rc;
    if (!is_half(dtype) || (cache->bits == 16 && dtype != cache->dtype))
        return set_error(NANOVLLM_GEMM_EUNSUPPORTED,
                         "kv_gather: rows are f16 or bf16, those of a 16-bit cache in its own dtype");
    if (rows == 0) return NANOVLLM_GEMM_OK;
    rc = check_pointers(op, {k_out, v_out}, {slots});
    if (rc != NANOVLLM_GEMM_OK) return rc;
    const GatherArgs p{slots, static_cast<uint16_t*>(k_out), static_cast<uint16_t*>(v_out),
                       static_cast<int32_t>(rows), kernel_cache(*cache)};
    return launch_kv_gather(p, static_cast<int>(cache->head_dim), cache->bits, dtype, static_cast<hipStream_t>(stream));
}

int nanovllm_rope_append_check(const nanovllm_kv_cache* cache, int64_t tokens, int64_t heads) {
    nvg::clear_error();
    return nvg::check_append("rope_append", cache, tokens, heads, false);
}

int nanovllm_kv_gather_check(const nanovllm_kv_cache* cache, int64_t rows) {
    nvg::clear_error();
    return nvg::check_gather("kv_gather", cache, rows, false);
}

int nanovllm_attention_prompt(const void* q, const void* k, const void* v, const int32_t* cu_q, const int32_t* cu_k,
                              void* out, int64_t batch, int64_t q_rows, int64_t k_rows, int64_t heads,
                              int64_t kv_heads, int64_t head_dim, int64_t q_row, int64_t q_head, int64_t k_row,
                              int64_t k_head, int64_t v_row, int64_t v_head, float scale, int causal, int dtype,
                              void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace nvg;
    const char* op = "attention_prompt";
    clear_error();
    int rc = check_prompt(op, batch, q_rows, k_rows, heads, kv_heads, head_dim, dtype);
    if (rc == NANOVLLM_GEMM_OK) rc = check_strides(op, "q", q_row, q_head);
    if (rc == NANOVLLM_GEMM_OK) rc = check_strides(op, "k", k_row, k_head);
    if (rc == NANOVLLM_GEMM_OK) rc = check_strides(op, "v", v_row, v_head);
    if (rc == NANOVLLM_GEMM_OK) rc = check_scale(op, scale);
    if (rc != NANOVLLM_GEMM_OK) return rc;
    if (q_rows == 0) return NANOVLLM_GEMM_OK;
    rc = k_rows > 0 ? check_pointers(op, {q, k, v, out}, {cu_q, cu_k}) : check_pointers(op, {q, out}, {cu_q, cu_k});
    if (rc != NANOVLLM_GEMM_OK) return rc;
    const int64_t need = attention_prompt_workspace(batch, q_rows, k_rows, heads, head_dim);
    if (need > 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < need))
        return set_error(NANOVLLM_GEMM_EINVAL, "attention_prompt: a 16-byte aligned workspace of %lld bytes is needed, got %lld",
                         (long long)need, (long long)workspace_bytes);
    const PromptArgs p{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k),
                       static_cast<const uint16_t*>(v), cu_q, cu_k, static_cast<uint16_t*>(out), q_row, q_head, k_row,
                       k_head, v_row, v_head, static_cast<int32_t>(batch), static_cast<int32_t>(q_rows),
                       static_cast<int32_t>(k_rows), static_cast<int32_t>(heads), static_cast<int32_t>(kv_heads),
                       causal != 0, scale * kLog2e};
    return launch_attention_prompt(p, workspace, static_cast<int>(head_dim), dtype, static_cast<hipStream_t>(stream));
}

int64_t nanovllm_attention_prompt_workspace_bytes(int64_t batch, int64_t q_rows, int64_t k_rows, int64_t heads,
                                                  int64_t kv_heads, int64_t head_dim, int dtype) {
    using namespace nvg;
    clear_error();
    const int rc = check_prompt("attention_prompt", batch, q_rows, k_rows, heads, kv_heads, head_dim, dtype);
    if (rc != NANOVLLM_GEMM_OK || q_rows == 0) return rc;
    return attention_prompt_workspace(batch, q_rows, k_rows, heads, head_dim);
}

int64_t nanovllm_attention_paged_workspace_bytes(const nanovllm_kv_cache* cache, int64_t batch, int64_t heads,
                                                 int64_t table_blocks) {
    using namespace nvg;
    clear_error();
    const int rc = check_paged("attention_paged", cache, batch, heads, table_blocks, false);
    if (rc != NANOVLLM_GEMM_OK) return rc;
    return attention_paged_workspace(batch, heads, cache->kv_heads, cache->head_dim, table_blocks * cache->block_size,
                                     cache->bits);
}

int nanovllm_attention_paged(const void* q, const nanovllm_kv_cache* cache, const int32_t* tables, const int32_t* lens,
                             void* out, int64_t batch, int64_t heads, int64_t table_blocks, int64_t table_stride,
                             int64_t q_row, int64_t q_head, float scale, int dtype, void* workspace,
                             int64_t workspace_bytes, void* stream) {
    using namespace nvg;
    const char* op = "attention_paged";
    clear_error();
    int rc = check_paged(op, cache, batch, heads, table_blocks, batch > 0);
    if (rc == NANOVLLM_GEMM_OK) rc = check_strides(op, "q", q_row, q_head);
    if (rc == NANOVLLM_GEMM_OK) rc = check_scale(op, scale);
    if (rc != NANOVLLM_GEMM_OK) return rc;
    if (!is_half(dtype) || (cache->bits == 16 && dtype != cache->dtype))
        return set_error(NANOVLLM_GEMM_EUNSUPPORTED,
                         "attention_paged: queries are f16 or bf16, in the dtype of a 16-bit cache");
    if (table_stride < table_blocks)
        return set_error(NANOVLLM_GEMM_EINVAL, "attention_paged: table_stride (%lld) must be >= table_blocks (%lld)",
                         (long long)table_stride, (long long)table_blocks);
    if (batch == 0) return NANOVLLM_GEMM_OK;
    rc = table_blocks > 0 ? check_pointers(op, {q, out}, {tables, lens}) : check_pointers(op, {q, out}, {lens});
    if (rc != NANOVLLM_GEMM_OK) return rc;
    const int64_t need = attention_paged_workspace(batch, heads, cache->kv_heads, cache->head_dim,
                                                   table_blocks * cache->block_size, cache->bits);
    if (need > 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < need))
        return set_error(NANOVLLM_GEMM_EINVAL, "attention_paged: a 16-byte aligned workspace of %lld bytes is needed, got %lld",
                         (long long)need, (long long)workspace_bytes);
    const PagedArgs p{static_cast<const uint16_t*>(q), tables, lens, static_cast<uint16_t*>(out),
                      static_cast<float*>(workspace), q_row, q_head, table_stride, static_cast<int32_t>(batch),
                      static_cast<int32_t>(heads), static_cast<int32_t>(table_blocks), scale * kLog2e,
                      kernel_cache(*cache)};
    return launch_attention_paged(p, static_cast<int>(cache->head_dim), cache->bits, dtype,
                                  static_cast<hipStream_t>(stream));
}

}  // extern "C"
