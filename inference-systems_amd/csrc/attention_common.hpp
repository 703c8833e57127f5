// What the attention operators share: the paged cache as kernels see it, the
// places of 4-bit codes, cross-lane moves and the launchers capi_attention.cpp
// dispatches to.
#pragma once

#include "../../include/nanovllm_attention.h"
#include "gemm_common.hpp"

namespace nvg {

// A paged cache (see nanovllm_kv_cache); strides between pages in bytes.
struct Cache {
    char *k, *v, *k_scales, *v_scales;
    int64_t k_stride, v_stride, ks_stride, vs_stride;
    int64_t slots;        // num_blocks * block_size
    int32_t num_blocks, block_size, kv_heads;
};

// A launch has fewer than 2^32 threads, here of 256 a workgroup.
constexpr int64_t kMostGroups = (int64_t(1) << 24) - 1;
constexpr int kGroup = 64;   // channels that share a 4-bit scale and minimum

struct AppendArgs {
    const uint16_t *q, *k, *v;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;   // elements
    const int64_t* positions;
    const float* cos_sin;
    const int32_t* slots;
    uint16_t *q_out, *k_out;
    int64_t positions_max;
    int32_t tokens, heads, rotary;
    Cache cache;
};

struct GatherArgs {
    const int32_t* slots;
    uint16_t *k_out, *v_out;
    int32_t rows;
    Cache cache;
};

struct PromptArgs {
    const uint16_t *q, *k, *v;
    const int32_t *cu_q, *cu_k;
    uint16_t* out;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;   // elements
    int32_t batch, q_rows, k_rows, heads, kv_heads, causal;
    float c;   // scale * log2(e): the softmax runs on base 2
};

struct PagedArgs {
    const uint16_t* q;
    const int32_t *tables, *lens;
    uint16_t* out;
    float* partial;
    int64_t q_row, q_head, table_stride;
    int32_t batch, heads, table_blocks;
    float c;
    Cache cache;
};

// Word u of group g of a 4-bit row with `groups` groups: its place among the
// row's words (those of two neighbouring groups take turns two by two).
template <int GROUPS, int PER_GROUP>
__device__ __forceinline__ int word_place(int g, int u) {
    if constexpr (GROUPS == 1) return u;
    else return (g / 2) * (2 * PER_GROUP) + (u / 2) * 4 + (g % 2) * 2 + u % 2;
}

// Largest value over lanes l, l ^ 16, l ^ 32, l ^ 48 (the four lanes that hold
// one column of a 16 x 16 product) and over l, l ^ 32 (two, of a 32 x 32 one).
__device__ __forceinline__ float max_across32(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return fmaxf(__builtin_bit_cast(float, uint32_t(r[0])), __builtin_bit_cast(float, uint32_t(r[1])));
}
__device__ __forceinline__ float max_across16(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    return fmaxf(__builtin_bit_cast(float, uint32_t(r[0])), __builtin_bit_cast(float, uint32_t(r[1])));
}
__device__ __forceinline__ float sum_across32(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return __builtin_bit_cast(float, uint32_t(r[0])) + __builtin_bit_cast(float, uint32_t(r[1]));
}
__device__ __forceinline__ float sum_across16(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    return __builtin_bit_cast(float, uint32_t(r[0])) + __builtin_bit_cast(float, uint32_t(r[1]));
}

// Sum over lanes 0 .. l of a wave.
__device__ __forceinline__ int prefix_sum(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);    // 1, 2, 4, 8 lanes up in rows of 16
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);    // lane 15 of a row into the next
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);    // lane 31 into the upper half
    return x;
}

// A weight is 2^(c s - c m) of a score s and the maximum m, one multiply-add where
// the rounding of c m, up to c m 2^-24, does not matter.  Behind this it would (at
// 2^29 float16 weights overflow): there s - m, which is exact near the maximum, is
// taken first.  The question costs a tile a few instructions: 512 tokens behind 8188
// cached 87.9 -> 88.6 us, 16384 tokens 1148 -> 1150, over pages nothing.
constexpr float kFarScore = 1024.0f;

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// The index of a lane-uniform value in a scalar register.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// A word at a lane-uniform address that nothing writes during the kernel, by a
// scalar load: it does not wait for the vector loads in flight.
__device__ __forceinline__ int scalar_load(const int32_t* p) {
    typedef const __attribute__((address_space(4))) int32_t* constant_ptr;
    return *(constant_ptr)(p);
}

// dma16 (gemm_common.hpp) from a lane-uniform address and a 32-bit offset per lane.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16_at(const void* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 :: "v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
#pragma clang diagnostic pop

template <int N, typename F, int I = 0>
__device__ __forceinline__ void static_for(F&& f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        static_for<N, F, I + 1>(static_cast<F&&>(f));
    }
}

// Workgroups of a launch: kMostGroups at most, which the C ABI checks.
int64_t rope_append_groups(int64_t tokens, int64_t heads, int64_t kv_heads, int head_dim, int bits);
int64_t kv_gather_groups(int64_t rows, int64_t kv_heads, int head_dim, int bits);
int64_t attention_prompt_groups(int64_t batch, int64_t q_rows, int64_t k_rows, int64_t heads, int64_t head_dim);

int launch_rope_append(const AppendArgs& p, int head_dim, int bits, int dtype, hipStream_t s);
int launch_kv_gather(const GatherArgs& p, int head_dim, int bits, int dtype, hipStream_t s);
int launch_attention_prompt(const PromptArgs& p, void* workspace, int head_dim, int dtype, hipStream_t s);
int64_t attention_prompt_workspace(int64_t batch, int64_t q_rows, int64_t k_rows, int64_t heads, int64_t head_dim);
int launch_attention_paged(const PagedArgs& p, int head_dim, int bits, int dtype, hipStream_t s);
int64_t attention_paged_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                  int64_t table_tokens, int bits);

void clear_error();

}  // namespace nvg
