// Rotation and append to a paged cache, and reads of cached rows.
//
// Both only move bytes.  A row (token, head) is taken by head_dim / 8 lanes of
// 8 channels each, so a lane reads and writes 16-byte chunks and the 64
// channels of a 4-bit group are 8 neighbouring lanes.
#include <type_traits>

#include "attention_common.hpp"

namespace nvg {
namespace {

constexpr int kThreads = 256;

struct F8 { float x[8]; };

template <int DT>
__device__ __forceinline__ F8 widen8(u32x4_t v) {
    F8 f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f.x[2 * i] = half_to_f32<DT>(uint16_t(v[i]));
        f.x[2 * i + 1] = half_to_f32<DT>(uint16_t(v[i] >> 16));
    }
    return f;
}

template <int DT>
__device__ __forceinline__ u32x4_t narrow8(const F8& f) {
    return u32x4_t{pack2<DT>(f.x[0], f.x[1]), pack2<DT>(f.x[2], f.x[3]), pack2<DT>(f.x[4], f.x[5]),
                   pack2<DT>(f.x[6], f.x[7])};
}

// Chunk c (8 channels) of a row, rotated.  Products and the sum are rounded
// one by one (no fused multiply-add), as the formula reads.
template <int DT>
__device__ __forceinline__ u32x4_t rotate8(const uint16_t* row, int c, const float* turn, int rotary, bool known) {
#pragma clang fp contract(off)
    const int half = rotary / 16;   // chunks of a half
    const u32x4_t raw = load16(row + 8 * c);
    if (c >= 2 * half) return raw;
    const bool second = c >= half;
    const int at = second ? c - half : c;
    const F8 x = widen8<DT>(raw), p = widen8<DT>(load16(row + 8 * (second ? at : at + half)));
    F8 y;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float cs = known ? turn[8 * at + i] : __builtin_nanf("");
        const float sn = known ? turn[rotary / 2 + 8 * at + i] : __builtin_nanf("");
        const float a = x.x[i] * cs, b = p.x[i] * sn;
        y.x[i] = second ? a + b : a - b;
    }
    return narrow8<DT>(y);
}

// Codes of a lane's 8 channels, with the scale and minimum of its group of 64
// (8 lanes): the arithmetic of nanovllm_rope_append, fp32, IEEE divisions.
struct Coded { uint32_t code[8]; uint32_t scale; };   // scale: float16 scale, minimum << 16

template <int DT>
__device__ __forceinline__ Coded quantise8(u32x4_t raw) {
#pragma clang fp contract(off)
    F8 f = widen8<DT>(raw);
    float lo = __builtin_inff(), hi = -__builtin_inff();
    int nan = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        nan |= f.x[i] != f.x[i];
        f.x[i] = fminf(fmaxf(f.x[i], -65504.0f), 65504.0f);
        lo = fminf(lo, f.x[i]);
        hi = fmaxf(hi, f.x[i]);
    }
#pragma unroll
    for (int off = 1; off < 8; off <<= 1) {
        lo = fminf(lo, __shfl_xor(lo, off));
        hi = fmaxf(hi, __shfl_xor(hi, off));
        nan |= __shfl_xor(nan, off);
    }
    if (nan) lo = hi = __builtin_nanf("");
    const _Float16 s16 = static_cast<_Float16>((hi - lo) / 15.0f), m16 = static_cast<_Float16>(lo);
    const float s = static_cast<float>(s16), m = static_cast<float>(m16);
    Coded r;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float q = fminf(fmaxf(rintf((f.x[i] - m) / s), 0.0f), 15.0f);
        r.code[i] = s > 0.0f ? static_cast<uint32_t>(q) : 0u;
    }
    r.scale = uint32_t(__builtin_bit_cast(uint16_t, s16)) | uint32_t(__builtin_bit_cast(uint16_t, m16)) << 16;
    return r;
}

// Where four neighbouring rows of a call are the four tokens of one aligned
// word of a 4-bit cache, the first takes all four, so that values are stored
// and read as whole words; any other row is taken alone, a byte at a time.
// Returns the tokens this row takes: 4, 1, or 0 where another row takes it.
__device__ __forceinline__ int row_share(const int32_t* slots, int row, int rows, int slot) {
    const int at = slot & 3, first = row - at;
    if (first < 0 || first + 3 >= rows) return 1;
    const int base = slot - at;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (slots[first + i] != base + i) return 1;
    return at == 0 ? 4 : 0;
}

template <int DT, int D, int BITS>
__global__ __launch_bounds__(kThreads) void rope_append_kernel(const AppendArgs p) {
    constexpr int CH = D / 8, GROUPS = D / kGroup;
    const int c = threadIdx.x % CH, kvh = p.cache.kv_heads;
    const int per_token = p.heads + 2 * kvh;
    const int64_t row = int64_t(blockIdx.x) * (kThreads / CH) + threadIdx.x / CH;
    if (row >= int64_t(p.tokens) * per_token) return;
    const int t = int(uint32_t(row) / uint32_t(per_token));
    int h = int(row - int64_t(t) * per_token);
    const int64_t pos = p.positions[t];
    const bool known = pos >= 0 && pos < p.positions_max;
    const float* turn = p.cos_sin + (known ? pos : 0) * p.rotary;
    if (h < p.heads) {
        const u32x4_t y = rotate8<DT>(p.q + t * p.q_row + h * p.q_head, c, turn, p.rotary, known);
        *reinterpret_cast<u32x4_t*>(p.q_out + (int64_t(t) * p.heads + h) * D + 8 * c) = y;
        return;
    }
    h -= p.heads;
    const bool value = h >= kvh;
    if (value) h -= kvh;
    const int slot = p.slots[t];
    const bool kept = slot >= 0 && slot < p.cache.slots;
    if constexpr (BITS == 16) {
        u32x4_t y;
        if (value) {
            y = load16(p.v + t * p.v_row + h * p.v_head + 8 * c);
        } else {
            y = rotate8<DT>(p.k + t * p.k_row + h * p.k_head, c, turn, p.rotary, known);
            *reinterpret_cast<u32x4_t*>(p.k_out + (int64_t(t) * kvh + h) * D + 8 * c) = y;
        }
        if (!kept) return;
        const uint32_t page = uint32_t(slot) / uint32_t(p.cache.block_size), at = slot - page * p.cache.block_size;
        char* dst = value ? p.cache.v + page * p.cache.v_stride : p.cache.k + page * p.cache.k_stride;
        *reinterpret_cast<u32x4_t*>(dst + ((int64_t(at) * kvh + h) * D + 8 * c) * 2) = y;
    } else {
        const uint32_t page = uint32_t(kept ? slot : 0) / uint32_t(p.cache.block_size);
        const uint32_t at = (kept ? slot : 0) - page * p.cache.block_size;
        const int g = c / 8;
        if (!value) {
            const u32x4_t y = rotate8<DT>(p.k + t * p.k_row + h * p.k_head, c, turn, p.rotary, known);
            *reinterpret_cast<u32x4_t*>(p.k_out + (int64_t(t) * kvh + h) * D + 8 * c) = y;
            const Coded r = quantise8<DT>(y);
            if (!kept) return;
            uint32_t word = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) word |= r.code[j] << (4 * (j / 2) + 16 * (j % 2));
            const int64_t line = int64_t(h) * p.cache.block_size + at;
            *reinterpret_cast<uint32_t*>(p.cache.k + page * p.cache.k_stride + line * (D / 2) +
                                         4 * word_place<GROUPS, 8>(g, c % 8)) = word;
            if (c % 8 == 0)
                *reinterpret_cast<uint32_t*>(p.cache.k_scales + page * p.cache.ks_stride +
                                             4 * (line * GROUPS + g)) = r.scale;
            return;
        }
        if (!kept) return;
        const int share = row_share(p.slots, t, p.tokens, slot);
        if (share == 0) return;
        char* words = p.cache.v + page * p.cache.v_stride +
                      (int64_t(h) * p.cache.block_size + (at & ~3u)) * (D / 2);
        char* scales = p.cache.v_scales + page * p.cache.vs_stride +
                       4 * ((int64_t(h) * GROUPS + g) * p.cache.block_size + at);
        const uint16_t* src = p.v + t * p.v_row + h * p.v_head + 8 * c;
        if (share == 4) {
            u32x4_t w = {0, 0, 0, 0}, sc;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const Coded r = quantise8<DT>(load16(src + i * p.v_row));
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] |= (r.code[2 * e] | r.code[2 * e + 1] << 4) << (8 * i);
                sc[i] = r.scale;
            }
#pragma unroll
            for (int e = 0; e < 4; e += 2)
                *reinterpret_cast<u32x2_t*>(words + 4 * word_place<GROUPS, 32>(g, 4 * (c % 8) + e)) =
                    u32x2_t{w[e], w[e + 1]};
            if (c % 8 == 0) *reinterpret_cast<u32x4_t*>(scales) = sc;
        } else {
            const Coded r = quantise8<DT>(load16(src));
#pragma unroll
            for (int e = 0; e < 4; ++e)
                words[4 * word_place<GROUPS, 32>(g, 4 * (c % 8) + e) + (at & 3)] =
                    static_cast<char>(r.code[2 * e] | r.code[2 * e + 1] << 4);
            if (c % 8 == 0) *reinterpret_cast<uint32_t*>(scales) = r.scale;
        }
    }
}

// Eight elements of codes `code(j)` with a scale word.
template <int DT, typename F>
__device__ __forceinline__ u32x4_t dequantise8(uint32_t scale, F&& code) {
    const float s = f16_to_f32(uint16_t(scale)), m = f16_to_f32(uint16_t(scale >> 16));
    F8 f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f.x[j] = __builtin_fmaf(static_cast<float>(code(j)), s, m);
    return narrow8<DT>(f);
}

template <int DT, int D, int BITS>
__global__ __launch_bounds__(kThreads) void kv_gather_kernel(const GatherArgs p) {
    constexpr int CH = D / 8, GROUPS = D / kGroup;
    const int c = threadIdx.x % CH, kvh = p.cache.kv_heads;
    const int64_t row = int64_t(blockIdx.x) * (kThreads / CH) + threadIdx.x / CH;
    if (row >= int64_t(p.rows) * 2 * kvh) return;
    const int n = int(uint32_t(row) / uint32_t(2 * kvh));
    int h = int(row - int64_t(n) * 2 * kvh);
    const bool value = h >= kvh;
    if (value) h -= kvh;
    uint16_t* out = (value ? p.v_out : p.k_out) + (int64_t(n) * kvh + h) * D + 8 * c;
    const int slot = p.slots[n];
    if (slot < 0 || slot >= p.cache.slots) {
        *reinterpret_cast<u32x4_t*>(out) = u32x4_t{0, 0, 0, 0};
        return;
    }
    const uint32_t page = uint32_t(slot) / uint32_t(p.cache.block_size), at = slot - page * p.cache.block_size;
    if constexpr (BITS == 16) {
        const char* src = value ? p.cache.v + page * p.cache.v_stride : p.cache.k + page * p.cache.k_stride;
        *reinterpret_cast<u32x4_t*>(out) = load16(src + ((int64_t(at) * kvh + h) * D + 8 * c) * 2);
    } else {
        const int g = c / 8;
        if (!value) {
            const int64_t line = int64_t(h) * p.cache.block_size + at;
            const uint32_t word = *reinterpret_cast<const uint32_t*>(
                p.cache.k + page * p.cache.k_stride + line * (D / 2) + 4 * word_place<GROUPS, 8>(g, c % 8));
            const uint32_t scale = *reinterpret_cast<const uint32_t*>(
                p.cache.k_scales + page * p.cache.ks_stride + 4 * (line * GROUPS + g));
            *reinterpret_cast<u32x4_t*>(out) =
                dequantise8<DT>(scale, [&](int j) { return (word >> (4 * (j / 2) + 16 * (j % 2))) & 15u; });
            return;
        }
        const int share = row_share(p.slots, n, p.rows, slot);
        if (share == 0) return;
        const char* words = p.cache.v + page * p.cache.v_stride +
                            (int64_t(h) * p.cache.block_size + (at & ~3u)) * (D / 2);
        const char* scales = p.cache.v_scales + page * p.cache.vs_stride +
                             4 * ((int64_t(h) * GROUPS + g) * p.cache.block_size + at);
        u32x2_t w[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
            w[e] = *reinterpret_cast<const u32x2_t*>(words + 4 * word_place<GROUPS, 32>(g, 4 * (c % 8) + 2 * e));
        auto token = [&](uint32_t scale, int i) {
            return dequantise8<DT>(scale, [&](int j) { return (w[j / 4][(j / 2) % 2] >> (8 * i + 4 * (j % 2))) & 15u; });
        };
        if (share == 4) {
            const u32x4_t sc = load16(scales);
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<u32x4_t*>(out + int64_t(i) * kvh * D) = token(sc[i], i);
        } else {
            *reinterpret_cast<u32x4_t*>(out) = token(*reinterpret_cast<const uint32_t*>(scales), at & 3);
        }
    }
}

template <typename F>
int pick(int dtype, int head_dim, int bits, F&& f) {
    auto with_bits = [&](auto dt, auto d) {
        return bits == 4 ? f(dt, d, std::integral_constant<int, 4>{}) : f(dt, d, std::integral_constant<int, 16>{});
    };
    auto with_dim = [&](auto dt) {
        return head_dim == 64    ? with_bits(dt, std::integral_constant<int, 64>{})
               : head_dim == 128 ? with_bits(dt, std::integral_constant<int, 128>{})
                                 : with_bits(dt, std::integral_constant<int, 256>{});
    };
    return dtype == NANOVLLM_GEMM_BF16 ? with_dim(std::integral_constant<int, NANOVLLM_GEMM_BF16>{})
                                       : with_dim(std::integral_constant<int, NANOVLLM_GEMM_F16>{});
}

}  // namespace

int launch_rope_append(const AppendArgs& p, int head_dim, int bits, int dtype, hipStream_t s) {
    const int64_t rows = int64_t(p.tokens) * (p.heads + 2 * p.cache.kv_heads), per = kThreads / (head_dim / 8);
    const dim3 grid(static_cast<uint32_t>((rows + per - 1) / per));
    return pick(dtype, head_dim, bits, [&](auto dt, auto d, auto b) {
        hipLaunchKernelGGL((rope_append_kernel<dt.value, d.value, b.value>), grid, dim3(kThreads), 0, s, p);
        return check_launch("rope_append");
    });
}

int launch_kv_gather(const GatherArgs& p, int head_dim, int bits, int dtype, hipStream_t s) {
    const int64_t rows = int64_t(p.rows) * 2 * p.cache.kv_heads, per = kThreads / (head_dim / 8);
    const dim3 grid(static_cast<uint32_t>((rows + per - 1) / per));
    return pick(dtype, head_dim, bits, [&](auto dt, auto d, auto b) {
        hipLaunchKernelGGL((kv_gather_kernel<dt.value, d.value, b.value>), grid, dim3(kThreads), 0, s, p);
        return check_launch("kv_gather");
    });
}

}  // namespace nvg
