// Rotation and append to a paged cache, and reads of cached rows.
//
// Both only move bytes and are bound by HBM where a call is long, by the chain
// of loads (position or slot, then what it points to) where it is short.  A row
// (token, head) is taken by head_dim / 8 lanes of 8 channels each, so a lane
// reads and writes 16-byte chunks and the 64 channels of a 4-bit group are 8
// neighbouring lanes.  Measured on MI355X (a large copy: 5.1 TB/s): 8000 tokens
// of 16 + 2 x 4 heads of 128 into a 4-bit cache 23-24 us for 101 MB, 4.3 TB/s (a row
// a team, with its own cosines and divisions: 49 us); 20000 tokens of 8 + 2 x 2
// heads of 256, 16 bits, 45 us for 272 MB, partly through the last-level cache; one
// token 2.6 us.  Rows of 4 + 4 heads of 128 gathered: 20000 from 16-bit pages 13 us,
// partly from the last-level cache, 8000 and 20000 from 4-bit ones 6.6 and 13.2 us
// (values by a team a row, three of four of them idle: 9.2 and 19.1 us).
#include <type_traits>

#include "attention_common.hpp"

namespace nvg {
namespace {

constexpr int kThreads = 256;
constexpr int kFull = 1024;     // workgroups that fill the chip's 256 CUs

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

// cos and sin of a lane's chunk (8 channels) of a token: of the first half of
// the channels that turn, y = x cos - partner sin, of the second
// y = x cos + partner sin; the sign is kept with the sine.
struct Turn { F8 cs, sn; };

__device__ __forceinline__ Turn turn_of(const AppendArgs& p, int64_t pos, int c) {
    const int half = p.rotary / 16;   // chunks of a half
    Turn t{};
    if (c >= 2 * half) return t;
    const bool known = pos >= 0 && pos < p.positions_max, second = c >= half;
    const float* row = p.cos_sin + (known ? pos : 0) * p.rotary + 8 * (second ? c - half : c);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float cs = row[i], sn = row[p.rotary / 2 + i];
        t.cs.x[i] = known ? cs : __builtin_nanf("");
        t.sn.x[i] = !known ? __builtin_nanf("") : second ? sn : -sn;
    }
    return t;
}

// A chunk and its partner, rotated.  Products and the sum are rounded one by
// one (no fused multiply-add), as the formula reads.
template <int DT>
__device__ __forceinline__ u32x4_t rotate8(u32x4_t raw, u32x4_t partner, const Turn& t) {
#pragma clang fp contract(off)
    const F8 x = widen8<DT>(raw), p = widen8<DT>(partner);
    F8 y;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = x.x[i] * t.cs.x[i], b = p.x[i] * t.sn.x[i];
        y.x[i] = a + b;
    }
    return narrow8<DT>(y);
}

// Codes of a lane's 8 channels, with the scale and minimum of its group of 64
// (8 lanes): the arithmetic of nanovllm_rope_append, fp32, quotients correctly
// rounded.  With y = 1 / s correctly rounded, one step q + y (a - q s) on a
// quotient within one unit of the last place gives the correctly rounded one
// (Markstein); a y may be two units off, so the step is taken twice: 5
// operations an element for the 10 or so of a division.  s is a positive
// float16, so y is finite and a - q s exact; quotients far below 1, where it
// may not be, are code 0 either way.
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
    _Float16 s16 = static_cast<_Float16>((hi - lo) / 15.0f);
    const _Float16 m16 = static_cast<_Float16>(lo);
    const float m = static_cast<float>(m16);
    // A scale rounded up may carry code 15 past float16's range (15 s is exact, so the sum is rounded once).
    if (15.0f * static_cast<float>(s16) + m > 65504.0f)
        s16 = __builtin_bit_cast(_Float16, static_cast<uint16_t>(__builtin_bit_cast(uint16_t, s16) - 1));
    const float s = static_cast<float>(s16);
    const float y = 1.0f / s;
    Coded r;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = f.x[i] - m;
        float q = a * y;
        q = __builtin_fmaf(__builtin_fmaf(-q, s, a), y, q);
        q = __builtin_fmaf(__builtin_fmaf(-q, s, a), y, q);
        q = fminf(fmaxf(rintf(q), 0.0f), 15.0f);
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

// The work of a call: head_dim / 8 lanes (a team) take a token, a workgroup as
// many neighbouring tokens as it has teams, and `EACH` heads of them, which
// share the token's cosines and sines.  Values of a 4-bit cache have workgroups
// of their own, which come first.
struct AppendSplit {
    AppendArgs a;
    int32_t parts;          // workgroups that share a run of tokens
    int32_t v_rows;         // 4 bits: rows of a workgroup of values, 64 at most
    int32_t v_groups;       // 4 bits: workgroups of values
};

// Rows first .. first + n - 1 (64 at most) that have a share of the values: how
// many, and in lane i of every wave the i-th of them and its share << 8.  Lane l
// looks at row l.  So no team waits for rows that another takes with its own.
__device__ __forceinline__ int list_shares(const int32_t* slots, int first, int n, int rows, int most, int& listed) {
    const int lane = threadIdx.x & 63;
    int share = 0;
    if (lane < n) {
        const int slot = slots[first + lane];
        if (slot >= 0 && slot < most) share = row_share(slots, first + lane, rows, slot);
    }
    const uint64_t taken = __ballot(share != 0);
    const int count = __popcll(taken), rank = __popcll(taken & ((uint64_t(1) << lane) - 1));
    listed = __builtin_amdgcn_ds_permute(4 * (share != 0 ? rank : count + lane - rank), lane | share << 8);
    return count;
}

// 4-bit values of up to 64 rows of one head.
template <int DT, int D>
__device__ __forceinline__ void append_values(const AppendArgs& p, int first, int rows, int h) {
    constexpr int CH = D / 8, GROUPS = D / kGroup, TEAMS = kThreads / CH;
    const int c = threadIdx.x % CH, g = c / 8;
    int listed;
    const int count = list_shares(p.slots, first, min(rows, p.tokens - first), p.tokens, p.cache.slots, listed);
    for (int i = threadIdx.x / CH; i - int(threadIdx.x / CH) < count; i += TEAMS) {      // all lanes stay for the shuffles
        const int what = __shfl(listed, min(i, count - 1));
        const int t = first + (what & 255), four = (what >> 8) == 4;
        const int slot = p.slots[t];
        const uint32_t page = uint32_t(slot) / uint32_t(p.cache.block_size), at = slot - page * p.cache.block_size;
        char* words = p.cache.v + page * p.cache.v_stride +
                      (int64_t(h) * p.cache.block_size + (at & ~3u)) * (D / 2);
        char* scales = p.cache.v_scales + page * p.cache.vs_stride +
                       4 * ((int64_t(h) * GROUPS + g) * p.cache.block_size + at);
        const uint16_t* src = p.v + t * p.v_row + h * p.v_head + 8 * c;
        if (i >= count) continue;
        if (four) {
            u32x4_t raw[4], w = {0, 0, 0, 0}, sc;
#pragma unroll
            for (int j = 0; j < 4; ++j) raw[j] = load16(src + j * p.v_row);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const Coded r = quantise8<DT>(raw[j]);
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] |= (r.code[2 * e] | r.code[2 * e + 1] << 4) << (8 * j);
                sc[j] = r.scale;
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

template <int DT, int D, int BITS, int EACH>
__global__ __launch_bounds__(kThreads) void rope_append_kernel(const AppendSplit sp) {
    constexpr int CH = D / 8, GROUPS = D / kGroup, TEAMS = kThreads / CH;
    const AppendArgs& p = sp.a;
    const int kvh = p.cache.kv_heads;
    int block = blockIdx.x;
    if constexpr (BITS == 4) {
        if (block < sp.v_groups) {
            const int run = block / kvh;
            append_values<DT, D>(p, run * sp.v_rows, sp.v_rows, block - run * kvh);
            return;
        }
        block -= sp.v_groups;
    }
    const int c = threadIdx.x % CH, run = block / sp.parts, h0 = (block - run * sp.parts) * EACH;
    const int heads = p.heads + (BITS == 4 ? 1 : 2) * kvh, t = run * TEAMS + threadIdx.x / CH;
    if (t >= p.tokens) return;
    const int64_t pos = p.positions[t];
    const int slot = p.slots[t];
    const bool kept = slot >= 0 && slot < p.cache.slots;
    const uint32_t page = uint32_t(kept ? slot : 0) / uint32_t(p.cache.block_size);
    const uint32_t at = (kept ? slot : 0) - page * p.cache.block_size;
    const int half = p.rotary / 16;
    const bool turns = c < 2 * half;
    const int partner = !turns ? c : c < half ? c + half : c - half;
    u32x4_t x[EACH], y[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int h = min(h0 + i, heads - 1);
        const uint16_t* src = h < p.heads         ? p.q + t * p.q_row + h * p.q_head
                              : h < p.heads + kvh ? p.k + t * p.k_row + (h - p.heads) * p.k_head
                                                  : p.v + t * p.v_row + (h - p.heads - kvh) * p.v_head;
        x[i] = load16(src + 8 * c);
        y[i] = load16(src + 8 * partner);
    }
    const Turn turn = turn_of(p, pos, c);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        int h = h0 + i;
        if (h >= heads) return;
        const u32x4_t turned = turns ? rotate8<DT>(x[i], y[i], turn) : x[i];
        if (h < p.heads) {
            *reinterpret_cast<u32x4_t*>(p.q_out + (int64_t(t) * p.heads + h) * D + 8 * c) = turned;
            continue;
        }
        h -= p.heads;
        if (BITS == 4 || h < kvh)
            *reinterpret_cast<u32x4_t*>(p.k_out + (int64_t(t) * kvh + h) * D + 8 * c) = turned;
        if constexpr (BITS == 16) {
            const bool value = h >= kvh;
            if (value) h -= kvh;
            char* dst = value ? p.cache.v + page * p.cache.v_stride : p.cache.k + page * p.cache.k_stride;
            if (kept) *reinterpret_cast<u32x4_t*>(dst + ((int64_t(at) * kvh + h) * D + 8 * c) * 2) = value ? x[i] : turned;
        } else {
            const int g = c / 8;
            const Coded r = quantise8<DT>(turned);
            if (!kept) continue;
            uint32_t word = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) word |= r.code[j] << (4 * (j / 2) + 16 * (j % 2));
            const int64_t line = int64_t(h) * p.cache.block_size + at;
            *reinterpret_cast<uint32_t*>(p.cache.k + page * p.cache.k_stride + line * (D / 2) +
                                         4 * word_place<GROUPS, 8>(g, c % 8)) = word;
            if (c % 8 == 0)
                *reinterpret_cast<uint32_t*>(p.cache.k_scales + page * p.cache.ks_stride +
                                             4 * (line * GROUPS + g)) = r.scale;
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

// 4-bit values of up to 64 rows of one head, and zeros for those outside the cache.
template <int DT, int D>
__device__ __forceinline__ void gather_values(const GatherArgs& p, int first, int rows, int h) {
    constexpr int CH = D / 8, GROUPS = D / kGroup, TEAMS = kThreads / CH;
    const int c = threadIdx.x % CH, g = c / 8, team = threadIdx.x / CH, kvh = p.cache.kv_heads;
    rows = min(rows, p.rows - first);
    auto out = [&](int n) { return reinterpret_cast<u32x4_t*>(p.v_out + (int64_t(n) * kvh + h) * D + 8 * c); };
    int listed;
    const int count = list_shares(p.slots, first, rows, p.rows, p.cache.slots, listed);
    for (int i = team; i - team < count; i += TEAMS) {      // all lanes stay for the shuffle
        const int what = __shfl(listed, min(i, count - 1));
        if (i >= count) continue;
        const int n = first + (what & 255), slot = p.slots[n];
        const uint32_t page = uint32_t(slot) / uint32_t(p.cache.block_size), at = slot - page * p.cache.block_size;
        const char* words = p.cache.v + page * p.cache.v_stride +
                            (int64_t(h) * p.cache.block_size + (at & ~3u)) * (D / 2);
        const char* scales = p.cache.v_scales + page * p.cache.vs_stride +
                             4 * ((int64_t(h) * GROUPS + g) * p.cache.block_size + at);
        u32x2_t w[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
            w[e] = *reinterpret_cast<const u32x2_t*>(words + 4 * word_place<GROUPS, 32>(g, 4 * (c % 8) + 2 * e));
        auto token = [&](uint32_t scale, int j) {
            return dequantise8<DT>(scale, [&](int x) { return (w[x / 4][(x / 2) % 2] >> (8 * j + 4 * (x % 2))) & 15u; });
        };
        if ((what >> 8) == 4) {
            const u32x4_t sc = load16(scales);
#pragma unroll
            for (int j = 0; j < 4; ++j) *out(n + j) = token(sc[j], j);
        } else {
            *out(n) = token(*reinterpret_cast<const uint32_t*>(scales), at & 3);
        }
    }
    for (int i = team; i < rows; i += TEAMS) {
        const int slot = p.slots[first + i];
        if (slot < 0 || slot >= p.cache.slots) *out(first + i) = u32x4_t{0, 0, 0, 0};
    }
}

// Keys of a 4-bit cache, keys and values of a 16-bit one: a team a row.
template <int DT, int D, int BITS>
__global__ __launch_bounds__(kThreads) void kv_gather_kernel(const GatherArgs p, int v_rows, int v_groups) {
    constexpr int CH = D / 8, GROUPS = D / kGroup;
    const int c = threadIdx.x % CH, kvh = p.cache.kv_heads;
    int block = blockIdx.x;
    if constexpr (BITS == 4) {
        if (block < v_groups) {
            const int run = block / kvh;
            gather_values<DT, D>(p, run * v_rows, v_rows, block - run * kvh);
            return;
        }
        block -= v_groups;
    }
    const int heads = BITS == 4 ? kvh : 2 * kvh;
    const int64_t row = int64_t(block) * (kThreads / CH) + threadIdx.x / CH;
    if (row >= int64_t(p.rows) * heads) return;
    const int n = int(uint32_t(row) / uint32_t(heads));
    int h = int(row - int64_t(n) * heads);
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
        const int64_t line = int64_t(h) * p.cache.block_size + at;
        const uint32_t word = *reinterpret_cast<const uint32_t*>(
            p.cache.k + page * p.cache.k_stride + line * (D / 2) + 4 * word_place<GROUPS, 8>(g, c % 8));
        const uint32_t scale = *reinterpret_cast<const uint32_t*>(
            p.cache.k_scales + page * p.cache.ks_stride + 4 * (line * GROUPS + g));
        *reinterpret_cast<u32x4_t*>(out) =
            dequantise8<DT>(scale, [&](int j) { return (word >> (4 * (j / 2) + 16 * (j % 2))) & 15u; });
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

// 4 bits: rows of a workgroup of values.  64 where enough workgroups are left: 8000
// tokens of 4 heads of 128 are appended in 23.1 us, 24.1 with 16.
int value_rows(int64_t rows, int64_t kv_heads, int teams) {
    return rows * kv_heads >= 64 * kFull / 8 ? 64 : teams;
}

// The workgroups of an append, see AppendSplit.
struct AppendGrid {
    int each, v_rows;
    int64_t parts, v_groups, all;

    AppendGrid(int64_t tokens, int64_t q_heads, int64_t kv_heads, int head_dim, int bits) {
        const int teams = kThreads / (head_dim / 8);
        const int64_t heads = q_heads + (bits == 4 ? 1 : 2) * kv_heads, runs = (tokens + teams - 1) / teams;
        // Four heads to a team where enough workgroups are left: at 16 + 4 heads of 128, 4 bits, 64 tokens take 3.4 us
        // with one head and 5.8 with four, 1500 8.7 and 9.2, 3500 13.3 and 12.6; at 8 + 4 heads of 256, 16 bits, 300
        // tokens 3.7 and 4.5, 1000 5.6 and 5.5, 2500 9.3 and 8.5, 20000 61 and 45.
        each = runs * heads >= 2 * kFull ? 4 : 1;
        parts = (heads + each - 1) / each;
        v_rows = bits == 4 ? value_rows(tokens, kv_heads, teams) : 0;
        v_groups = bits == 4 ? (tokens + v_rows - 1) / v_rows * kv_heads : 0;
        all = runs * parts + v_groups;
    }
};

// The workgroups of a gather.
struct GatherGrid {
    int v_rows;
    int64_t v_groups, all;

    GatherGrid(int64_t rows, int64_t kv_heads, int head_dim, int bits) {
        const int teams = kThreads / (head_dim / 8);
        v_rows = value_rows(rows, kv_heads, teams);
        v_groups = bits == 4 ? (rows + v_rows - 1) / v_rows * kv_heads : 0;
        all = (rows * (bits == 4 ? 1 : 2) * kv_heads + teams - 1) / teams + v_groups;
    }
};

}  // namespace

int64_t rope_append_groups(int64_t tokens, int64_t heads, int64_t kv_heads, int head_dim, int bits) {
    return AppendGrid(tokens, heads, kv_heads, head_dim, bits).all;
}

int64_t kv_gather_groups(int64_t rows, int64_t kv_heads, int head_dim, int bits) {
    return GatherGrid(rows, kv_heads, head_dim, bits).all;
}

int launch_rope_append(const AppendArgs& p, int head_dim, int bits, int dtype, hipStream_t s) {
    const AppendGrid g(p.tokens, p.heads, p.cache.kv_heads, head_dim, bits);
    const AppendSplit sp{p, static_cast<int32_t>(g.parts), g.v_rows, static_cast<int32_t>(g.v_groups)};
    const int each = g.each;
    const dim3 grid(static_cast<uint32_t>(g.all));
    return pick(dtype, head_dim, bits, [&](auto dt, auto d, auto b) {
        if (each == 4)
            hipLaunchKernelGGL((rope_append_kernel<dt.value, d.value, b.value, 4>), grid, dim3(kThreads), 0, s, sp);
        else
            hipLaunchKernelGGL((rope_append_kernel<dt.value, d.value, b.value, 1>), grid, dim3(kThreads), 0, s, sp);
        return check_launch("rope_append");
    });
}

int launch_kv_gather(const GatherArgs& p, int head_dim, int bits, int dtype, hipStream_t s) {
    const GatherGrid g(p.rows, p.cache.kv_heads, head_dim, bits);
    const dim3 grid(static_cast<uint32_t>(g.all));
    return pick(dtype, head_dim, bits, [&](auto dt, auto d, auto b) {
        hipLaunchKernelGGL((kv_gather_kernel<dt.value, d.value, b.value>), grid, dim3(kThreads), 0, s, p, g.v_rows,
                           static_cast<int>(g.v_groups));
        return check_launch("kv_gather");
    });
}

}  // namespace nvg
