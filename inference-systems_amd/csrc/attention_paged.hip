// Attention of one query token per sequence over a paged cache.
//
// For a key-value head the up to 16 query heads that share it are the columns
// of a 16 x 16 x 32 matrix product, so each cached byte is read once for all of
// them.  A wave takes 32 tokens at a time, straight from global memory into
// registers:
//   S^T[token, head] = K Q^T     A rows are tokens; accumulator i of lane l is
//                                token 4 (l / 16) + i, head l % 16
//   P = 2^(c S - c max)          online softmax, the head's maximum in its lanes
//   O^T[channel, head] += V^T P  contraction over tokens: the order of the
//                                accumulators of S^T is taken as the order of the
//                                contraction, so P is packed where it is
// V^T needs 8 tokens of one channel per lane.  16-bit pages give that by a
// 2 x 2 transposition in registers, 4-bit pages by their layout (4 tokens of a
// channel in one word).
//
// 4 bits: with an element c s + m, s and m per token and 64 channels,
//   S = sum_g s_g (sum c q) + m_g (sum q): products on the codes (16 + c as a
//   16-bit float, from bits alone), the rest in fp32 on the accumulators;
//   O = sum_t (P s_g) (c - 7.5) + sum_t P (m_g + 7.5 s_g): the products take P s_g
//   in fp16 against 64 + c, the sum of P s_g is taken off in fp32, and one more
//   product adds up P (m_g + 7.5 s_g) and P.  Around its middle a group's values
//   are small, so the roundings of P s_g and P weigh as much as they would on
//   the values themselves (131072 tokens, fp16: 6.2e-4 off with c and m_g
//   taken apart and 1024 + c, 2.8e-4 so).
//
// The work is split over a fixed grid: all (sequence, key-value head) pairs in
// units of 128 tokens, laid end to end, each workgroup an equal run of units.
// The lengths are read on the device, so a captured graph follows them.  A pair
// that lies in one run is finished there; the parts of others go to a workspace
// (at most two per workgroup) and a second kernel joins them.
#include <type_traits>

#include "attention_common.hpp"

namespace nvg {
namespace {

constexpr int kUnit = 128;          // tokens of a unit: 4 waves x 32
constexpr int kMaxGroups = 512;     // workgroups of the grid: two per CU
constexpr float kBoost = 10.0f;     // P is held as 2^10 p, see the kernel

struct Division { uint32_t mul; int shift; };   // x / d for x < 2^27

struct Split {
    PagedArgs a;
    Division pages;    // tokens / 16 -> page
    int32_t cap;       // tokens a table holds
    int32_t vheads;    // key-value heads x blocks of 16 query heads
    int32_t qblocks;
    int32_t group;     // query heads per key-value head
    int32_t grid;
};

__device__ __forceinline__ int divide(int x, Division d) {
    return int((uint64_t(uint32_t(x)) * d.mul) >> d.shift);
}

// Units of a sequence, one at least: an empty one still has its output written.
__device__ __forceinline__ int units_of(int len, int cap) {
    const int n = min(max(len, 0), cap);
    return max(1, (n + kUnit - 1) / kUnit);
}

// Every wave adds the lengths up for itself, 64 sequences at a time.
__device__ __forceinline__ int all_units(const Split& s) {
    const int lane = threadIdx.x & 63;
    int mine = 0;
    for (int b = lane; b < s.a.batch; b += 64) mine += units_of(s.a.lens[b], s.cap);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) mine += __shfl_xor(mine, off);
    return uniform(mine) * s.vheads;
}

__device__ __forceinline__ void find_unit(const Split& s, int unit, int& seq, int& first) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int b0 = 0; b0 < s.a.batch; b0 += 64) {
        const int u = b0 + lane < s.a.batch ? units_of(s.a.lens[b0 + lane], s.cap) : 0;
        int sum = u;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int up = __shfl_up(sum, off);
            if (lane >= off) sum += up;
        }
        const uint64_t past = __ballot((base + sum) * s.vheads > unit);
        if (past) {
            const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
            seq = uniform(b0 + at);
            first = uniform((base + __shfl(sum - u, at)) * s.vheads);
            return;
        }
        base += uniform(__shfl(sum, 63));
    }
    seq = s.a.batch;   // not reached for a unit below the total
    first = unit;
}

// The value lane N of each row of 16 lanes holds, in all of the row.
template <int N>
__device__ __forceinline__ uint32_t row_lane(uint32_t x) {
    return __builtin_amdgcn_update_dpp(0u, x, 0x150 + N, 0xf, 0xf, false);
}
template <int N>
__device__ __forceinline__ float row_lane(float x) {
    return __builtin_bit_cast(float, row_lane<N>(__builtin_bit_cast(uint32_t, x)));
}

// 8 key codes of a word as 16 + code in the operand type, channels in order.
template <int DT>
__device__ __forceinline__ u32x4_t key_codes(uint32_t w) {
    if constexpr (DT == NANOVLLM_GEMM_BF16) {   // 16.0 is 0x4180, a code its bits 3..6
        constexpr uint32_t mask = 0x00780078u, one = 0x41804180u;
        return u32x4_t{((w << 3) & mask) | one, ((w >> 1) & mask) | one, ((w >> 5) & mask) | one,
                       ((w >> 9) & mask) | one};
    } else {                                    // 16.0 is 0x4c00, a code its bits 6..9
        constexpr uint32_t mask = 0x03c003c0u, one = 0x4c004c00u;
        return u32x4_t{((w << 6) & mask) | one, ((w << 2) & mask) | one, ((w >> 2) & mask) | one,
                       ((w >> 6) & mask) | one};
    }
}

// m + 7.5 s of two words (scale, minimum).
__device__ __forceinline__ uint32_t group_middle(uint32_t a, uint32_t b) {
    const f16x2_t s = __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(b, a, 0x05040100u));
    const f16x2_t m = __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(b, a, 0x07060302u));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(s, f16x2_t{7.5, 7.5}, m));
}

// The partial result of a workgroup's run: rows of fp32 sums, then the maxima
// and the totals of P, for up to 16 query heads.
template <int D>
__device__ __forceinline__ float* part(const Split& s, int slot) {
    const int rows = min(16, s.group);
    return s.a.partial + int64_t(slot) * rows * (D + 4);
}

template <int DT, int D, int BITS>
struct Tile;

// 32 tokens of a 16-bit cache.
template <int DT, int D>
struct Tile<DT, D, 16> {
    static constexpr int E = D >= 128 ? 8 : 4;     // channels of a lane's load of V
    static constexpr int NB = D / (16 * E);        // such loads per token
    static constexpr int KS = D / 32;              // steps of the contraction over channels
    u32x4_t k[2][KS];
    uint32_t v[2][4][NB][E / 2];
    __device__ __forceinline__ static int q_channel(int step, int quad) { return 32 * step + 8 * quad; }
    __device__ __forceinline__ static int out_channel(int nb, int row) { return 16 * E * nb + E * row; }
};

// 32 tokens of a 4-bit cache.
template <int DT, int D>
struct Tile<DT, D, 4> {
    static constexpr int E = 4;
    static constexpr int NB = D / kGroup;          // groups
    static constexpr int KS = D / 32;
    static constexpr int WL = D >= 128 ? 4 : 2;    // words of a lane's load
    static constexpr int NL = D / 32 / WL;         // such loads
    uint32_t k[2][NL][WL], v[2][NL][WL];
    uint32_t ka[2];                                // key scale and minimum of token l % 16, group l / 16
    uint32_t kb[2], vb[2];                         // of the token and group that row_lane() takes from this lane
    u32x4_t vm[2];                                 // value scales and minima, 4 tokens of group l % 16
    __device__ __forceinline__ static int q_channel(int step, int quad) {
        return kGroup * (step / 2) + 16 * quad + 8 * (step % 2);
    }
    __device__ __forceinline__ static int out_channel(int nb, int row) { return kGroup * nb + 4 * row; }
};

template <int DT, int D, int BITS>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attention_paged_kernel(const Split s) {
    using T = Tile<DT, D, BITS>;
    constexpr int KS = T::KS, E = T::E, NB = T::NB;
    constexpr int PT = BITS == 4 ? NANOVLLM_GEMM_F16 : DT;   // type of P and of V's operand
    // P is held as 2^10 p where it is rounded to fp16, so that small
    // probabilities stay normal numbers; 2^10 cancels in O / l.
    constexpr bool kHalfP = PT == NANOVLLM_GEMM_F16;
    __shared__ float sm[4][16], sl[4][16];
    __shared__ __attribute__((aligned(16))) float so[2][16][D + 4];

    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const Cache& cache = s.a.cache;
    const int total = all_units(s);
    const int per = (total + s.grid - 1) / s.grid;
    int unit = int(blockIdx.x) * per;
    const int end = min(unit + per, total);
    if (unit >= end) return;
    int b, first;
    find_unit(s, unit, b, first);

    while (unit < end && b < s.a.batch) {
        const int raw_len = uniform(s.a.lens[b]);
        const int len = min(max(raw_len, 0), s.cap);
        const int units = units_of(raw_len, s.cap);
        const int rel = unit - first, vh = rel / units, u0 = rel - vh * units;
        const int n = min(units - u0, end - unit);
        const int kvh = vh / s.qblocks, qb = vh - kvh * s.qblocks;
        const int rows = min(16, s.group - 16 * qb);
        const int t_begin = u0 * kUnit, t_end = min(len, (u0 + n) * kUnit);

        // Queries: column `col`, 8 channels per step.
        u32x4_t q[KS];
        {
            const int head = kvh * s.group + qb * 16 + (col < rows ? col : 0);
            const uint16_t* src = s.a.q + b * s.a.q_row + head * s.a.q_head;
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                q[i] = load16(src + T::q_channel(i, quad));
                if (col >= rows) q[i] = u32x4_t{0, 0, 0, 0};
            }
        }
        float qsum[BITS == 4 ? NB : 1], qpick = 0.0f;
        if constexpr (BITS == 4) {
#pragma unroll
            for (int g = 0; g < NB; ++g) {
                float x = 0.0f;
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int w = 0; w < 4; ++w)
                        x += half_to_f32<DT>(uint16_t(q[2 * g + e][w])) + half_to_f32<DT>(uint16_t(q[2 * g + e][w] >> 16));
                qsum[g] = sum_across16(sum_across32(x));
                if (quad == g) qpick = qsum[g];
            }
        }

        f32x4_t o[NB][E], extra = {0, 0, 0, 0};
        float psum[BITS == 4 ? NB : 1] = {};
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < E; ++e) o[nb][e] = f32x4_t{0, 0, 0, 0};
        float m = -__builtin_inff();
        float boost = kHalfP ? kBoost : 0.0f;

        T tile;
        int page[2], in_page[2];
        bool bad[2];
        const int32_t* table = s.a.tables + b * s.a.table_stride;
        auto locate = [&](int t) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int t16 = t / 16 + h, idx = divide(t16, s.pages);
                const int id = idx < s.a.table_blocks && 16 * t16 < len ? table[idx] : 0;
                bad[h] = id < 0 || id >= cache.num_blocks || raw_len > s.cap;
                page[h] = uniform(id < 0 || id >= cache.num_blocks ? 0 : id);
                in_page[h] = uniform(16 * t16 - idx * cache.block_size);
            }
        };
        auto load_k = [&]() {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const char* base = cache.k + page[h] * cache.k_stride;
                if constexpr (BITS == 16) {
                    const char* row = base + (int64_t(in_page[h] + col) * cache.kv_heads + kvh) * (2 * D) + 16 * quad;
#pragma unroll
                    for (int i = 0; i < KS; ++i) tile.k[h][i] = load16(row + 64 * i);
                } else {
                    const int64_t line = int64_t(kvh) * cache.block_size + in_page[h];
                    const char* row = base + (line + col) * (D / 2) + 4 * T::WL * quad;
#pragma unroll
                    for (int i = 0; i < T::NL; ++i) {
                        if constexpr (T::WL == 4) {
                            const u32x4_t w = load16(row + 64 * i);
#pragma unroll
                            for (int j = 0; j < 4; ++j) tile.k[h][i][j] = w[j];
                        } else {
                            const u32x2_t w = *reinterpret_cast<const u32x2_t*>(row);
                            tile.k[h][i][0] = w[0];
                            tile.k[h][i][1] = w[1];
                        }
                    }
                    const char* sc = cache.k_scales + page[h] * cache.ks_stride + 4 * NB * line;
                    tile.ka[h] = *reinterpret_cast<const uint32_t*>(sc + 4 * (NB * col + (NB > 1 ? quad % NB : 0)));
                    tile.kb[h] = *reinterpret_cast<const uint32_t*>(
                        sc + 4 * (NB * (4 * quad + (col / NB) % 4) + col % NB));
                }
            }
        };
        auto load_v = [&]() {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const char* base = cache.v + page[h] * cache.v_stride;
                if constexpr (BITS == 16) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const char* row = base +
                            (int64_t(in_page[h] + 4 * quad + i) * cache.kv_heads + kvh) * (2 * D) + 2 * E * col;
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            if constexpr (E == 8) {
                                const u32x4_t w = load16(row + 256 * nb);
#pragma unroll
                                for (int j = 0; j < 4; ++j) tile.v[h][i][nb][j] = w[j];
                            } else {
                                const u32x2_t w = *reinterpret_cast<const u32x2_t*>(row);
                                tile.v[h][i][0][0] = w[0];
                                tile.v[h][i][0][1] = w[1];
                            }
                        }
                    }
                } else {
                    const int64_t line = int64_t(kvh) * cache.block_size + in_page[h];
                    const char* row = base + (line + 4 * quad) * (D / 2) + 4 * T::WL * col;
#pragma unroll
                    for (int i = 0; i < T::NL; ++i) {
                        if constexpr (T::WL == 4) {
                            const u32x4_t w = load16(row + 256 * i);
#pragma unroll
                            for (int j = 0; j < 4; ++j) tile.v[h][i][j] = w[j];
                        } else {
                            const u32x2_t w = *reinterpret_cast<const u32x2_t*>(row);
                            tile.v[h][i][0] = w[0];
                            tile.v[h][i][1] = w[1];
                        }
                    }
                    const char* sc = cache.v_scales + page[h] * cache.vs_stride;
                    auto at = [&](int g, int tok) {
                        return sc + 4 * ((int64_t(kvh) * NB + g) * cache.block_size + in_page[h] + tok);
                    };
                    tile.vb[h] = *reinterpret_cast<const uint32_t*>(at(col % NB, 4 * quad + (col / NB) % 4));
                    tile.vm[h] = load16(at(col < NB ? col : 0, 4 * quad));
                }
            }
        };

        int t = t_begin + 32 * wave;
        if (t < t_end) {
            locate(t);
            load_k();
            load_v();
        }
        for (; t < t_end; t += kUnit) {
            const bool poison[2] = {bad[0], bad[1]};
            const bool ragged = t + 32 > t_end;      // only where the sequence ends: units are whole tiles
            // S^T
            f32x4_t sc[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if constexpr (BITS == 16) {
                    sc[h] = f32x4_t{0, 0, 0, 0};
#pragma unroll
                    for (int i = 0; i < KS; ++i) sc[h] = mfma_16x16x32<DT>(tile.k[h][i], q[i], sc[h]);
                } else {
                    const float low = NB == 4 || quad < NB ? f16_to_f32(uint16_t(tile.ka[h] >> 16)) : 0.0f;
                    sc[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(low, qpick, f32x4_t{0, 0, 0, 0}, 0, 0, 0);
                    const float ks = f16_to_f32(uint16_t(tile.kb[h]));
                    static_for<NB>([&](auto gc) {
                        constexpr int g = gc.value;
                        const float z = -16.0f * qsum[g];
                        f32x4_t acc = {z, z, z, z};
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            acc = mfma_16x16x32<DT>(key_codes<DT>(tile.k[h][(2 * g + e) / T::WL][(2 * g + e) % T::WL]),
                                                    q[2 * g + e], acc);
                        static_for<4>([&](auto ic) {
                            constexpr int i = ic.value;
                            sc[h][i] = __builtin_fmaf(row_lane<g + NB * i>(ks), acc[i], sc[h][i]);
                        });
                    });
                }
            }
            if (ragged) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (t + 16 * h + 4 * quad + i >= t_end) sc[h][i] = -__builtin_inff();
            }
            if (poison[0] || poison[1]) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (poison[h] && t + 16 * h + 4 * quad + i < t_end) sc[h][i] = __builtin_nanf("");
            }
            // The next tile's keys travel while this one's softmax runs.
            const bool more = t + kUnit < t_end;
            if (more) {
                locate(t + kUnit);
                load_k();
            }
            // Softmax
            float top = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                              fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
            top = max_across32(max_across16(top));
            if constexpr (BITS == 4) {
                // 2^10 p s has to fit fp16.  Where a scale is too large for that,
                // this and the following tiles go without the factor.
                const float big = fmaxf(f16_to_f32(uint16_t(tile.vb[0])), f16_to_f32(uint16_t(tile.vb[1])));
                if (boost != 0.0f && __ballot(big > 32.0f)) {
                    const float down = exp2_hw(-kBoost);
                    boost = 0.0f;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        psum[nb] *= down;
#pragma unroll
                        for (int e = 0; e < E; ++e) o[nb][e] *= down;
                    }
                    extra *= down;
                }
            }
            if (__ballot(top > m)) {
                const float higher = fmaxf(m, top);
                const float down = higher == -__builtin_inff() ? 1.0f : exp2_hw((m - higher) * s.a.c);
                m = higher;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    if constexpr (BITS == 4) psum[nb] *= down;
#pragma unroll
                    for (int e = 0; e < E; ++e) o[nb][e] *= down;
                }
                extra *= down;
            }
            const float shift = (m == -__builtin_inff() ? 0.0f : m * s.a.c) - boost;
            float p[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) p[h][i] = exp2_hw(__builtin_fmaf(sc[h][i], s.a.c, -shift));
            if constexpr (BITS == 16) {
                if (ragged) {   // cached rows behind the end may hold anything
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (t + 16 * h + 4 * quad + i >= t_end)
#pragma unroll
                                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                                    for (int j = 0; j < E / 2; ++j) tile.v[h][i][nb][j] = 0;
                }
                const u32x4_t pk = {pack2<PT>(p[0][0], p[0][1]), pack2<PT>(p[0][2], p[0][3]),
                                    pack2<PT>(p[1][0], p[1][1]), pack2<PT>(p[1][2], p[1][3])};
                constexpr uint32_t one = DT == NANOVLLM_GEMM_BF16 ? 0x3f803f80u : 0x3c003c00u;
                extra = mfma_16x16x32<PT>(u32x4_t{one, one, one, one}, pk, extra);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        constexpr uint32_t even = 0x05040100u, odd = 0x07060302u;
                        const uint32_t sel = e % 2 ? odd : even;
                        u32x4_t a;
#pragma unroll
                        for (int w = 0; w < 4; ++w)
                            a[w] = __builtin_amdgcn_perm(tile.v[w / 2][2 * (w % 2) + 1][nb][e / 2],
                                                         tile.v[w / 2][2 * (w % 2)][nb][e / 2], sel);
                        o[nb][e] = mfma_16x16x32<PT>(a, pk, o[nb][e]);
                    }
            } else {
                if (ragged) {   // scales behind the end may be NaN
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (t + 16 * h + 4 * quad + (col / NB) % 4 >= t_end) tile.vb[h] = 0;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (t + 16 * h + 4 * quad + i >= t_end) tile.vm[h][i] = 0;
                    }
                }
                // Tokens of an operand in the order 0 2 1 3 of each four.
                u32x4_t pk, am;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        pk[2 * h + i] = pack2<PT>(p[h][i], p[h][i + 2]);
                        am[2 * h + i] = group_middle(tile.vm[h][i], tile.vm[h][i + 2]);
                    }
                // Rows 0 .. NB - 1: sums of P (m_g + 7.5 s_g); row 4: of P.
#pragma unroll
                for (int w = 0; w < 4; ++w) am[w] = col < NB ? am[w] : col == 4 ? 0x3c003c00u : 0u;
                extra = mfma_16x16x32<PT>(am, pk, extra);
                const float vs[2] = {f16_to_f32(uint16_t(tile.vb[0])), f16_to_f32(uint16_t(tile.vb[1]))};
                static_for<NB>([&](auto gc) {
                    constexpr int g = gc.value;
                    u32x4_t ps;
                    static_for<2>([&](auto hc) {
                        constexpr int h = hc.value;
                        ps[2 * h] = pack2<PT>(p[h][0] * row_lane<g>(vs[h]), p[h][2] * row_lane<g + NB * 2>(vs[h]));
                        ps[2 * h + 1] =
                            pack2<PT>(p[h][1] * row_lane<g + NB>(vs[h]), p[h][3] * row_lane<g + NB * 3>(vs[h]));
                    });
#pragma unroll
                    for (int w = 0; w < 4; ++w)
                        psum[g] = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, uint32_t(ps[w])),
                                                         f16x2_t{1, 1}, psum[g], false);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t x0 = tile.v[0][(2 * g + j) / T::WL][(2 * g + j) % T::WL];
                        const uint32_t x1 = tile.v[1][(2 * g + j) / T::WL][(2 * g + j) % T::WL];
                        // 16 (64 + c): 1024 is 0x6400, a code its bits 4..7.
                        constexpr uint32_t mask = 0x00f000f0u, k1024 = 0x64006400u;
                        o[g][2 * j] = mfma_16x16x32<PT>(
                            u32x4_t{((x0 << 4) & mask) | k1024, ((x0 >> 4) & mask) | k1024,
                                    ((x1 << 4) & mask) | k1024, ((x1 >> 4) & mask) | k1024}, ps, o[g][2 * j]);
                        o[g][2 * j + 1] = mfma_16x16x32<PT>(
                            u32x4_t{(x0 & mask) | k1024, ((x0 >> 8) & mask) | k1024, (x1 & mask) | k1024,
                                    ((x1 >> 8) & mask) | k1024}, ps, o[g][2 * j + 1]);
                    }
                });
            }
            if (more) load_v();
        }

        // The head's total of P and, in 4 bits, what the products left out.
        float l = extra[0];
        if constexpr (BITS == 4) {
            l = __shfl(extra[0], 16 + col);
#pragma unroll
            for (int g = 0; g < NB; ++g) {
                const float middle = __shfl(extra[g], col);
                const float off = 16.0f * (64.0f + 7.5f) * sum_across16(sum_across32(psum[g]));
#pragma unroll
                for (int e = 0; e < E; ++e)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        o[g][e][i] = __builtin_fmaf(o[g][e][i] - off, 0.0625f, middle);
            }
        }
        if constexpr (kHalfP) {
            const float down = exp2_hw(-boost);
            l *= down;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < E; ++e) o[nb][e] *= down;
        }

        // Join the waves that had tokens.
        const bool several = t_end - t_begin > 32;
        if (several) {
            if (quad == 0) {
                sm[wave][col] = m;
                sl[wave][col] = l;
            }
            __syncthreads();
            float top = sm[0][col];
#pragma unroll
            for (int w = 1; w < 4; ++w) top = fmaxf(top, sm[w][col]);
            l = 0.0f;
            float mine = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = sm[w][col] == -__builtin_inff() ? 0.0f : exp2_hw((sm[w][col] - top) * s.a.c);
                // A wave whose maximum is -infinity has no part but NaN.
                l += sm[w][col] == -__builtin_inff() ? sl[w][col] : f * sl[w][col];
                if (w == wave) mine = sm[w][col] == -__builtin_inff() ? 1.0f : f;
            }
            m = top;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < E; ++e) o[nb][e] *= mine;
            auto put = [&](int slot) {
                if (col < rows)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int e = 0; e < E; e += 4)
                                *reinterpret_cast<f32x4_t*>(&so[slot][col][T::out_channel(nb, 4 * quad + i) + e]) =
                                    f32x4_t{o[nb][e][i], o[nb][e + 1][i], o[nb][e + 2][i], o[nb][e + 3][i]};
            };
            auto add = [&](int slot) {
                if (col < rows)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int e = 0; e < E; e += 4) {
                                const f32x4_t x = *reinterpret_cast<const f32x4_t*>(
                                    &so[slot][col][T::out_channel(nb, 4 * quad + i) + e]);
#pragma unroll
                                for (int j = 0; j < 4; ++j) o[nb][e + j][i] += x[j];
                            }
            };
            if (wave >= 2) put(wave - 2);
            __syncthreads();
            if (wave < 2) add(wave);
            if (wave == 1) put(1);
            __syncthreads();
            if (wave == 0) add(1);
        }
        if (wave == 0 && col < rows) {
            if (n == units) {
                const int head = kvh * s.group + qb * 16 + col;
                uint16_t* out = s.a.out + (int64_t(b) * s.a.heads + head) * D;
                const float inv = 1.0f / l;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int e = 0; e < E; e += 4) {
                            float y[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                y[j] = raw_len > s.cap ? __builtin_nanf("") : len == 0 ? 0.0f : o[nb][e + j][i] * inv;
                            *reinterpret_cast<u32x2_t*>(out + T::out_channel(nb, 4 * quad + i) + e) =
                                u32x2_t{pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3])};
                        }
            } else {
                const int most = min(16, s.group);
                float* dst = part<D>(s, 2 * int(blockIdx.x) + (u0 == 0 ? 1 : 0));
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int e = 0; e < E; e += 4)
                            *reinterpret_cast<f32x4_t*>(dst + col * D + T::out_channel(nb, 4 * quad + i) + e) =
                                f32x4_t{o[nb][e][i], o[nb][e + 1][i], o[nb][e + 2][i], o[nb][e + 3][i]};
                if (quad == 0) {
                    dst[most * D + col] = m;
                    dst[most * D + most + col] = l;
                }
            }
        }
        unit += n;
        if (unit - first >= units * s.vheads) {
            first = unit;
            ++b;
        }
    }
}

// Joins the parts of a (sequence, key-value head) pair that lies in several
// runs: one workgroup per query head of it.  Parts are added in a fixed order.
template <int DT, int D>
__global__ __launch_bounds__(256) void attention_paged_join_kernel(const Split s) {
    constexpr int TPR = D / 4, ROWS = 256 / TPR;      // threads per row of channels, parts added at once
    __shared__ float weight[kMaxGroups];
    __shared__ float red[4];
    __shared__ __attribute__((aligned(16))) float acc[ROWS][D];
    const int tid = threadIdx.x;
    const int vh = int(blockIdx.x) % s.vheads, b = int(blockIdx.x) / s.vheads, row = blockIdx.y;
    const int kvh = vh / s.qblocks, qb = vh - kvh * s.qblocks;
    if (row >= s.group - 16 * qb) return;
    // First unit of the pair.
    const int lane = tid & 63;
    int before = 0, all = 0;
    for (int i = lane; i < s.a.batch; i += 64) {
        const int u = units_of(s.a.lens[i], s.cap);
        all += u;
        if (i < b) before += u;
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        all += __shfl_xor(all, off);
        before += __shfl_xor(before, off);
    }
    const int units = units_of(s.a.lens[b], s.cap);
    const int per = (all * s.vheads + s.grid - 1) / s.grid;
    const int begin = before * s.vheads + vh * units, end = begin + units;
    const int w0 = begin / per, w1 = (end - 1) / per;
    if (w0 == w1) return;
    const int n = w1 - w0 + 1, most = min(16, s.group);
    auto source = [&](int i) { return part<D>(s, 2 * (w0 + i) + (i == 0 ? 1 : 0)); };

    float top = -__builtin_inff();
    for (int i = tid; i < n; i += 256) top = fmaxf(top, source(i)[most * D + row]);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
    if (lane == 0) red[tid >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    __syncthreads();
    float l = 0.0f;
    for (int i = tid; i < n; i += 256) {
        const float m = source(i)[most * D + row];
        const float f = m == -__builtin_inff() ? 1.0f : exp2_hw((m - top) * s.a.c);
        weight[i] = f;
        l += f * source(i)[most * D + most + row];
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) l += __shfl_xor(l, off);
    if (lane == 0) red[tid >> 6] = l;
    __syncthreads();
    l = (red[0] + red[1]) + (red[2] + red[3]);
    f32x4_t o = {0, 0, 0, 0};
    const int ch = 4 * (tid % TPR), r = tid / TPR;
#pragma unroll 4
    for (int i = r; i < n; i += ROWS) {
        const f32x4_t x = *reinterpret_cast<const f32x4_t*>(source(i) + row * D + ch);
        const float f = weight[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = __builtin_fmaf(f, x[j], o[j]);
    }
    *reinterpret_cast<f32x4_t*>(&acc[r][ch]) = o;
    __syncthreads();
    if (tid < TPR) {
#pragma unroll
        for (int i = 1; i < ROWS; ++i) o += *reinterpret_cast<const f32x4_t*>(&acc[i][ch]);
        const float inv = 1.0f / l;
        const int head = kvh * s.group + qb * 16 + row;
        const bool over = s.a.lens[b] > s.cap;
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = over ? __builtin_nanf("") : o[j] * inv;
        *reinterpret_cast<u32x2_t*>(s.a.out + (int64_t(b) * s.a.heads + head) * D + ch) =
            u32x2_t{pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3])};
    }
}

// Workgroups of the grid: as many as there can be units, at most two per CU.
int grid_of(int64_t batch, int64_t vheads, int64_t table_tokens) {
    const int64_t per = table_tokens > kUnit ? (table_tokens + kUnit - 1) / kUnit : 1;
    const int64_t units = batch * vheads * per;
    return units < kMaxGroups ? static_cast<int>(units) : kMaxGroups;
}

template <int DT, int D, int BITS>
int launch(const Split& s, hipStream_t stream) {
    hipLaunchKernelGGL((attention_paged_kernel<DT, D, BITS>), dim3(s.grid), dim3(256), 0, stream, s);
    int rc = check_launch("attention_paged");
    if (rc != NANOVLLM_GEMM_OK || s.cap <= kUnit) return rc;   // every pair is one unit: nothing to join
    const dim3 grid(static_cast<uint32_t>(s.a.batch * s.vheads), static_cast<uint32_t>(s.group < 16 ? s.group : 16));
    hipLaunchKernelGGL((attention_paged_join_kernel<DT, D>), grid, dim3(256), 0, stream, s);
    return check_launch("attention_paged_join");
}

template <int DT, int D>
int launch_bits(const Split& s, int bits, hipStream_t stream) {
    return bits == 4 ? launch<DT, D, 4>(s, stream) : launch<DT, D, 16>(s, stream);
}

template <int DT>
int launch_dim(const Split& s, int head_dim, int bits, hipStream_t stream) {
    return head_dim == 64    ? launch_bits<DT, 64>(s, bits, stream)
           : head_dim == 128 ? launch_bits<DT, 128>(s, bits, stream)
                             : launch_bits<DT, 256>(s, bits, stream);
}

}  // namespace

int64_t attention_paged_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                  int64_t table_tokens) {
    if (table_tokens <= kUnit) return 0;
    const int64_t group = heads / kv_heads, vheads = kv_heads * ((group + 15) / 16);
    return int64_t(2) * grid_of(batch, vheads, table_tokens) * (group < 16 ? group : 16) * (head_dim + 4) * 4;
}

int launch_attention_paged(const PagedArgs& p, int head_dim, int bits, int dtype, hipStream_t stream) {
    Split s;
    s.a = p;
    s.cap = p.table_blocks * p.cache.block_size;
    s.group = p.heads / p.cache.kv_heads;
    s.qblocks = (s.group + 15) / 16;
    s.vheads = p.cache.kv_heads * s.qblocks;
    s.grid = grid_of(p.batch, s.vheads, s.cap);
    // x / d for x < 2^27 as (x mul) >> shift, mul = ceil(2^shift / d), shift = 27 + ceil(log2 d).
    const uint32_t d = static_cast<uint32_t>(p.cache.block_size / 16);
    int bits_d = 0;
    while ((uint64_t(1) << bits_d) < d) ++bits_d;
    s.pages.shift = 27 + bits_d;
    s.pages.mul = static_cast<uint32_t>(((uint64_t(1) << s.pages.shift) + d - 1) / d);
    return dtype == NANOVLLM_GEMM_BF16 ? launch_dim<NANOVLLM_GEMM_BF16>(s, head_dim, bits, stream)
                                       : launch_dim<NANOVLLM_GEMM_F16>(s, head_dim, bits, stream);
}

}  // namespace nvg
