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
// P is rounded to the operands' type for its product, and its total is that of the
// rounded P: 0.0021 off in bf16 against 64 bits, 0.0017 with P in fp32.
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
//   taken apart and 1024 + c, 2.8e-4 so).  P is held 2^10 fold in fp16 (here and in
//   16-bit fp16 pages), so that P, or P s_g, is lost below 2^-35 of the largest P.
//
// The work is split over a fixed grid: all (sequence, key-value head) pairs in
// units of 128 tokens, laid end to end, each workgroup an equal run of units.
// A pair starts with a few units that hold no token and stand for what it costs
// to begin one.  The lengths are read on the device, so a captured graph follows
// them.  A pair whose tokens lie in one run is finished there; the parts of
// others go to a workspace (at most two per workgroup) and a second kernel joins
// them.
//
// Bound by HBM in 16 bits: on MI355X 32 sequences of 4100 tokens, 2 heads of 256,
// take 58 us, 53 of them at 5.05 TB/s (a large copy: 5.1).  In 4 bits by the
// vector instructions that turn codes into numbers as much as by the pages: 64
// sequences of 1 to 16000 tokens (8 heads of 128, 173 MB) 48.6 us, 131072 tokens
// (2 heads of 256, 75 MB) 29 us; 4000 tokens 12.8 us, all latency.
#include <type_traits>

#include "attention_common.hpp"

namespace nvg {
namespace {

constexpr int kUnit = 128;          // tokens of a unit: 4 waves x 32
constexpr int kBegin = 3;           // units a pair costs before its first token
constexpr int kMaxGroups = 1024;    // workgroups of any grid, see resident()
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
    int32_t many;        // units from which half of the grid takes them all
    uint32_t k_pages, v_pages, ks_pages, vs_pages;   // bytes between pages, / 16
};

__device__ __forceinline__ int divide(int x, Division d) {
    return int((uint64_t(uint32_t(x)) * d.mul) >> d.shift);
}

// Units of a pair: kBegin, then those of its tokens, one at least, since an
// empty sequence has its output written too.
__device__ __forceinline__ int units_of(int len, int cap) {
    const int n = min(max(len, 0), cap);
    return kBegin + max(1, (n + kUnit - 1) / kUnit);
}

// The units of all pairs, per sequence in a lane: every wave adds them up for
// itself, 64 sequences at a time.
struct Units { int total, len, mine, sum; };    // all of them; of sequence `lane` of the last 64: its length, units,
                                                // and the units up to it

__device__ __forceinline__ Units all_units(const Split& s) {
    const int lane = threadIdx.x & 63;
    Units u{0, 0, 0, 0};
    for (int b0 = 0; b0 < s.a.batch; b0 += 64) {
        u.len = s.a.lens[min(b0 + lane, s.a.batch - 1)];
        u.mine = b0 + lane < s.a.batch ? units_of(u.len, s.cap) : 0;
        u.sum = prefix_sum(u.mine);
        u.total += __builtin_amdgcn_readlane(u.sum, 63);
    }
    u.total *= s.vheads;
    return u;
}

// Units of a workgroup's run.  16-bit pages are bound by HBM, and where there is
// work for it half of the grid (at head_dim 256 as many workgroups as fit at once)
// stream it better and leave half of the parts: 32 sequences of 4100 tokens 64.7 ->
// 57.9 us (2 heads of 256), 62.4 -> 57.7 (4 of 128), 68.5 -> 63.4 (8 of 64); at 128
// and 64 not for every batch: 40 of 3000 63.5 -> 55.1, 56.4 -> 57.7, 55.5 -> 56.7.
// Where there is little, their number is what keeps loads in flight: 32 ragged
// sequences (64 pairs of 8 units or so) 27.8 us, 33.9 on half.  Pages of 4 bits wait
// on the arithmetic and take the whole grid.
__device__ __forceinline__ int units_per_group(const Split& s, int total) {
    const int groups = total >= s.many ? s.grid / 2 : s.grid;
    return (total + groups - 1) / groups;
}

// The sequence that holds a unit below the total, and its first unit.
__device__ __forceinline__ void find_unit(const Split& s, Units u, int unit, int& seq, int& first) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    seq = first = 0;
    for (int b0 = 0; b0 < s.a.batch; b0 += 64) {
        if (s.a.batch > 64) {      // else all_units has left them
            u.mine = b0 + lane < s.a.batch ? units_of(s.a.lens[b0 + lane], s.cap) : 0;
            u.sum = prefix_sum(u.mine);
        }
        const uint64_t past = __ballot((base + u.sum) * s.vheads > unit);
        if (past) {
            const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
            seq = b0 + at;
            first = (base + __builtin_amdgcn_readlane(u.sum - u.mine, at)) * s.vheads;
            return;
        }
        base += __builtin_amdgcn_readlane(u.sum, 63);
    }
}

// The value lane N of each row of 16 lanes holds, in all of the row.
template <int N>
__device__ __forceinline__ uint32_t row_lane(uint32_t x) {
    return __builtin_amdgcn_mov_dpp(x, 0x150 + N, 0xf, 0xf, true);
}
template <int N>
__device__ __forceinline__ float row_lane(float x) {
    return __builtin_bit_cast(float, row_lane<N>(__builtin_bit_cast(uint32_t, x)));
}

// The value of lane l + N of a row of 16 lanes (0 behind its end).
template <int N>
__device__ __forceinline__ uint32_t lane_ahead(uint32_t x) {
    return __builtin_amdgcn_mov_dpp(x, 0x100 + N, 0xf, 0xf, true);
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
    __device__ __forceinline__ static int q_channel(int step, int quad) {
        return kGroup * (step / 2) + 16 * quad + 8 * (step % 2);
    }
    __device__ __forceinline__ static int out_channel(int nb, int row) { return kGroup * nb + 4 * row; }
};

// Where 32 tokens lie: the page of each half and its first token there.
struct Where { int page[2], at[2]; bool bad[2]; };

__device__ __forceinline__ uint64_t page_offset(int page, uint32_t sixteenths) {
    return (uint64_t(uint32_t(page)) * sixteenths) << 4;
}

// N words (2 or 4) at a lane's place behind a lane-uniform address.
template <int N>
__device__ __forceinline__ void load_words(uint32_t (&dst)[N], const char* base, uint32_t off) {
    if constexpr (N == 4) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(base + off);
#pragma unroll
        for (int j = 0; j < 4; ++j) dst[j] = w[j];
    } else {
        const u32x2_t w = *reinterpret_cast<const u32x2_t*>(base + off);
        dst[0] = w[0];
        dst[1] = w[1];
    }
}

// A constant the compiler does not see: it would put a 32-bit literal into an
// instruction of its own where v_and_or_b32 takes registers.
__device__ __forceinline__ uint32_t in_vgpr(uint32_t x) {
    uint32_t r;
    asm("v_mov_b32 %0, %1" : "=v"(r) : "i"(x));
    return r;
}
__device__ __forceinline__ uint32_t in_sgpr(uint32_t x) {
    uint32_t r;
    asm("s_mov_b32 %0, %1" : "=s"(r) : "i"(x));
    return r;
}

template <int DT, int D, int BITS>
__global__ __launch_bounds__(256, D == 256 && BITS == 16 ? 1 : 2) void attention_paged_kernel(const Split s) {
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
    const Units all = all_units(s);
    const int per = units_per_group(s, all.total);
    int unit = int(blockIdx.x) * per;
    const int end = min(unit + per, all.total);
    if (unit >= end) return;
    int b, first;
    find_unit(s, all, unit, b, first);

    // 4 bits: 16 + c (keys) and 16 (64 + c) (values) from bits alone, two to a word.
    const uint32_t kmask = in_sgpr(DT == NANOVLLM_GEMM_BF16 ? 0x00780078u : 0x03c003c0u);
    const uint32_t kone = in_vgpr(DT == NANOVLLM_GEMM_BF16 ? 0x41804180u : 0x4c004c00u);
    const uint32_t vmask = in_sgpr(0x00f000f0u), vone = in_vgpr(0x64006400u);
    auto key_codes = [&](uint32_t w) {
        if constexpr (DT == NANOVLLM_GEMM_BF16)   // 16.0 is 0x4180, a code its bits 3..6
            return u32x4_t{((w << 3) & kmask) | kone, ((w >> 1) & kmask) | kone, ((w >> 5) & kmask) | kone,
                           ((w >> 9) & kmask) | kone};
        else                                      // 16.0 is 0x4c00, a code its bits 6..9
            return u32x4_t{((w << 6) & kmask) | kone, ((w << 2) & kmask) | kone, ((w >> 2) & kmask) | kone,
                           ((w >> 6) & kmask) | kone};
    };
    // 1024.0 is 0x6400, a code its bits 4..7.
    auto value_codes = [&](uint32_t w) { return (w & vmask) | vone; };

    const int token_bytes = cache.kv_heads * 2 * D;    // 16 bits
    // A lane's places in a run of 16 tokens, in bytes.
    uint32_t k_off, v_off, ka_off = 0, kb_off = 0, vb_off = 0;
    if constexpr (BITS == 16) {
        k_off = uint32_t(col * token_bytes + 16 * quad);
        v_off = uint32_t(4 * quad * token_bytes + 2 * E * col);
    } else {
        k_off = uint32_t(col * (D / 2) + 4 * T::WL * quad);
        v_off = uint32_t(4 * quad * (D / 2) + 4 * T::WL * col);
        ka_off = uint32_t(4 * (NB * col + quad % NB));
        kb_off = uint32_t(4 * (NB * (4 * quad + (col / NB) % 4) + col % NB));
        vb_off = uint32_t(4 * ((col % NB) * cache.block_size + 4 * quad + (col / NB) % 4));
    }

    while (unit < end && b < s.a.batch) {
        const int raw_len = s.a.batch <= 64 ? __builtin_amdgcn_readlane(all.len, b) : scalar_load(s.a.lens + b);
        const int len = min(max(raw_len, 0), s.cap);
        const int units = units_of(raw_len, s.cap);
        const int rel = unit - first, vh = rel / units, from = rel - vh * units;
        const int to = min(units, from + end - unit);
        unit += to - from;
        if (to <= kBegin) continue;      // the run ends before the pair's first token
        // Units of tokens: u0 .. u1.
        const int u0 = max(0, from - kBegin), u1 = to - kBegin;
        const bool whole = u0 == 0 && to == units;
        const int kvh = vh / s.qblocks, qb = vh - kvh * s.qblocks;
        const int rows = min(16, s.group - 16 * qb);
        const int t_begin = u0 * kUnit, t_end = min(len, u1 * kUnit);

        // The head's share of a page.
        const int64_t head_rows = int64_t(kvh) * (BITS == 16 ? 1 : cache.block_size);
        const char* k_head = cache.k + head_rows * (BITS == 16 ? 2 * D : D / 2);
        const char* v_head = cache.v + head_rows * (BITS == 16 ? 2 * D : D / 2);
        const char* ks_head = cache.k_scales + head_rows * (4 * NB);
        const char* vs_head = cache.v_scales + head_rows * (4 * NB);
        const int32_t* table = s.a.tables + b * s.a.table_stride;
        auto locate = [&](int t) {      // both entries are read, in the table or not, so that neither waits
            Where w;
            int idx[2], id[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                idx[h] = divide(t / 16 + h, s.pages);
                id[h] = scalar_load(table + min(idx[h], s.a.table_blocks - 1));
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const bool there = t + 16 * h < len, out = id[h] < 0 || id[h] >= cache.num_blocks;
                w.bad[h] = (there && out) || raw_len > s.cap;
                w.page[h] = there && !out ? id[h] : 0;
                w.at[h] = t + 16 * h - idx[h] * cache.block_size;
            }
            return w;
        };
        auto load_k = [&](T& tile, const Where& w) {
            asm volatile("" : "+v"(k_off), "+v"(ka_off), "+v"(kb_off));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if constexpr (BITS == 16) {
                    const char* kp = k_head + page_offset(w.page[h], s.k_pages) + uint32_t(w.at[h] * token_bytes);
#pragma unroll
                    for (int i = 0; i < KS; ++i) tile.k[h][i] = *reinterpret_cast<const u32x4_t*>(kp + 64 * i + k_off);
                } else {
                    const char* kp = k_head + page_offset(w.page[h], s.k_pages) + uint32_t(w.at[h] * (D / 2));
                    const char* sp = ks_head + page_offset(w.page[h], s.ks_pages) + uint32_t(w.at[h] * (4 * NB));
                    tile.ka[h] = *reinterpret_cast<const uint32_t*>(sp + ka_off);
                    tile.kb[h] = *reinterpret_cast<const uint32_t*>(sp + kb_off);
#pragma unroll
                    for (int i = 0; i < T::NL; ++i) load_words(tile.k[h][i], kp + 64 * i, k_off);
                }
            }
        };
        auto load_v = [&](T& tile, const Where& w) {
            asm volatile("" : "+v"(v_off), "+v"(vb_off));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if constexpr (BITS == 16) {
                    const char* vp = v_head + page_offset(w.page[h], s.v_pages) + uint32_t(w.at[h] * token_bytes);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb)
                            load_words(tile.v[h][i][nb], vp + uint32_t(i * token_bytes) + 256 * nb, v_off);
                } else {
                    const char* vp = v_head + page_offset(w.page[h], s.v_pages) + uint32_t(w.at[h] * (D / 2));
                    const char* sp = vs_head + page_offset(w.page[h], s.vs_pages) + uint32_t(w.at[h] * 4);
                    tile.vb[h] = *reinterpret_cast<const uint32_t*>(sp + vb_off);
#pragma unroll
                    for (int i = 0; i < T::NL; ++i) load_words(tile.v[h][i], vp + 256 * i, v_off);
                }
            }
        };

        // Queries: column `col`, 8 channels per step.
        u32x4_t q[KS];
        {
            const int head = kvh * s.group + qb * 16 + (col < rows ? col : 0);
            const uint16_t* src = s.a.q + b * s.a.q_row + head * s.a.q_head;
#pragma unroll
            for (int i = 0; i < KS; ++i) q[i] = load16(src + T::q_channel(i, quad));
        }
        // This wave's tiles: t, t + 128, ...
        int t = t_begin + 32 * wave;
        T tile[BITS == 4 ? 2 : 1];
        Where now{}, next{};
        if (t < t_end) {
            now = locate(t);
            next = locate(t + kUnit);
            load_k(tile[0], now);
            load_v(tile[0], now);
        }

#pragma unroll
        for (int i = 0; i < KS; ++i)
            if (col >= rows) q[i] = u32x4_t{0, 0, 0, 0};
        float qpick = 0.0f;      // 4 bits: the sum of the column's channels of group `quad`
        if constexpr (BITS == 4) {
#pragma unroll
            for (int g = 0; g < NB; ++g) {
                float x = 0.0f;
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int w = 0; w < 4; ++w)
                        x += half_to_f32<DT>(uint16_t(q[2 * g + e][w])) + half_to_f32<DT>(uint16_t(q[2 * g + e][w] >> 16));
                x = sum_across16(sum_across32(x));
                if (quad == g) qpick = x;
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

        // One tile; the next one's bytes travel meanwhile: 4-bit tiles into
        // registers of their own, 16-bit ones, four times as large, into what the
        // keys, and then the values, of this one have left.  They are read behind
        // the end too (rows of page 0, where a tile has no page): were they not
        // always in flight, every wait would have to be for all of them.
        auto step = [&](T& tile, T& ahead) {
            const bool poison[2] = {now.bad[0], now.bad[1]};
            const bool ragged = t + 32 > t_end;      // only where the sequence ends: units are whole tiles
            now = next;
            if constexpr (BITS == 4) {
                load_k(ahead, now);
                load_v(ahead, now);
            }
            next = locate(t + 2 * kUnit);
            __builtin_amdgcn_sched_barrier(0);      // the loads are issued here, not where registers are spare
            // S^T
            f32x4_t sc[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if constexpr (BITS == 16) {
                    sc[h] = f32x4_t{0, 0, 0, 0};
#pragma unroll
                    for (int i = 0; i < KS; ++i) sc[h] = mfma_16x16x32<DT>(tile.k[h][i], q[i], sc[h]);
                } else {
                    // The products below count 16 + c: (m - 16 s) sum q first.
                    const float low = __builtin_fmaf(f16_to_f32(uint16_t(tile.ka[h])), -16.0f,
                                                     f16_to_f32(uint16_t(tile.ka[h] >> 16)));
                    sc[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(NB == 4 || quad < NB ? low : 0.0f, qpick,
                                                                 f32x4_t{0, 0, 0, 0}, 0, 0, 0);
                    const float ks = f16_to_f32(uint16_t(tile.kb[h]));
                    static_for<NB>([&](auto gc) {
                        constexpr int g = gc.value;
                        f32x4_t acc = {0, 0, 0, 0};
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            acc = mfma_16x16x32<DT>(key_codes(tile.k[h][(2 * g + e) / T::WL][(2 * g + e) % T::WL]),
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
            if constexpr (BITS == 16) {
                load_k(tile, now);
                __builtin_amdgcn_sched_barrier(0);
            }
            // Softmax
            float top = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                              fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
            top = max_across32(max_across16(top));
            if constexpr (BITS == 4) {
                if (ragged) {   // scales behind the end may be anything, and are not the sequence's
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (t + 16 * h + 4 * quad + (col / NB) % 4 >= t_end) tile.vb[h] = 0;
                }
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
            const float base = m == -__builtin_inff() ? 0.0f : m;
            float shift = base * s.a.c - boost;
            if (__ballot(fabsf(base) * s.a.c > kFarScore)) {
                shift = -boost;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc[h][i] -= base;
            }
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
                // Tokens of an operand in the order 0 2 1 3 of each four.  The four
                // of group l % 16 lie NB lanes apart in vb.
                u32x4_t pk, am;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    pk[2 * h] = pack2<PT>(p[h][0], p[h][2]);
                    pk[2 * h + 1] = pack2<PT>(p[h][1], p[h][3]);
                    am[2 * h] = group_middle(tile.vb[h], lane_ahead<2 * NB>(tile.vb[h]));
                    am[2 * h + 1] = group_middle(lane_ahead<NB>(tile.vb[h]), lane_ahead<3 * NB>(tile.vb[h]));
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
                        o[g][2 * j] = mfma_16x16x32<PT>(u32x4_t{value_codes(x0 << 4), value_codes(x0 >> 4),
                                                                value_codes(x1 << 4), value_codes(x1 >> 4)},
                                                        ps, o[g][2 * j]);
                        o[g][2 * j + 1] = mfma_16x16x32<PT>(u32x4_t{value_codes(x0), value_codes(x0 >> 8),
                                                                    value_codes(x1), value_codes(x1 >> 8)},
                                                            ps, o[g][2 * j + 1]);
                    }
                });
            }
            if constexpr (BITS == 16) load_v(tile, now);
            t += kUnit;
        };
        if constexpr (BITS == 4) {
            while (t < t_end) {
                step(tile[0], tile[1]);
                if (t < t_end) step(tile[1], tile[0]);
            }
        } else {
            while (t < t_end) step(tile[0], tile[0]);
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

        // (Hidden from the compiler, which would keep the addresses made of them in
        // registers over the whole loop.)
        int oc = col, oq = quad;
        asm volatile("" : "+v"(oc), "+v"(oq));
        // Join the waves that had tokens.
        const bool several = t_end - t_begin > 32;
        if (several) {
            if (oq == 0) {
                sm[wave][oc] = m;
                sl[wave][oc] = l;
            }
            __syncthreads();
            float top = sm[0][oc];
#pragma unroll
            for (int w = 1; w < 4; ++w) top = fmaxf(top, sm[w][oc]);
            l = 0.0f;
            float mine = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = sm[w][oc] == -__builtin_inff() ? 0.0f : exp2_hw((sm[w][oc] - top) * s.a.c);
                // A wave whose maximum is -infinity has no part but NaN.
                l += sm[w][oc] == -__builtin_inff() ? sl[w][oc] : f * sl[w][oc];
                if (w == wave) mine = sm[w][oc] == -__builtin_inff() ? 1.0f : f;
            }
            m = top;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < E; ++e) o[nb][e] *= mine;
            auto put = [&](int slot) {
                if (oc < rows)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int e = 0; e < E; e += 4)
                                *reinterpret_cast<f32x4_t*>(&so[slot][oc][T::out_channel(nb, 4 * oq + i) + e]) =
                                    f32x4_t{o[nb][e][i], o[nb][e + 1][i], o[nb][e + 2][i], o[nb][e + 3][i]};
            };
            auto add = [&](int slot) {
                if (oc < rows)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int e = 0; e < E; e += 4) {
                                const f32x4_t x = *reinterpret_cast<const f32x4_t*>(
                                    &so[slot][oc][T::out_channel(nb, 4 * oq + i) + e]);
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
        if (wave == 0 && oc < rows) {
            if (whole) {
                const int head = kvh * s.group + qb * 16 + oc;
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
                            *reinterpret_cast<u32x2_t*>(out + T::out_channel(nb, 4 * oq + i) + e) =
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
                            *reinterpret_cast<f32x4_t*>(dst + oc * D + T::out_channel(nb, 4 * oq + i) + e) =
                                f32x4_t{o[nb][e][i], o[nb][e + 1][i], o[nb][e + 2][i], o[nb][e + 3][i]};
                if (oq == 0) {
                    dst[most * D + oc] = m;
                    dst[most * D + most + oc] = l;
                }
            }
        }
        if (unit - first >= units * s.vheads) {
            first = unit;
            ++b;
        }
    }
}

// Joins the parts of (sequence, key-value head) pairs that lie in several runs.
// An item is one of a pair's query heads and 64 channels: up to 32 parts are
// one wave's work, more a workgroup's, a quarter of them a wave.  A wave reads 4
// parts at once, 16 bytes a lane, the first 32 before it knows their weights.
// Parts are added in a fixed order.
constexpr int kJoinChannels = 64;
constexpr int kJoinAlone = 32;

struct Joined { f32x4_t o; float m, l; };    // 4 channels of the sum in each lane of 16; maximum and total in all

// Parts i0 .. i1 (at least one) of an item; ml(i) -> its maximum and total, sums(i) -> its channels.
template <typename ML, typename Sums>
__device__ __forceinline__ Joined join_parts(int i0, int i1, float c, ML&& ml, Sums&& sums) {
    const int lane = threadIdx.x & 63, quad = lane >> 4;
    Joined r{{0, 0, 0, 0}, -__builtin_inff(), 0.0f};
    for (int at = i0; at < i1; at += 64) {
        const int n = min(64, i1 - at);
        f32x4_t x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = sums(at + min(4 * j + quad, n - 1));
        float m = -__builtin_inff(), l = 0.0f;
        if (lane < n) ml(at + lane, m, l);
        float top = m;
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) top = fmaxf(top, __shfl_xor(top, off));
        top = fmaxf(r.m, max_across32(max_across16(top)));
        // A part whose maximum is -infinity has nothing, or NaN.
        const float w = lane >= n ? 0.0f : m == -__builtin_inff() ? 1.0f : exp2_hw((m - top) * c);
        const float down = r.m == -__builtin_inff() ? 1.0f : exp2_hw((r.m - top) * c);
        r.m = top;
        r.l = __builtin_fmaf(r.l, down, lane < n ? w * l : 0.0f);
        r.o *= down;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float f = __shfl(w, 4 * j + quad);
            if (4 * j + quad < n) r.o += f * x[j];
        }
        for (int j = 8; 4 * j < n; ++j) {
            const float f = __shfl(w, 4 * j + quad);
            if (4 * j + quad < n) r.o += f * sums(at + 4 * j + quad);
        }
    }
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) r.l += __shfl_xor(r.l, off);
    r.l = sum_across32(sum_across16(r.l));
#pragma unroll
    for (int j = 0; j < 4; ++j) r.o[j] = sum_across32(sum_across16(r.o[j]));
    return r;
}

template <int DT, int D>
__global__ __launch_bounds__(256) void attention_paged_join_kernel(const Split s) {
    constexpr int SLICES = D / kJoinChannels;
    __shared__ float sm[4], sl[4];
    __shared__ __attribute__((aligned(16))) float so[4][kJoinChannels];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int vh = int(blockIdx.x) % s.vheads, b = int(blockIdx.x) / s.vheads;
    const int kvh = vh / s.qblocks, qb = vh - kvh * s.qblocks;
    // First unit of the pair.
    int before = 0, all = 0;
    for (int b0 = 0; b0 < s.a.batch; b0 += 64) {
        const int u = b0 + lane < s.a.batch ? units_of(s.a.lens[b0 + lane], s.cap) : 0, sum = prefix_sum(u);
        if (b >= b0 && b < b0 + 64) before = all + __builtin_amdgcn_readlane(sum - u, b - b0);
        all += __builtin_amdgcn_readlane(sum, 63);
    }
    const int len = scalar_load(s.a.lens + b);
    const int units = units_of(len, s.cap);
    const int per = units_per_group(s, all * s.vheads);
    const int begin = before * s.vheads + vh * units, end = begin + units;
    const int w0 = (begin + kBegin) / per, w1 = (end - 1) / per;
    if (w0 == w1) return;
    const int n = w1 - w0 + 1, most = min(16, s.group), items = min(16, s.group - 16 * qb) * SLICES;
    auto source = [&](int i) { return part<D>(s, 2 * (w0 + i) + (i == 0 ? 1 : 0)); };
    auto parts = [&](int item, int i0, int i1) {
        const int row = item / SLICES, ch = item % SLICES * kJoinChannels + 4 * (lane & 15);
        return join_parts(i0, i1, s.a.c,
                          [&](int i, float& m, float& l) {
                              m = source(i)[most * D + row];
                              l = source(i)[most * D + most + row];
                          },
                          [&](int i) { return *reinterpret_cast<const f32x4_t*>(source(i) + row * D + ch); });
    };
    auto store = [&](int item, f32x4_t o, float l) {
        const int row = item / SLICES, ch = item % SLICES * kJoinChannels + 4 * (lane & 15);
        const float inv = 1.0f / l;
        const int head = kvh * s.group + qb * 16 + row;
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = len > s.cap ? __builtin_nanf("") : o[j] * inv;
        if (lane < 16)
            *reinterpret_cast<u32x2_t*>(s.a.out + (int64_t(b) * s.a.heads + head) * D + ch) =
                u32x2_t{pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3])};
    };
    if (n <= kJoinAlone) {
        for (int item = 4 * int(blockIdx.y) + wave; item < items; item += 4 * int(gridDim.y)) {
            const Joined r = parts(item, 0, n);
            store(item, r.o, r.l);
        }
        return;
    }
    for (int item = blockIdx.y; item < items; item += gridDim.y) {
        const int share = (n + 3) / 4, i0 = wave * share;      // n > 32: every wave has some
        const Joined r = parts(item, i0, min(n, i0 + share));
        if (lane == 0) {
            sm[wave] = r.m;
            sl[wave] = r.l;
        }
        if (lane < 16) *reinterpret_cast<f32x4_t*>(&so[wave][4 * lane]) = r.o;
        __syncthreads();
        if (wave == 0) {
            const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
            f32x4_t o = {0, 0, 0, 0};
            float l = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = sm[w] == -__builtin_inff() ? 1.0f : exp2_hw((sm[w] - top) * s.a.c);
                l = __builtin_fmaf(f, sl[w], l);
                o += f * *reinterpret_cast<const f32x4_t*>(&so[w][4 * (lane & 15)]);
            }
            store(item, o, l);
        }
        __syncthreads();      // sm, sl and so are the next item's
    }
}

// Workgroups of a grid that has work for all of them, 2 to 4 a CU.  By the registers
// of its kernel a CU runs 4 at once at head_dim 64, 3 at 128, and at 256 2 in 4 bits
// and 1 in 16.  16 bits take 2 a CU at 128 and at 256, where half of them run at
// first; large calls take half of the grid (units_per_group).
int resident(int head_dim, int bits) {
    const int per_cu = head_dim == 64 ? 4 : head_dim == 128 ? (bits == 4 ? 3 : 2) : 2;
    return 256 * per_cu;
}

// Workgroups of the grid: those, or as many as there can be units.
int grid_of(int64_t batch, int64_t vheads, int64_t table_tokens, int head_dim, int bits) {
    const int64_t per = kBegin + (table_tokens > kUnit ? (table_tokens + kUnit - 1) / kUnit : 1);
    const int64_t units = batch * vheads * per;
    const int most = resident(head_dim, bits);
    return units < most ? static_cast<int>(units) : most;
}

template <int DT, int D, int BITS>
int launch(const Split& s, hipStream_t stream) {
    hipLaunchKernelGGL((attention_paged_kernel<DT, D, BITS>), dim3(s.grid), dim3(256), 0, stream, s);
    int rc = check_launch("attention_paged");
    if (rc != NANOVLLM_GEMM_OK || s.cap <= kUnit) return rc;   // every pair has one unit of tokens: nothing to join
    // Few pairs: a workgroup for each item; many: for four.
    const int64_t pairs = int64_t(s.a.batch) * s.vheads, items = (s.group < 16 ? s.group : 16) * (D / kJoinChannels);
    const int64_t each = pairs >= 64 ? (items + 3) / 4 : items;
    const dim3 grid(static_cast<uint32_t>(pairs), static_cast<uint32_t>(each));
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
                                  int64_t table_tokens, int bits) {
    if (table_tokens <= kUnit) return 0;
    const int64_t group = heads / kv_heads, vheads = kv_heads * ((group + 15) / 16);
    return int64_t(2) * grid_of(batch, vheads, table_tokens, static_cast<int>(head_dim), bits) *
           (group < 16 ? group : 16) * (head_dim + 4) * 4;
}

int launch_attention_paged(const PagedArgs& p, int head_dim, int bits, int dtype, hipStream_t stream) {
    Split s;
    s.a = p;
    s.cap = p.table_blocks * p.cache.block_size;
    s.group = p.heads / p.cache.kv_heads;
    s.qblocks = (s.group + 15) / 16;
    s.vheads = p.cache.kv_heads * s.qblocks;
    s.grid = grid_of(p.batch, s.vheads, s.cap, head_dim, bits);
    s.many = bits == 16 && s.grid == resident(head_dim, bits) ? 2 * s.grid : INT32_MAX;
    s.k_pages = static_cast<uint32_t>(p.cache.k_stride / 16);
    s.v_pages = static_cast<uint32_t>(p.cache.v_stride / 16);
    s.ks_pages = static_cast<uint32_t>(p.cache.ks_stride / 16);
    s.vs_pages = static_cast<uint32_t>(p.cache.vs_stride / 16);
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
