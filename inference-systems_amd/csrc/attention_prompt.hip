// Attention of packed prompts: causal, grouped heads, sequences of different
// lengths.
//
// A workgroup takes 128 queries of one head of one sequence, 32 a wave, and
// walks over the keys in tiles of 64 that all waves share in LDS:
//   S^T[key, query] = K Q^T      32 x 32 x 16 products; accumulator v of lane l
//                                is key 8 (v / 4) + 4 (l / 32) + v % 4, query l % 32
//   P = 2^(c S - c max)          online softmax: a query's scores lie in two
//                                lanes, so its maximum and sum are lane values
//   O^T[channel, query] += V^T P with the keys of a product in the order in which
//                                the accumulators of S^T hold them: P never moves
// P is rounded to the operands' type, as the matrix cores take it, and its total is
// that of the rounded P: against 64 bits the output is 0.0020 off in bf16, 0.0015
// with P in fp32, and 0.00024 for 0.00019 in fp16; a second product for what the
// rounding leaves would cost as much as the first.
// V^T is read from LDS transposed (ds_read_b64_tr_b16), 4 keys of a channel at
// a time, which is the run of keys a lane's accumulators hold.
//
// Many blocks, and the short ones of one sequence, have a workgroup each.  The
// others (see in_runs: of several sequences the host knows only the sum of keys, so
// short ones are among them) are split over a fixed grid: all (sequence, head, 128
// queries) blocks in units of one tile of keys, laid end to end, each workgroup an
// equal run of units; a block starts with six units that hold no key and stand for
// what it costs to begin one.  So a causal prompt's long rows and short ones, a few
// queries against many keys, and sequences of any lengths load the chip evenly.  A
// block whose keys lie in one run is finished there; the parts of others go to a
// workspace (at most two per workgroup) and a second kernel joins them.
//
// Bound by the matrix cores, which run at the chip's power limit: on MI355X 16384
// tokens of 8 heads of 256 take 1121-1150 us, 960-980 TFLOP/s (a large library
// product 1265; the products alone 807 us); a chunk of 512 behind 8188 cached
// tokens, 32 heads of 128, 85-89 us, 12 of them in the join; 2048 tokens of 8
// heads of 256 48 us, 18 of them for the traffic of 35 MB of parts.
#include <type_traits>

#include "attention_common.hpp"

namespace nvg {
namespace {

constexpr int kRows = 128;      // queries of a block
constexpr int kKeys = 64;       // keys of a tile
constexpr int kBegin = 6;       // units a block costs before its first tile, and by its masked ones (2, 4, 6:
                                // 43.0, 42.1, 40.6 us for 2048 tokens, 79 -> 77 for a chunk of 512)

// Sums are rescaled when a maximum grows by more than 2^kLazy, and P is held
// 2^kBoost fold, which cancels in O / l; together they fit the type.  Without the
// factor float16 loses weights below 2^-25 next to 1, which count where there are
// many: 131072 keys 2^-25.4 below another one came out 2.4e-3 off, with it 4.7e-4
// (half a step of the output: 4.9e-4).  By (kLazy, kBoost), float16: 16384 tokens
// of 8 heads of 256 (8, 0) 1181 us, (8, 7) 1181, (3, 12) 1184, (0, 15) 1238; 24
// ragged prompts 117, 118, 118, 123.
template <int DT> constexpr float kLazy = DT == NANOVLLM_GEMM_F16 ? 3.0f : 8.0f;
template <int DT> constexpr float kBoost = DT == NANOVLLM_GEMM_F16 ? 12.0f : 0.0f;

struct Split {
    PromptArgs a;
    float* partial;
    int32_t grid;
    int32_t runs;      // equal runs of units; else a block per workgroup
};

// One sequence: its rows, and the tiles of keys of its blocks.
struct Sequence {
    int q0, lq, k0, lk;
    int blocks;     // of 128 queries
    int ahead;      // causal: keys of the first block's tiles before its rows, in tiles rounded up
    int causal;

    // Tiles of keys of block i.
    __device__ __forceinline__ int tiles(int i) const {
        if (!causal || i == blocks - 1) return (lk + kKeys - 1) / kKeys;
        return max(0, (kRows / kKeys) * (i + 1) + ahead);
    }
    // Units of the blocks before i < blocks, and of all.  A block has one unit
    // of keys at least, since one that sees no key has its rows written too.
    __device__ __forceinline__ int64_t before(int i) const {
        static_assert(kRows == 2 * kKeys, "the sum below is of 2 (j + 1) + ahead");
        int64_t sum = int64_t(kBegin) * i;
        if (!causal) return sum + int64_t(max(1, (lk + kKeys - 1) / kKeys)) * i;
        const int from = max(0, (1 - ahead + 1) / 2 - 1);      // blocks below see one unit
        if (i <= from) return sum + i;
        return sum + from + int64_t(i - from) * ahead + int64_t(i) * (i + 1) - int64_t(from) * (from + 1);
    }
    __device__ __forceinline__ int64_t units() const {
        return blocks == 0 ? 0 : before(blocks - 1) + kBegin + max(1, tiles(blocks - 1));
    }
};

// Sequence b of the call, or, behind the last one, the rows that belong to none
// (they see no key).  Offsets are taken within the operands whatever they hold.
__device__ __forceinline__ Sequence sequence(const PromptArgs& p, int b) {
    auto at = [](const int32_t* cu, int i, int rows) { return min(max(cu[i], 0), rows); };
    Sequence s;
    s.q0 = at(p.cu_q, b, p.q_rows);
    const int q1 = b < p.batch ? at(p.cu_q, b + 1, p.q_rows) : p.q_rows;
    s.k0 = b < p.batch ? at(p.cu_k, b, p.k_rows) : 0;
    const int k1 = b < p.batch ? at(p.cu_k, b + 1, p.k_rows) : 0;
    s.lq = max(0, q1 - s.q0);
    s.lk = max(0, k1 - s.k0);
    s.blocks = (s.lq + kRows - 1) / kRows;
    const int more = s.lk - s.lq;
    s.ahead = more > 0 ? (more + kKeys - 1) / kKeys : -(-more / kKeys);
    s.causal = p.causal;
    return s;
}

// The sequence that lane `lane` holds, in all lanes.
__device__ __forceinline__ Sequence from_lane(const Sequence& s, int lane) {
    auto at = [&](int x) { return __builtin_amdgcn_readlane(x, lane); };
    return Sequence{at(s.q0), at(s.lq), at(s.k0), at(s.lk), at(s.blocks), at(s.ahead), s.causal};
}

__device__ __forceinline__ int64_t uniform64(int64_t x, int lane) {
    return int64_t(uint32_t(__builtin_amdgcn_readlane(int(x), lane))) |
           int64_t(__builtin_amdgcn_readlane(int(x >> 32), lane)) << 32;
}

// Units of 64 sequences from b0 on, and the sum up to each: a lane a sequence.
struct Units { Sequence s; int64_t mine, sum; };

__device__ __forceinline__ Units units_from(const PromptArgs& p, int b0) {
    const int lane = threadIdx.x & 63;
    Units u;
    u.s = sequence(p, min(b0 + lane, p.batch));
    u.mine = b0 + lane <= p.batch ? u.s.units() : 0;
    u.sum = u.mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int64_t up = __shfl_up(u.sum, off);
        if (lane >= off) u.sum += up;
    }
    return u;
}

// A block, and its first unit.
struct Block {
    Sequence s;
    int b, head, index;
    int64_t first;
};

// Units of all sequences and heads; `u`: of the last 64 sequences.
__device__ __forceinline__ int64_t all_units(const PromptArgs& p, Units& u) {
    int64_t total = 0;
    for (int b0 = 0; b0 <= p.batch; b0 += 64) {
        u = units_from(p, b0);
        total += uniform64(u.sum, 63);
    }
    return total * p.heads;
}

// The block that holds a unit below the total.
__device__ __forceinline__ Block find_block(const PromptArgs& p, Units u, int64_t unit) {
    const int lane = threadIdx.x & 63;
    int64_t base = 0;
    Block r{};
    for (int b0 = 0; b0 <= p.batch; b0 += 64) {
        if (p.batch >= 64) u = units_from(p, b0);      // else all_units has left them
        const uint64_t past = __ballot((base + u.sum) * p.heads > unit);
        if (past) {
            const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
            r.b = b0 + at;
            r.first = (base + uniform64(u.sum - u.mine, at)) * p.heads;
            r.s = from_lane(u.s, at);
            break;
        }
        base += uniform64(u.sum, 63);
    }
    const int64_t each = r.s.units();
    r.head = int((unit - r.first) / each);
    r.first += r.head * each;
    // The last block that starts at or before the unit: 64 candidates at a time.
    int lo = 0, n = r.s.blocks;
    while (n > 1) {
        const int step = (n + 63) / 64, i = lane * step;
        const uint64_t before = __ballot(i < n && r.first + r.s.before(lo + i) <= unit);
        const int at = (__popcll(static_cast<unsigned long long>(before)) - 1) * step;
        lo += at;
        n = min(step, n - at);
    }
    r.index = lo;
    r.first += r.s.before(r.index);
    return r;
}

// Block `index` of all sequences' (of one head), the last of a sequence first,
// since it sees the most keys; false behind the last block.
__device__ __forceinline__ bool nth_block(const PromptArgs& p, int index, Block& r) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int b0 = 0; b0 <= p.batch; b0 += 64) {
        const Sequence s = sequence(p, min(b0 + lane, p.batch));
        const int n = b0 + lane <= p.batch ? s.blocks : 0, sum = prefix_sum(n);
        const uint64_t past = __ballot(base + sum > index);
        if (past) {
            const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
            r.b = b0 + at;
            r.s = from_lane(s, at);
            r.index = r.s.blocks - 1 - (index - base - __builtin_amdgcn_readlane(sum - n, at));
            r.first = 0;
            return true;
        }
        base += __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

// The next block in order.
__device__ __forceinline__ void advance(const PromptArgs& p, Block& r) {
    r.first += kBegin + max(1, r.s.tiles(r.index));
    if (++r.index < r.s.blocks) return;
    r.index = 0;
    if (++r.head < p.heads) return;
    r.head = 0;
    do r.s = sequence(p, ++r.b);
    while (r.s.blocks == 0 && r.b < p.batch);
}

// The part of a block a workgroup leaves: fp32 sums as the waves' lanes hold
// them, 16 bytes a lane, then the rows' maxima and totals of P.
template <int D>
__device__ __forceinline__ float* part(const Split& s, int slot) {
    return s.partial + int64_t(slot) * kRows * (D + 2);
}

// Place of 16-byte chunk `chunk` of row `row` in a tile: chunks are exchanged
// within a row so that the 64 LDS banks are evenly used by what one read
// instruction takes: of keys the same chunk of 16 rows, of values 64 bytes of
// 4 rows.
template <int D>
__device__ __forceinline__ int k_chunk(int row, int chunk) {
    if constexpr (D == 64) return chunk ^ ((row >> 1) & 7);
    else return chunk ^ (row & 15);
}
template <int D>
__device__ __forceinline__ int v_chunk(int row, int chunk) {
    if constexpr (D == 64) return chunk ^ (((row >> 1) & 1) << 2);
    else return chunk ^ ((row & 3) << 2);
}

template <int DT>
__device__ __forceinline__ bool finite1(uint32_t x) {
    constexpr uint32_t e = DT == NANOVLLM_GEMM_BF16 ? 0x7f80u : 0x7c00u;
    return (x & e) != e;
}

// a . b + c over two 16-bit elements.
template <int DT>
__device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c) {
    if constexpr (DT == NANOVLLM_GEMM_BF16)
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, a), __builtin_bit_cast(bf16x2_t, b), c, false);
    else
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, a), __builtin_bit_cast(f16x2_t, b), c, false);
}

// Values of a masked tile that hold an infinity or a NaN.  A product would carry
// it into rows that do not attend to its key (0 x infinity), so such elements
// are 0 in the products and added here, slowly, after all tiles, to the sums in
// LDS: for every key a row attends to, P times the elements that are not finite.
// Finite values never come here.  `sums`: the lane's row, of which it has the
// channels 8 i + 4 half + 0..3.
template <int DT, int D>
__device__ __forceinline__ void add_keys(const PromptArgs& p, const uint16_t* qrow, const uint16_t* kbase,
                                         const uint16_t* vbase, int key0, int key1, int last, int half, float base,
                                         float* sums) {
    for (int j = key0; j < key1; ++j) {
        const uint16_t* vrow = vbase + int64_t(j) * p.v_row;
        const uint16_t* krow = kbase + int64_t(j) * p.k_row;
        bool finite = true;
        for (int ch = 0; ch < D; ch += 2) {
            const uint32_t x = *reinterpret_cast<const uint32_t*>(vrow + ch);
            finite = finite && finite1<DT>(x) && finite1<DT>(x >> 16);
        }
        if (finite || j > last) continue;
        float s = 0.0f;
        for (int ch = 0; ch < D; ch += 8) {
            const u32x4_t a = load16(qrow + ch), b = load16(krow + ch);
#pragma unroll
            for (int w = 0; w < 4; ++w) s = dot2<DT>(a[w], b[w], s);
        }
        const float pj = exp2_hw(__builtin_fmaf(s - base, p.c, kBoost<DT>));
        for (int ch = 4 * half; ch < D; ch += 8)
            for (int i = ch; i < ch + 4; ++i)
                if (!finite1<DT>(vrow[i])) sums[i] = __builtin_fmaf(pj, half_to_f32<DT>(vrow[i]), sums[i]);
    }
}

template <int DT, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attention_prompt_kernel(const Split s) {
    constexpr int CH = D / 8;                  // 16-byte chunks of a row
    constexpr int KS = D / 16;                 // steps of the contraction over channels
    constexpr int DTILES = D / 32, NB = kKeys / 32;
    constexpr int LOADS = kKeys * CH / 256;    // 16-byte copies per thread and tile of K, or of V
    constexpr uint32_t PITCH = CH * 16, TILE = kKeys * PITCH;      // bytes of a row and of a tile in LDS
    typedef short v4i16_t __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) v4i16_t* lds_v4;
    typedef const __attribute__((address_space(3))) u32x4_t* lds_u4;
    // Two stages of keys and of values: as many bytes as the block's sums, which
    // take their place where add_keys runs.
    __shared__ __attribute__((aligned(1024))) u32x4_t tiles_lds[4][kKeys * CH];
    static_assert(sizeof(tiles_lds) == kRows * D * sizeof(float), "the sums fill the tiles");
    u32x4_t (*kt)[kKeys * CH] = tiles_lds, (*vt)[kKeys * CH] = tiles_lds + 2;

    const PromptArgs& p = s.a;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int group = p.heads / p.kv_heads;
    int wg = blockIdx.x;
    int64_t unit = 0, end;
    Block blk{};
    if (s.runs) {
        wg = xcd_remap(wg, s.grid);      // neighbouring runs share keys: they go to one XCD
        Units u;
        const int64_t total = all_units(p, u), per = (total + s.grid - 1) / s.grid;
        unit = wg * per;
        end = unit + per < total ? unit + per : total;
        if (unit >= end) return;
        blk = find_block(p, u, unit);
    } else {
        if (!nth_block(p, wg / p.heads, blk)) return;
        blk.head = wg % p.heads;
        end = kBegin + max(1, blk.s.tiles(blk.index));
    }

    // LDS addresses of a lane's reads, of stage 0.  Chunk exchanges are exclusive
    // ors, so what step i of a read adds to them is one too.
    // K: row l % 32, chunk 2 i + l / 32.  V^T: lane j of 16 points at key j / 4 and
    // channels 4 (j % 4) of its 16-channel half; keys of a read differ from one
    // another in their two lowest bits only, which give the exchange.
    const int vr = 4 * half + ((lane & 15) >> 2);
    const int vc = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    const uint32_t k_read = lds_address(kt[0]) + col * PITCH + 16 * k_chunk<D>(col, half);
    const uint32_t v_read = lds_address(vt[0]) + vr * PITCH + 16 * v_chunk<D>(vr, vc) + 8 * (lane & 1);

    // A tile is copied by instructions that fill 64 neighbouring chunks of LDS,
    // 64 / CH rows, each lane from the chunk that belongs there; the next
    // instruction of a wave is STEP rows on.  A lane's offsets from the first row:
    // the exchange of K's chunks may change from one instruction to the next.
    constexpr int STEP = 4 * 64 / CH;
    const int r0 = wave * (64 / CH) + lane / CH, c0 = lane % CH;
    const uint32_t k_bytes = uint32_t(p.k_row) * 2, v_bytes = uint32_t(p.v_row) * 2;
    const uint32_t k_off[2] = {r0 * k_bytes + 16 * k_chunk<D>(r0, c0), r0 * k_bytes + 16 * k_chunk<D>(r0 + STEP, c0)};
    const uint32_t v_each = r0 * v_bytes + 16 * v_chunk<D>(r0, c0), v_off[2] = {v_each, v_each};

    for (;; advance(p, blk)) {
        const int all_tiles = blk.s.tiles(blk.index), units = kBegin + max(1, all_tiles);
        const int from = int(unit - blk.first), to = int(end - blk.first < units ? end - blk.first : units);
        unit += to - from;
        if (to <= kBegin) break;      // the run ends before the block's first tile
        const int t0 = max(0, from - kBegin), t1 = min(all_tiles, to - kBegin);
        const bool whole = t0 == 0 && to == units;

        const int lq = blk.s.lq, lk = blk.s.lk, head = blk.head, kvh = head / group;
        const int row0 = blk.index * kRows, row = row0 + 32 * wave + col;      // row: this lane's query
        const int ahead = p.causal ? lk - lq : lk;
        // Keys a row attends to: 0 .. last.
        const int last = p.causal ? min(row + ahead, lk - 1) : lk - 1;
        // Tiles that every row of the block attends to in full.
        const int full = p.causal ? max(0, min(lk, row0 + ahead + 1)) / kKeys : lk / kKeys;

        const uint16_t* qrow = p.q + int64_t(blk.s.q0 + min(row, lq - 1)) * p.q_row + head * p.q_head;
        const uint16_t* kbase = p.k + int64_t(blk.s.k0) * p.k_row + kvh * p.k_head;
        const uint16_t* vbase = p.v + int64_t(blk.s.k0) * p.v_row + kvh * p.v_head;

        auto copy = [&](const uint16_t* rows, uint32_t bytes, const uint32_t (&off)[2], uint32_t lds, int t) {
            const uint32_t to = lds + (t & 1) * TILE + wave * 1024;
            const char* base = reinterpret_cast<const char*>(rows) + int64_t(t) * kKeys * bytes;
            const int left = lk - t * kKeys;
            if (left >= kKeys) {
#pragma unroll
                for (int i = 0; i < LOADS; ++i) dma16_at(base + i * STEP * bytes, off[i % 2], to + i * 4096);
            } else {
                // Rows behind the end repeat the last one (their scores are masked).
                // Where that lies before an instruction's first row, the base moves.
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const int behind = max(0, i * STEP - (left - 1)), back = max(0, r0 + i * STEP - (left - 1));
                    dma16_at(base + (i * STEP - behind) * bytes, off[i % 2] - (back - behind) * bytes, to + i * 4096);
                }
            }
        };
        auto copy_k = [&](int t) { copy(kbase, k_bytes, k_off, lds_address(kt[0]), t); };
        auto copy_v = [&](int t) { copy(vbase, v_bytes, v_off, lds_address(vt[0]), t); };
        __syncthreads();      // the last block's tiles have been read
        if (t0 < t1) {
            copy_k(t0);
            copy_v(t0);
        }
        u32x4_t q[KS];
#pragma unroll
        for (int i = 0; i < KS; ++i) q[i] = load16(qrow + 16 * i + 8 * half);

        f32x16_t o[DTILES];
#pragma unroll
        for (int i = 0; i < DTILES; ++i) o[i] = f32x16_t{};
        float m = -__builtin_inff(), l = 0.0f;
        uint32_t late = 0;      // masked tiles (3 at most) with values that add_keys adds

        // S^T of tile t.  A product occupies the matrix cores for 32 cycles, in which
        // the wave issues other work only if it stands between two products:
        // LDS reads, two steps ahead, and `beside(j)`, j of KS * NB.  The compiler,
        // which would issue one kind of work at a time, is kept to that order.
        auto scores = [&](int t, f32x16_t (&sc)[NB], auto&& beside) {
            const uint32_t k_at = k_read + (t & 1) * TILE;
            u32x4_t kf[3][NB];
            auto read = [&](int i, int n) { kf[i % 3][n] = *(lds_u4)(uintptr_t)((k_at ^ (32 * i)) + 32 * n * PITCH); };
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int n = 0; n < NB; ++n) read(i, n);
#pragma unroll
            for (int n = 0; n < NB; ++n) sc[n] = f32x16_t{};
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    sc[n] = mfma_32x32x16<DT>(kf[i % 3][n], q[i], sc[n]);
                    if (i + 2 < KS) read(i + 2, n);
                    beside(i * NB + n);
                    __builtin_amdgcn_sched_barrier(0);
                }
        };
        // P of two scores, packed, and its sum; `pair` of NB * 8.
        u32x4_t pk[NB][2];
        auto weigh = [&](const f32x16_t (&sc)[NB], int pair, float shift) {
            const int n = pair / 8, w = pair % 8;
            const uint32_t two = pack2<DT>(exp2_hw(__builtin_fmaf(sc[n][2 * w], p.c, -shift)),
                                           exp2_hw(__builtin_fmaf(sc[n][2 * w + 1], p.c, -shift)));
            pk[n][w / 4][w % 4] = two;
            l = dot2<DT>(two, DT == NANOVLLM_GEMM_BF16 ? 0x3f803f80u : 0x3c003c00u, l);
        };

        // The largest of the scores so far: 32 of them in `steps` steps.
        float top = -__builtin_inff();
        auto look = [&](const f32x16_t (&sc)[NB], int step, int steps) {
#pragma unroll
            for (int v = step * NB * 16 / steps; v < (step + 1) * NB * 16 / steps; ++v)
                top = fmaxf(v == 0 ? -__builtin_inff() : top, sc[v / 16][v % 16]);
        };

        // Tile t, whose scores are in sc and the largest in top; those of the next
        // tile are computed while this one's softmax runs, and looked through
        // during its products with the values.
        auto tile = [&](int t, f32x16_t (&sc)[NB], f32x16_t (&ahead_sc)[NB]) {
            const bool masked = t >= full, more = t + 1 < t1;
            wait_vmcnt<0>();      // keys of tile t + 1 and values of t
            __syncthreads();
            if (more) {
                if (t + 2 < t1) copy_k(t + 2);
                copy_v(t + 1);
            }
            if (masked) {
                const int seen = last - t * kKeys - 4 * half;
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int v = 0; v < 16; ++v)
                        if (32 * n + 8 * (v / 4) + v % 4 > seen) sc[n][v] = -__builtin_inff();
                // A look at the tile's values: see add_keys.
                u32x4_t* mine = vt[t & 1] + threadIdx.x;
                bool clean = true;
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const u32x4_t x = mine[i * 256];
#pragma unroll
                    for (int w = 0; w < 4; ++w) clean = clean && finite1<DT>(x[w]) && finite1<DT>(x[w] >> 16);
                }
                if (__syncthreads_or(!clean)) {
                    late |= 1u << (t - full);
                    for (int i = 0; i < LOADS; ++i) {
                        u32x4_t x = mine[i * 256];
#pragma unroll
                        for (int w = 0; w < 4; ++w)
                            x[w] &= (finite1<DT>(x[w]) ? 0xffffu : 0u) | (finite1<DT>(x[w] >> 16) ? 0xffff0000u : 0u);
                        mine[i * 256] = x;
                    }
                    __syncthreads();
                }
                look(sc, 0, 1);
            }
            top = max_across32(top);
            // A first score (m is -infinity), or one that outgrows the range P has been given.
            if (__ballot((top - m) * p.c > kLazy<DT>)) {
                const float higher = fmaxf(m, top);
                const float down = higher == -__builtin_inff() ? 1.0f : exp2_hw((m - higher) * p.c);
                m = higher;
                l *= down;
#pragma unroll
                for (int i = 0; i < DTILES; ++i) o[i] *= down;
            }
            const float base = m == -__builtin_inff() ? 0.0f : m;
            float shift = base * p.c - kBoost<DT>;
            if (__ballot(fabsf(base) * p.c > kFarScore)) {
                shift = -kBoost<DT>;
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int v = 0; v < 16; ++v) sc[n][v] -= base;
            }
            const uint32_t v_at = v_read + (t & 1) * TILE;
            u32x4_t vf[2][DTILES];      // values of 16 keys, and of the next 16
            auto read = [&](int g, int i) {
                const uint32_t at = (v_at ^ (64 * i)) + 16 * g * PITCH;
                const v4i16_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(uintptr_t)at);
                const v4i16_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(uintptr_t)(at + 8 * PITCH));
                const u32x2_t l2 = __builtin_bit_cast(u32x2_t, lo), h2 = __builtin_bit_cast(u32x2_t, hi);
                vf[g % 2][i] = u32x4_t{l2[0], l2[1], h2[0], h2[1]};
            };
            constexpr int STEPS = KS * NB;
            if (more) {
                scores(t + 1, ahead_sc, [&](int j) {
#pragma unroll
                    for (int w = j * NB * 8 / STEPS; w < (j + 1) * NB * 8 / STEPS; ++w) weigh(sc, w, shift);
                    if (j >= STEPS - DTILES) read(0, j - (STEPS - DTILES));
                });
            } else {
                // (Hidden, or the compiler would move what both branches share ahead of them.)
                float alone = shift;
                asm volatile("" : "+v"(alone));
#pragma unroll
                for (int i = 0; i < DTILES; ++i) read(0, i);
#pragma unroll
                for (int w = 0; w < NB * 8; ++w) weigh(sc, w, alone);
            }
#pragma unroll
            for (int g = 0; g < 2 * NB; ++g)
#pragma unroll
                for (int i = 0; i < DTILES; ++i) {
                    o[i] = mfma_32x32x16<DT>(vf[g % 2][i], pk[g / 2][g % 2], o[i]);
                    if (g + 1 < 2 * NB) read(g + 1, i);
                    look(ahead_sc, g * DTILES + i, 2 * NB * DTILES);
                    __builtin_amdgcn_sched_barrier(0);
                }
        };
        f32x16_t sc[2][NB] = {};
        if (t0 < t1) {
            wait_vmcnt<0>();
            __syncthreads();
            if (t0 + 1 < t1) copy_k(t0 + 1);
            scores(t0, sc[0], [](int) {});
            look(sc[0], 0, 1);
        }
        for (int t = t0; t < t1;) {
            tile(t, sc[0], sc[1]);
            if (++t < t1) {
                tile(t, sc[1], sc[0]);
                ++t;
            }
        }

        l = sum_across32(l);
        // (Hidden from the compiler, which would keep addresses made of it in
        // registers over the whole loop.)
        int oc = col;
        asm volatile("" : "+v"(oc));
        const int mine = 32 * wave + oc;      // this lane's row of the block
        const float inv = last < 0 ? 0.0f : 1.0f / l;     // no key: 0
        uint16_t* out = p.out + (int64_t(blk.s.q0 + row0 + mine) * p.heads + head) * D;
        float* slot = part<D>(s, 2 * wg + (t0 == 0 ? 1 : 0));
        const uint32_t slot_at = 4 * (64 * DTILES * 4 * wave + oc + 32 * half);
        auto store = [&](int ch, f32x4_t x) {      // channels ch .. ch + 3
            if (!whole)
                *reinterpret_cast<f32x4_t*>(slot + slot_at + 256 * (ch / 8)) = x;
            else if (row < lq)
                *reinterpret_cast<u32x2_t*>(out + ch) =
                    u32x2_t{pack2<DT>(x[0] * inv, x[1] * inv), pack2<DT>(x[2] * inv, x[3] * inv)};
        };
        if (!whole && half == 0) {
            slot[kRows * D + mine] = m;
            slot[kRows * D + kRows + mine] = l;
        }
        if (!late) {
#pragma unroll
            for (int i = 0; i < DTILES; ++i)
#pragma unroll
                for (int v = 0; v < 16; v += 4)
                    store(32 * i + 2 * v + 4 * half, f32x4_t{o[i][v], o[i][v + 1], o[i][v + 2], o[i][v + 3]});
        } else {
            __syncthreads();      // the tiles have been read
            float* sums = reinterpret_cast<float*>(tiles_lds) + mine * D;
#pragma unroll
            for (int i = 0; i < DTILES; ++i)
#pragma unroll
                for (int v = 0; v < 16; v += 4)
                    *reinterpret_cast<f32x4_t*>(sums + 32 * i + 2 * v + 4 * half) =
                        f32x4_t{o[i][v], o[i][v + 1], o[i][v + 2], o[i][v + 3]};
            const float base = m == -__builtin_inff() ? 0.0f : m;
            for (int t = full; t < t1; ++t)
                if (late >> (t - full) & 1)
                    add_keys<DT, D>(p, qrow, kbase, vbase, t * kKeys, min(lk, t * kKeys + kKeys), last, half, base, sums);
            for (int ch = 4 * half; ch < D; ch += 8) store(ch, *reinterpret_cast<const f32x4_t*>(sums + ch));
        }
        if (unit >= end) break;
    }
}

// Joins the parts of the block that the start of run blockIdx.x + 1 cuts first:
// a wave takes 32 rows and kJoin channels as the kernel's waves left them.  Parts
// are added in order.
constexpr int kJoin = 64;

template <int DT, int D>
__global__ __launch_bounds__(256) void attention_prompt_join_kernel(const Split s) {
    const PromptArgs& p = s.a;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), half = lane >> 5;
    const int wg = int(blockIdx.x) + 1;
    Units u;
    const int64_t total = all_units(p, u), per = (total + s.grid - 1) / s.grid, unit = wg * per;
    if (unit >= total) return;
    const Block blk = find_block(p, u, unit);
    const int64_t keys = blk.first + kBegin;      // the block's first unit with a key
    const int64_t behind = keys + max(1, blk.s.tiles(blk.index));
    if (unit <= keys || keys / per != wg - 1) return;
    const int first = wg - 1, last_wg = int((behind - 1) / per);
    const int mine = 32 * wave + (lane & 31), row = blk.index * kRows + mine;
    const int ahead = p.causal ? blk.s.lk - blk.s.lq : blk.s.lk;
    const float* src0 = part<D>(s, 0);
    auto source = [&](int w) { return src0 + int64_t(2 * w + (w == first)) * kRows * (D + 2); };
    const uint32_t at = 4 * (64 * (D / 8) * wave + 64 * (kJoin / 8) * int(blockIdx.y) + lane);
    float m = -__builtin_inff(), l = 0.0f;
    f32x4_t o[kJoin / 8] = {};
    for (int w = first; w <= last_wg; ++w) {
        const float* src = source(w);
        f32x4_t x[kJoin / 8];
#pragma unroll
        for (int i = 0; i < kJoin / 8; ++i) x[i] = *reinterpret_cast<const f32x4_t*>(src + at + 256 * i);
        const float mw = src[kRows * D + mine], lw = src[kRows * D + kRows + mine];
        // A part whose maximum is -infinity has nothing, or NaN.
        const float top = fmaxf(m, mw);
        const float f = mw == -__builtin_inff() ? 1.0f : exp2_hw((mw - top) * p.c);
        const float down = m == -__builtin_inff() ? 1.0f : exp2_hw((m - top) * p.c);
        m = top;
        l = __builtin_fmaf(l, down, f * lw);
#pragma unroll
        for (int i = 0; i < kJoin / 8; ++i) o[i] = o[i] * down + x[i] * f;
    }
    if (row >= blk.s.lq) return;
    const float inv = (p.causal ? min(row + ahead, blk.s.lk - 1) : blk.s.lk - 1) < 0 ? 0.0f : 1.0f / l;
    uint16_t* out = p.out + (int64_t(blk.s.q0 + row) * p.heads + blk.head) * D + kJoin * int(blockIdx.y) + 4 * half;
#pragma unroll
    for (int i = 0; i < kJoin / 8; ++i)
        *reinterpret_cast<u32x2_t*>(out + 8 * i) =
            u32x2_t{pack2<DT>(o[i][0] * inv, o[i][1] * inv), pack2<DT>(o[i][2] * inv, o[i][3] * inv)};
}

// Workgroups that the chip runs at once: two a CU, one of head_dim 256.
int resident(int head_dim) { return head_dim == 256 ? 256 : 512; }

// Blocks there can be: every sequence, and the rows behind the last, round up.
int64_t most_blocks(int64_t batch, int64_t q_rows, int64_t heads) { return (q_rows / kRows + batch + 1) * heads; }

// Whether blocks are dealt in equal runs, rather than one to a workgroup.  Not where
// there are three or more for every place on the chip (24 ragged prompts: 123 us a
// block a workgroup, 153 + 16 in runs).  Else runs save what the longest block has
// over the average place, and cost the parts and the join, as much as `worth` tiles.
// Of several sequences only the sum of keys is known here, so the longest is taken
// for all of it and the average for nothing.  A block a workgroup / in runs, us:
// 8 heads of 256, 300 tokens 19.9 / 24.2, 500 27.0 / 29.3, 700 31.2 / 30.8, 1000 42.4 /
// 33.2; 32 of them, 800 36.5 / 50.9; 100 tokens behind 400 26.3 / 23.5; 8 heads of 128,
// 300 12.7 / 18.3, 1200 27.1 / 30.3, 1500 33.4 / 32.7; 32 of them, 1900 48.3 / 58.4; 16
// heads of 64, 300 9.7 / 16.6, 1500 24.8 / 29.4.
bool in_runs(int64_t batch, int64_t q_rows, int64_t k_rows, int64_t heads, int head_dim) {
    const int64_t blocks = most_blocks(batch, q_rows, heads), worth = head_dim == 256 ? 7 : 18;
    if (blocks >= 3 * resident(head_dim)) return false;
    const int64_t longest = (k_rows + kKeys - 1) / kKeys, before = q_rows / kRows;
    const int64_t average = batch > 1 ? 0 : heads * (before + 1) * (longest > before ? longest - before : 0);
    return (longest - worth) * resident(head_dim) > average;
}

int64_t grid_of(int64_t batch, int64_t q_rows, int64_t k_rows, int64_t heads, int head_dim) {
    const int64_t blocks = most_blocks(batch, q_rows, heads);
    if (!in_runs(batch, q_rows, k_rows, heads, head_dim)) return blocks;
    const int64_t units = blocks * (kBegin + 1 + k_rows / kKeys), most = resident(head_dim);
    return units < most ? units : most;
}

template <int DT, int D>
int launch(const Split& s, hipStream_t stream) {
    hipLaunchKernelGGL((attention_prompt_kernel<DT, D>), dim3(s.grid), dim3(256), 0, stream, s);
    int rc = check_launch("attention_prompt");
    if (rc != NANOVLLM_GEMM_OK || !s.runs || s.grid == 1) return rc;
    hipLaunchKernelGGL((attention_prompt_join_kernel<DT, D>), dim3(s.grid - 1, D / kJoin), dim3(256), 0, stream, s);
    return check_launch("attention_prompt_join");
}

template <int DT>
int launch_dim(const Split& s, int head_dim, hipStream_t stream) {
    return head_dim == 64    ? launch<DT, 64>(s, stream)
           : head_dim == 128 ? launch<DT, 128>(s, stream)
                             : launch<DT, 256>(s, stream);
}

}  // namespace

int64_t attention_prompt_groups(int64_t batch, int64_t q_rows, int64_t k_rows, int64_t heads, int64_t head_dim) {
    return grid_of(batch, q_rows, k_rows, heads, static_cast<int>(head_dim));
}

int64_t attention_prompt_workspace(int64_t batch, int64_t q_rows, int64_t k_rows, int64_t heads, int64_t head_dim) {
    const int64_t grid = grid_of(batch, q_rows, k_rows, heads, static_cast<int>(head_dim));
    if (grid == 1 || !in_runs(batch, q_rows, k_rows, heads, static_cast<int>(head_dim))) return 0;
    return 2 * grid * kRows * (head_dim + 2) * 4;
}

int launch_attention_prompt(const PromptArgs& p, void* workspace, int head_dim, int dtype, hipStream_t s) {
    const int64_t grid = grid_of(p.batch, p.q_rows, p.k_rows, p.heads, head_dim);
    const Split split{p, static_cast<float*>(workspace), static_cast<int32_t>(grid),
                      in_runs(p.batch, p.q_rows, p.k_rows, p.heads, head_dim)};
    return dtype == NANOVLLM_GEMM_BF16 ? launch_dim<NANOVLLM_GEMM_BF16>(split, head_dim, s)
                                       : launch_dim<NANOVLLM_GEMM_F16>(split, head_dim, s);
}

}  // namespace nvg
