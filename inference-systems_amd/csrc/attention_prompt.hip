// Attention of packed prompts: causal, grouped heads, sequences of different
// lengths.
//
// A workgroup takes 128 queries of one head of one sequence, 32 a wave, and
// walks over the keys in tiles that all waves share in LDS:
//   S^T[key, query] = K Q^T      32 x 32 x 16 products; accumulator v of lane l
//                                is key 8 (v / 4) + 4 (l / 32) + v % 4, query l % 32
//   P = 2^(c S - c max)          online softmax: a query's scores lie in two
//                                lanes, so its maximum and sum are lane values
//   O^T[channel, query] += V^T P with the keys of a product in the order in which
//                                the accumulators of S^T hold them: P never moves
// V^T is read from LDS transposed (ds_read_b64_tr_b16), 4 keys of a channel at
// a time, which is the run of keys a lane's accumulators hold.
#include <type_traits>

#include "attention_common.hpp"

namespace nvg {
namespace {

constexpr int kRows = 128;      // queries of a workgroup
constexpr float kLazy = 8.0f;   // sums are rescaled when a maximum grows by more than 2^8

// Tiles of all sequences, 128 queries each, and of the rows behind the last one.
__device__ __forceinline__ int start_of(const int32_t* cu, int b, int rows) { return min(max(cu[b], 0), rows); }

__device__ __forceinline__ bool find_tile(const PromptArgs& p, int tile, int& seq, int& index) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int b0 = 0; b0 <= p.batch; b0 += 64) {
        const int b = b0 + lane;
        int n = 0;
        if (b <= p.batch) {
            const int from = start_of(p.cu_q, b, p.q_rows), to = b < p.batch ? start_of(p.cu_q, b + 1, p.q_rows) : p.q_rows;
            n = max(0, (to - from + kRows - 1) / kRows);
        }
        int sum = n;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int up = __shfl_up(sum, off);
            if (lane >= off) sum += up;
        }
        const uint64_t past = __ballot(base + sum > tile);
        if (past) {
            const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
            seq = uniform(b0 + at);
            index = uniform(tile - base - __shfl(sum - n, at));
            return true;
        }
        base += uniform(__shfl(sum, 63));
    }
    return false;
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
__device__ __forceinline__ bool finite8(u32x4_t x) {
    constexpr uint32_t e = DT == NANOVLLM_GEMM_BF16 ? 0x7f80u : 0x7c00u;
    bool ok = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) ok = ok && (x[i] & e) != e && ((x[i] >> 16) & e) != e;
    return ok;
}

template <int DT>
__device__ __forceinline__ bool finite1(uint16_t x) {
    constexpr uint32_t e = DT == NANOVLLM_GEMM_BF16 ? 0x7f80u : 0x7c00u;
    return (x & e) != e;
}

// Values of a masked tile that hold an infinity or a NaN.  Products would carry
// it into rows that do not attend to its key (0 x infinity), so such elements
// are 0 in the products and each row adds its own share here: for every key it
// attends to, P times the elements that are not finite.  Slow and exact in
// what spreads; never run on finite values.
template <int DT, int D>
__device__ __forceinline__ void add_nonfinite(const PromptArgs& p, const uint16_t* qrow, const uint16_t* kbase,
                                           const uint16_t* vbase, int key0, int key1, int last, int half, float shift,
                                           f32x16_t (&o)[D / 32]) {
    for (int j = key0; j < key1; ++j) {
        const uint16_t* vrow = vbase + j * p.v_row;
        const uint16_t* krow = kbase + j * p.k_row;
        float s = 0.0f;
        for (int ch = 0; ch < D; ch += 8) {
            const u32x4_t a = load16(qrow + ch), b = load16(krow + ch);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                s = __builtin_fmaf(half_to_f32<DT>(uint16_t(a[w])), half_to_f32<DT>(uint16_t(b[w])), s);
                s = __builtin_fmaf(half_to_f32<DT>(uint16_t(a[w] >> 16)), half_to_f32<DT>(uint16_t(b[w] >> 16)), s);
            }
        }
        const float pj = exp2_hw(__builtin_fmaf(s, p.c, -shift));
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const uint16_t x = vrow[32 * dt + 8 * (v / 4) + 4 * half + v % 4];
                if (j <= last && !finite1<DT>(x)) o[dt][v] = __builtin_fmaf(pj, half_to_f32<DT>(x), o[dt][v]);
            }
    }
}

template <int DT, int D, int BN>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attention_prompt_kernel(const PromptArgs p) {
    constexpr int CH = D / 8;                  // 16-byte chunks of a row
    constexpr int KS = D / 16;                 // steps of the contraction over channels
    constexpr int DTILES = D / 32, NB = BN / 32;
    constexpr int LOADS = BN * CH / 256;       // 16-byte copies per thread and tile of K, or of V
    typedef short v4i16_t __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) v4i16_t* lds_v4;
    __shared__ u32x4_t kt[2][BN * CH], vt[2][BN * CH];

    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int group = p.heads / p.kv_heads;
    const int head = int(blockIdx.x) % p.heads, kvh = head / group;
    int b, index;
    if (!find_tile(p, int(blockIdx.x) / p.heads, b, index)) return;

    const int q0 = start_of(p.cu_q, b, p.q_rows);
    const int q1 = b < p.batch ? start_of(p.cu_q, b + 1, p.q_rows) : p.q_rows;
    const int k0 = b < p.batch ? start_of(p.cu_k, b, p.k_rows) : 0;
    const int k1 = b < p.batch ? start_of(p.cu_k, b + 1, p.k_rows) : 0;
    const int lq = q1 - q0, lk = max(0, k1 - k0);
    // The last tiles see the most keys: they come first.
    const int row0 = ((lq + kRows - 1) / kRows - 1 - index) * kRows;
    const int row = row0 + 32 * wave + col;                 // this lane's query
    const int ahead = p.causal ? lk - lq : lk;
    // Keys a row attends to: 0 .. last.
    const int last = p.causal ? min(row + ahead, lk - 1) : lk - 1;
    const int keys = p.causal ? min(lk, max(0, min(row0 + kRows, lq) + ahead)) : lk;
    const int tiles = (keys + BN - 1) / BN;
    // Tiles that every row of the workgroup attends to in full.
    const int full = p.causal ? max(0, min(lk, row0 + ahead + 1)) / BN : lk / BN;

    const uint16_t* qrow = p.q + int64_t(q0 + min(row, lq - 1)) * p.q_row + head * p.q_head;
    const uint16_t* kbase = p.k + int64_t(k0) * p.k_row + kvh * p.k_head;
    const uint16_t* vbase = p.v + int64_t(k0) * p.v_row + kvh * p.v_head;
    u32x4_t q[KS];
#pragma unroll
    for (int i = 0; i < KS; ++i) q[i] = load16(qrow + 16 * i + 8 * half);

    // Thread copies of tile `t`: a wave's instruction fills 64 neighbouring
    // chunks of LDS, each lane from the chunk that belongs there.  Rows behind
    // the end repeat the last one (their scores are masked).
    auto copy_tile = [&](int t, int stage) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int base = (i * 4 + wave) * 64, at = base + lane;
            const int r = at / CH, c = at % CH;
            const int64_t key = min(t * BN + r, lk - 1);
            dma16(kbase + key * p.k_row + 8 * k_chunk<D>(r, c), lds_address(&kt[stage][base]));
            dma16(vbase + key * p.v_row + 8 * v_chunk<D>(r, c), lds_address(&vt[stage][base]));
        }
    };

    f32x16_t o[DTILES];
#pragma unroll
    for (int i = 0; i < DTILES; ++i) o[i] = f32x16_t{};
    float m = -__builtin_inff(), l = 0.0f;

    // Addresses of V^T: lane j of 16 points at key j / 4 and channels 4 (j % 4) of
    // its 16-channel half; rows of a read differ from one another in their two
    // lowest bits only, which give the chunk exchange.
    const int vr = 4 * half + ((lane & 15) >> 2);
    const int vc = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    const uint32_t v_off = uint32_t(vr * CH * 16 + (lane & 1) * 8);

    if (tiles > 0) copy_tile(0, 0);
    for (int t = 0; t < tiles; ++t) {
        const int stage = t & 1;
        wait_vmcnt<0>();
        __syncthreads();
        if (t + 1 < tiles) copy_tile(t + 1, stage ^ 1);
        const bool masked = t >= full;
        const u32x4_t* kp = kt[stage];
        const u32x4_t* vp = vt[stage];
        f32x16_t sc[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            sc[n] = f32x16_t{};
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const int r = 32 * n + col;
                sc[n] = mfma_32x32x16<DT>(kp[r * CH + k_chunk<D>(r, 2 * i + half)], q[i], sc[n]);
            }
        }
        if (masked) {
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    if (t * BN + 32 * n + 8 * (v / 4) + 4 * half + v % 4 > last) sc[n][v] = -__builtin_inff();
        }
        float top = sc[0][0];
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int v = 0; v < 16; ++v) top = fmaxf(top, sc[n][v]);
        top = max_across32(top);
        // A first score (m is -infinity), or one that outgrows the range P has been given.
        if (__ballot((top - m) * p.c > kLazy)) {
            const float higher = fmaxf(m, top);
            const float down = higher == -__builtin_inff() ? 1.0f : exp2_hw((m - higher) * p.c);
            m = higher;
            l *= down;
#pragma unroll
            for (int i = 0; i < DTILES; ++i) o[i] *= down;
        }
        const float shift = m == -__builtin_inff() ? 0.0f : m * p.c;
        u32x4_t pk[NB][2];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                sc[n][v] = exp2_hw(__builtin_fmaf(sc[n][v], p.c, -shift));
                l += sc[n][v];
            }
#pragma unroll
            for (int w = 0; w < 8; ++w) pk[n][w / 4][w % 4] = pack2<DT>(sc[n][2 * w], sc[n][2 * w + 1]);
        }
        bool clean = true;
        if (masked) {
            // A look at the tile's values: see add_nonfinite.
#pragma unroll
            for (int i = 0; i < LOADS; ++i) clean = clean && finite8<DT>(vp[i * 256 + threadIdx.x]);
            clean = !__syncthreads_or(!clean);
        }
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
                for (int i = 0; i < DTILES; ++i) {
                    const uint32_t at = lds_address(vp) + v_off + uint32_t((32 * n + 16 * ks) * CH * 16) +
                                        uint32_t(v_chunk<D>(vr, 4 * i + vc) * 16);
                    const v4i16_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(uintptr_t)at);
                    const v4i16_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(uintptr_t)(at + 8 * CH * 16));
                    const u32x2_t l2 = __builtin_bit_cast(u32x2_t, lo), h2 = __builtin_bit_cast(u32x2_t, hi);
                    u32x4_t a = {l2[0], l2[1], h2[0], h2[1]};
                    if (!clean) {
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            if (!finite1<DT>(uint16_t(a[w]))) a[w] &= 0xffff0000u;
                            if (!finite1<DT>(uint16_t(a[w] >> 16))) a[w] &= 0xffffu;
                        }
                    }
                    o[i] = mfma_32x32x16<DT>(a, pk[n][ks], o[i]);
                }
            }
        if (!clean)
            add_nonfinite<DT, D>(p, qrow, kbase, vbase, t * BN, min(lk, t * BN + BN), last, half, shift, o);
    }

    l = sum_across32(l);
    if (row >= lq) return;
    const float inv = last < 0 ? 0.0f : 1.0f / l;     // no key: 0
    uint16_t* out = p.out + (int64_t(q0 + row) * p.heads + head) * D;
#pragma unroll
    for (int i = 0; i < DTILES; ++i)
#pragma unroll
        for (int v = 0; v < 16; v += 4)
            *reinterpret_cast<u32x2_t*>(out + 32 * i + 2 * v + 4 * half) =
                u32x2_t{pack2<DT>(o[i][v] * inv, o[i][v + 1] * inv), pack2<DT>(o[i][v + 2] * inv, o[i][v + 3] * inv)};
}

template <int DT>
int launch_dim(const PromptArgs& p, int head_dim, hipStream_t s) {
    // Every sequence, and the rows behind the last, round up to a tile of their own.
    const int64_t tiles = p.q_rows / kRows + p.batch + 1;
    const int64_t grid = tiles * p.heads;
    if (grid > INT32_MAX) return set_error(NANOVLLM_GEMM_EINVAL, "attention_prompt: too many rows and heads");
    const dim3 g(static_cast<uint32_t>(grid)), block(256);
    if (head_dim == 64) hipLaunchKernelGGL((attention_prompt_kernel<DT, 64, 64>), g, block, 0, s, p);
    else if (head_dim == 128) hipLaunchKernelGGL((attention_prompt_kernel<DT, 128, 64>), g, block, 0, s, p);
    else hipLaunchKernelGGL((attention_prompt_kernel<DT, 256, 64>), g, block, 0, s, p);
    return check_launch("attention_prompt");
}

}  // namespace

int launch_attention_prompt(const PromptArgs& p, int head_dim, int dtype, hipStream_t s) {
    return dtype == NANOVLLM_GEMM_BF16 ? launch_dim<NANOVLLM_GEMM_BF16>(p, head_dim, s)
                                       : launch_dim<NANOVLLM_GEMM_F16>(p, head_dim, s);
}

}  // namespace nvg
