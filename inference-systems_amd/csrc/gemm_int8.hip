// The 8-bit GEMM for rows of any length and alignment: what the tiles that copy
// whole aligned 16-byte chunks into LDS (mfma_* and splitk_decode with kI8) do
// not take.  A chunk comes through registers instead, by one unaligned 16-byte
// load; the chunk in which a row ends is loaded as the row's last 16 bytes and
// shifted into place, so nothing behind a row is read and what lies there (the
// next row, or nothing) does not enter the sum.  The loads of the next K-tile
// are in flight while this one is multiplied; LDS holds two K-tiles of 128
// codes, with the places of the other tiles (chunk c of row r at c ^ (r / 2 % 8)).
#include "int8_common.hpp"

namespace nvg {
namespace {

constexpr int kBK = 128;              // codes per K-tile and row
constexpr int kChunks = kBK / 16;

// Codes at..at + 15 of a row of k codes; zeros past its end.
__device__ __forceinline__ u32x4_t chunk_of(const int8_t* row, int at, int k) {
    u32x4_t v{0u, 0u, 0u, 0u};
    if (at + 16 <= k) {
        __builtin_memcpy(&v, row + at, 16);
    } else if (at < k) {
        if (k >= 16) {
            uint64_t w[2];
            __builtin_memcpy(w, row + k - 16, 16);
            const int drop = 8 * (16 - (k - at));   // bits in front of the chunk, 8 .. 120
            const uint64_t lo = drop >= 64 ? w[1] >> (drop - 64) : w[0] >> drop | w[1] << (64 - drop);
            const uint64_t hi = drop >= 64 ? 0 : w[1] >> drop;
            v = u32x4_t{uint32_t(lo), uint32_t(lo >> 32), uint32_t(hi), uint32_t(hi >> 32)};
        } else {
            for (int i = 0; i < k; ++i) v[i >> 2] |= uint32_t(uint8_t(row[i])) << (8 * (i & 3));
        }
    }
    return v;
}

// BM x BN tile (W rows), 4 waves, 2 x 2 over it.
template <int DT_OUT, int BM, int BN, int EPI>
__global__ __launch_bounds__(256) void int8_any_kernel(const int8_t* __restrict__ a, const int8_t* __restrict__ w,
                                                       int64_t m, int64_t n, int32_t k, int64_t lda, int64_t ldw,
                                                       void* __restrict__ c, int64_t ldc, int c_vec,
                                                       const float* __restrict__ row_scale,
                                                       const float* __restrict__ col_scale) {
    constexpr int NT = 256, ROWS = BM + BN;
    constexpr int BNO = EPI == EPI_SILU_MUL ? BN / 2 : BN;
    constexpr int WM = BM / 2, WN = BN / 2, MI = WM / 16, NI = WN / 16;
    constexpr int LOADS = ROWS * kChunks / NT;
    static_assert(LOADS * NT == ROWS * kChunks && WM % 16 == 0 && WN % 16 == 0, "tile shape");
    static_assert(EPI != EPI_SILU_MUL || NI % 2 == 0, "gate/up pairs per wave");
    constexpr int OB = DT_OUT == NANOVLLM_GEMM_F32 ? 4 : 2;
    constexpr int PITCH = BNO * OB + 16;
    constexpr int RING = 2 * ROWS * kChunks * 16;
    constexpr int LDS = RING > BM * PITCH ? RING : BM * PITCH;
    __shared__ u32x4_t ring[LDS / 16];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave >> 1, wn = wave & 1, r16 = lane & 15, quad = lane >> 4;
    const int tiles_m = static_cast<int>((m + BM - 1) / BM), tiles_n = static_cast<int>((n + BNO - 1) / BNO);
    int tm, tn;
    grouped_tile(xcd_remap(blockIdx.x, tiles_m * tiles_n), tiles_m, tiles_n, 8, tm, tn);
    const int64_t m0 = int64_t(tm) * BM, n0 = int64_t(tn) * BNO;

    // Thread t loads chunk t % 8 of rows t / 8 + 32 j; rows past m or n repeat the last.
    const int chunk = tid % kChunks;
    const int8_t* src[LOADS];
    int place[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const int r = tid / kChunks + NT / kChunks * j;
        place[j] = r * kChunks + (chunk ^ ((r >> 1) & 7));
        if (r < BM) {
            src[j] = a + min_i64(m0 + r, m - 1) * lda;
        } else {
            const int wr = r - BM;
            int64_t row;
            // 16 gate rows, then the 16 up rows of the same columns.
            if constexpr (EPI == EPI_SILU_MUL)
                row = min_i64(n0 + 16 * (wr >> 5) + (wr & 15), n - 1) + ((wr & 16) ? n : 0);
            else
                row = min_i64(n0 + wr, n - 1);
            src[j] = w + row * ldw;
        }
    }
    i32x4_t acc[NI][MI];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < MI; ++j) acc[i][j] = i32x4_t{};
    const int ktiles = (k + kBK - 1) / kBK;
    u32x4_t next[LOADS];
    auto load = [&](int t) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) next[j] = chunk_of(src[j], t * kBK + 16 * chunk, k);
    };
    load(0);
    const int swz = (r16 >> 1) & 7;
    for (int t = 0; t < ktiles; ++t) {
        u32x4_t* tile = ring + (t & 1) * ROWS * kChunks;
#pragma unroll
        for (int j = 0; j < LOADS; ++j) tile[place[j]] = next[j];
        // One barrier a K-tile: a wave that stores K-tile t + 2 here has passed
        // the barrier of t + 1, which every wave reaches after it read t.
        __syncthreads();
        if (t + 1 < ktiles) load(t + 1);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            u32x4_t af[MI], wf[NI];
#pragma unroll
            for (int i = 0; i < MI; ++i) af[i] = tile[(wm * WM + 16 * i + r16) * kChunks + ((4 * s + quad) ^ swz)];
#pragma unroll
            for (int i = 0; i < NI; ++i) wf[i] = tile[(BM + wn * WN + 16 * i + r16) * kChunks + ((4 * s + quad) ^ swz)];
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < MI; ++j) acc[i][j] = mma_16<kI8>(wf[i], af[j], acc[i][j]);
        }
    }

    // Output through LDS: acc[i][j][v] is row 16 j + l % 16, column 16 i + 4 (l / 16) + v of the wave tile.
    constexpr int CPR = BNO * OB / 16, EPC = 16 / OB;
    constexpr int NJ = EPI == EPI_SILU_MUL ? NI / 2 : NI;
    char* ctile = reinterpret_cast<char*>(ring);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NJ; ++i) {
        const int64_t col = n0 + wn * 16 * NJ + 16 * i + 4 * quad;
        const f32x4_t cg = col_scales4(col_scale, col, n);
        f32x4_t cu{};
        if constexpr (EPI == EPI_SILU_MUL) cu = col_scales4(col_scale + n, col, n);
#pragma unroll
        for (int j = 0; j < MI; ++j) {
            const int row = wm * WM + 16 * j + r16;
            const float rs = row_scale[min_i64(m0 + row, m - 1)];
            f32x4_t x = scaled4<RS_BOTH>(acc[EPI == EPI_SILU_MUL ? 2 * i : i][j], rs, cg);
            if constexpr (EPI == EPI_SILU_MUL) {
                const f32x4_t u = scaled4<RS_BOTH>(acc[2 * i + 1][j], rs, cu);
#pragma unroll
                for (int v = 0; v < 4; ++v) x[v] = silu_f32(x[v]) * u[v];
            }
            char* p = ctile + row * PITCH + (wn * 16 * NJ + 16 * i + 4 * quad) * OB;
            if constexpr (OB == 4) *reinterpret_cast<f32x4_t*>(p) = x;
            else *reinterpret_cast<u32x2_t*>(p) = u32x2_t{pack2<DT_OUT>(x[0], x[1]), pack2<DT_OUT>(x[2], x[3])};
        }
    }
    __syncthreads();
    if (!c_vec) {
        store_unaligned<OB, BM, BNO, NT>(ctile, PITCH, static_cast<char*>(c) + (m0 * ldc + n0) * OB, ldc, m - m0, n - n0,
                                         tid);
        return;
    }
    for (int e = tid; e < BM * CPR; e += NT) {
        const int r = e / CPR, ch = e % CPR;
        const int64_t grow = m0 + r, gcol = n0 + ch * EPC;
        if (grow >= m || gcol >= n) continue;
        const u32x4_t val = *reinterpret_cast<const u32x4_t*>(ctile + r * PITCH + ch * 16);
        char* gdst = static_cast<char*>(c) + (grow * ldc + gcol) * OB;
        if (gcol + EPC <= n) {
            *reinterpret_cast<u32x4_t*>(gdst) = val;
        } else {
            const int valid = int(min_i64(EPC, n - gcol));
            if constexpr (OB == 4) {
                for (int x = 0; x < valid; ++x) reinterpret_cast<uint32_t*>(gdst)[x] = val[x];
            } else {
                for (int x = 0; x < valid; ++x)
                    reinterpret_cast<uint16_t*>(gdst)[x] = uint16_t(val[x >> 1] >> (16 * (x & 1)));
            }
        }
    }
}

template <int DT_OUT, int BM, int BN, int EPI>
int launch_tile(const Int8Args& p, hipStream_t s) {
    constexpr int BNO = EPI == EPI_SILU_MUL ? BN / 2 : BN, OB = DT_OUT == NANOVLLM_GEMM_F32 ? 4 : 2;
    const int64_t tiles = ((p.m + BM - 1) / BM) * ((p.n + BNO - 1) / BNO);
    if (tiles > INT32_MAX) return set_error(NANOVLLM_GEMM_EINVAL, "gemm_int8: grid too large");
    const int c_vec = (reinterpret_cast<uintptr_t>(p.c) % 16 == 0) && ((p.ldc * OB) % 16 == 0);
    hipLaunchKernelGGL((int8_any_kernel<DT_OUT, BM, BN, EPI>), dim3(static_cast<uint32_t>(tiles)), dim3(256), 0, s, p.a,
                       p.w, p.m, p.n, static_cast<int32_t>(p.k), p.lda, p.ldw, p.c, p.ldc, c_vec, p.a_scales,
                       p.w_scales);
    return check_launch("int8_any", BM, BNO);
}

// The largest tile that leaves every CU a workgroup, of 64 x 64 seven CUs in eight:
// 333 x 2501 x 1003 (240 such tiles) takes 9.3 us with it and 10.4 us with 32 x 32,
// 200 x 4003 x 3001 (252) 18.8 and 23.3 us; 500 x 1501 x 2003 (192) 13.3 and 12.0 us,
// 300 x 2000 x 1003 (160) 8.4 and 7.9 us.
template <int DT_OUT, int EPI>
int launch_typed(const Int8Args& p, hipStream_t s) {
    constexpr int64_t kCus = 256;
    const int64_t rows = EPI == EPI_SILU_MUL ? 2 * p.n : p.n;
    auto tiles = [&](int64_t bm, int64_t bn) { return (p.m + bm - 1) / bm * ((rows + bn - 1) / bn); };
    if (tiles(128, 128) >= kCus) return launch_tile<DT_OUT, 128, 128, EPI>(p, s);
    if (tiles(64, 64) >= kCus - kCus / 8) return launch_tile<DT_OUT, 64, 64, EPI>(p, s);
    return launch_tile<DT_OUT, 32, EPI == EPI_SILU_MUL ? 64 : 32, EPI>(p, s);
}

template <int DT_OUT>
int launch_epi(const Int8Args& p, hipStream_t s) {
    return p.silu ? launch_typed<DT_OUT, EPI_SILU_MUL>(p, s) : launch_typed<DT_OUT, EPI_NONE>(p, s);
}

}  // namespace

int launch_int8_any(const Int8Args& p, hipStream_t s) {
    if (p.dtype_out == NANOVLLM_GEMM_F32) return launch_epi<NANOVLLM_GEMM_F32>(p, s);
    if (p.dtype_out == NANOVLLM_GEMM_F16) return launch_epi<NANOVLLM_GEMM_F16>(p, s);
    return launch_epi<NANOVLLM_GEMM_BF16>(p, s);
}

}  // namespace nvg
