// Rows in 8 bits with a scale each, from plain rows and behind the residual add
// and RMSNorm (the definition is in nanovllm_int8.h).
//
// Both are bound by memory: a row is read once, held in registers across the
// reduction of its maximum, and written once as codes.  A row belongs to 16, 64
// or 256 threads: short rows share a wave, those up to 2048 elements need no
// barrier, and only rows beyond 16384 are read twice (the sum is stored the second
// time).  Longer rows go to more
// threads, not to more chunks a thread: 8192 x 3584 fp16 takes 16.8 us with two
// chunks of 8 elements in each of 256 threads, 22.1 us with eight in a wave's.
//
// Measured: 8192 x 3584 fp16 16.8 us (88 MB, 5.3 TB/s), with four instructions for
// a code where its remainder proves it (22.5 us with the proof and its mend for each
// one); behind the norm 4100 x 1024 bf16 7.1 us (29 MB, 4.1 TB/s).
//
// The norm's row is z * c with z = s * (1 + w) and c = rsqrt(mean s^2 + eps)
// common to the row, so its codes are those of z and its scale is that of z
// times c: one reduction finds the maximum of |z| and the sum of s^2 together.
#include "gemm_common.hpp"
#include "int8_common.hpp"

namespace nvg {
namespace {

constexpr int kThreads = 256;

// A scale with what codes need of it.
struct Scale {
    float s;      // times `lift` where lifted
    float r;      // near 1 / s
    float lift;   // 1, or 2^64 where the row is so small that 1 / s overflows
};

// Scale of a row whose largest |x| has the bits `top`.  Returns the scale as it
// is written; `q` has s == 0 where the codes are 0.
__device__ __forceinline__ float row_scale_of(uint32_t top, Scale& q) {
    q = Scale{0.0f, 0.0f, 1.0f};
    if (top >= 0x7F800000u) return __builtin_nanf("");
    const float s = __builtin_bit_cast(float, top) / 127.0f;
    if (s == 0.0f) return 0.0f;
    q.lift = s < 0x1p-64f ? 0x1p64f : 1.0f;
    q.s = s * q.lift;
    q.r = 1.0f / q.s;
    return s;
}

// Code of x: rint(x / s), exact.  The product with the reciprocal is off by less
// than 2^-15 of a code, so rint of it is off by one at most, next to a half; the
// remainder x - q s, which fp32 holds, tells.  The sum with 1.5 * 2^23 rounds to a
// whole number whose low bits are the code.
constexpr float kMagic = 12582912.0f;
__device__ __forceinline__ uint32_t code_of(float x, const Scale& sc) {
    x *= sc.lift;
    const float y = x * sc.r + kMagic;
    const float q = y - kMagic;
    const float e = __builtin_fmaf(-q, sc.s, x), h = 0.5f * sc.s;
    const float far = __builtin_fabsf(e);
    int c = __builtin_bit_cast(int, y) - 0x4B400000;
    if (far > h || (far == h && (c & 1))) c += e > 0.0f ? 1 : -1;
    // A denormal scale may be so coarse that a quotient passes 127.
    return static_cast<uint32_t>(c < -127 ? -127 : c > 127 ? 127 : c);
}

// The codes of 8 elements, a byte each.  Four instructions an element where every
// remainder is below half a step (one in 2^15 is not), which proves the codes; a
// row of zeros or of NaN has s == 0 and never is.
__device__ __forceinline__ u32x2_t codes_of(const float (&x)[8], const Scale& sc) {
    uint32_t c[8];
    float far = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float y = x[i] * sc.r + kMagic;
        far = __builtin_fmaxf(far, __builtin_fabsf(__builtin_fmaf(kMagic - y, sc.s, x[i])));
        c[i] = __builtin_bit_cast(uint32_t, y);
    }
    if (!(far < 0.5f * sc.s) || sc.lift != 1.0f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = sc.s == 0.0f ? 0u : code_of(x[i], sc);
    }
    u32x2_t v;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        v[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[4 * i + 3], c[4 * i + 2], 0x0C0C0400u),
                                     __builtin_amdgcn_perm(c[4 * i + 1], c[4 * i], 0x0C0C0400u), 0x05040100u);
    return v;
}

// 8 elements at p as fp32; those at and past `left` are 0.
template <int DT>
__device__ __forceinline__ void load8(const char* p, int left, float (&x)[8]) {
    if (left >= 8) {
        if constexpr (DT == NANOVLLM_GEMM_F32) {
            f32x4_t v[2];
            __builtin_memcpy(v, p, 32);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = v[i >> 2][i & 3];
        } else {
            u32x4_t v;
            __builtin_memcpy(&v, p, 16);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = half_to_f32<DT>(uint16_t(v[i >> 1] >> (16 * (i & 1))));
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = 0.0f;
        if (i < left) {
            if constexpr (DT == NANOVLLM_GEMM_F32) x[i] = reinterpret_cast<const float*>(p)[i];
            else x[i] = half_to_f32<DT>(reinterpret_cast<const uint16_t*>(p)[i]);
        }
    }
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu; }

__device__ __forceinline__ void store_codes(int8_t* p, int left, const float (&x)[8], const Scale& sc) {
    const u32x2_t v = codes_of(x, sc);
    if (left >= 8) {
        __builtin_memcpy(p, &v, 8);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < left) p[i] = static_cast<int8_t>(v[i >> 2] >> (8 * (i & 3)));
}

// Maximum and sum over the TPR threads of a row (the sum in a fixed order).
template <int TPR>
__device__ __forceinline__ void reduce_row(uint32_t& top, float& sum) {
#pragma unroll
    for (int off = (TPR < 64 ? TPR : 64) / 2; off >= 1; off >>= 1) {
        const uint32_t o = static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off));
        top = o > top ? o : top;
        sum += __shfl_xor(sum, off);
    }
    if constexpr (TPR > 64) {
        __shared__ uint32_t tops[kThreads / 64];
        __shared__ float sums[kThreads / 64];
        if ((threadIdx.x & 63) == 0) {
            tops[threadIdx.x >> 6] = top;
            sums[threadIdx.x >> 6] = sum;
        }
        __syncthreads();
        top = 0;
        sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kThreads / 64; ++w) {
            top = tops[w] > top ? tops[w] : top;
            sum += sums[w];
        }
    }
}

// What a row's values are: plain elements, or s * (1 + w) of the norm.
struct RowArgs {
    const char *x, *r, *w;   // r, w: the norm's residual and weight
    int64_t ldx, ldr;        // elements
    char* res;
    int8_t* codes;
    float* scales;
    float eps;
    int32_t m, k;
};

template <int DT, int NORM, int STORE>
__device__ __forceinline__ void row_values(const char* __restrict__ x, const char* __restrict__ res_in,
                                           const char* __restrict__ weight, char* __restrict__ res, int c, int k,
                                           float (&z)[8], float& ss) {
    constexpr int B = DT == NANOVLLM_GEMM_F32 ? 4 : 2;
    const int left = k - c;
    load8<DT>(x + int64_t(c) * B, left, z);
    if constexpr (NORM) {
        float r[8], w[8];
        load8<DT>(res_in + int64_t(c) * B, left, r);
        load8<DT>(weight + int64_t(c) * B, left, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float s = z[i] + r[i];
            ss = __builtin_fmaf(s, s, ss);
            r[i] = s;
            z[i] = s * (1.0f + w[i]);
        }
        if constexpr (!STORE) return;
        uint16_t* out = reinterpret_cast<uint16_t*>(res) + c;
        if (left >= 8) {
            const u32x4_t v{pack2<DT>(r[0], r[1]), pack2<DT>(r[2], r[3]), pack2<DT>(r[4], r[5]), pack2<DT>(r[6], r[7])};
            __builtin_memcpy(out, &v, 16);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < left) out[i] = round_half<DT>(r[i]);
        }
    }
}

// CH chunks of 8 elements a thread; CH == 0: rows of any length, read twice.
template <int DT, int NORM, int TPR, int CH>
__global__ __launch_bounds__(kThreads) void quantize_kernel(
    const char* __restrict__ x, const char* __restrict__ res_in, const char* __restrict__ weight, int64_t ldx,
    int64_t ldr, char* __restrict__ res, int8_t* __restrict__ codes, float* __restrict__ scales, float eps, int32_t m,
    int32_t k) {
    constexpr int ROWS = kThreads / TPR, B = DT == NANOVLLM_GEMM_F32 ? 4 : 2;
    const int t = threadIdx.x % TPR;
    const int64_t row = int64_t(blockIdx.x) * ROWS + threadIdx.x / TPR;
    if (row >= m) return;   // whole rows' threads; a workgroup of one row has no such
    x += row * ldx * B;
    codes += row * k;
    if constexpr (NORM) {
        res_in += row * ldr * B;
        res += row * k * B;
    }
    uint32_t top = 0;
    float ss = 0.0f;
    auto higher = [&](const float (&z)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) top = abs_bits(z[i]) > top ? abs_bits(z[i]) : top;
    };
    float z[CH == 0 ? 1 : CH][8];
    if constexpr (CH > 0) {
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            const int c = 8 * (t + TPR * j);
#pragma unroll
            for (int i = 0; i < 8; ++i) z[j][i] = 0.0f;
            if (c < k) row_values<DT, NORM, 1>(x, res_in, weight, res, c, k, z[j], ss);
        }
#pragma unroll
        for (int j = 0; j < CH; ++j) higher(z[j]);
    } else {
        for (int c = 8 * t; c < k; c += 8 * TPR) {
            row_values<DT, NORM, 0>(x, res_in, weight, res, c, k, z[0], ss);
            higher(z[0]);
        }
    }
    reduce_row<TPR>(top, ss);
    Scale sc;
    float scale = row_scale_of(top, sc);
    if constexpr (NORM) {
        // Codes 0 with a scale of 0 (a sum of squares beyond fp32) or of no number
        // (one that rounds to 0, at eps = 0), as in rows that are so themselves.
        scale *= norm_scale(ss, k, eps);
        if (!(scale < __builtin_inff())) scale = __builtin_nanf("");
        if (!(scale > 0.0f)) sc.s = 0.0f;
    }
    if (t == 0) scales[row] = scale;
    if constexpr (CH > 0) {
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            const int c = 8 * (t + TPR * j);
            if (c < k) store_codes(codes + c, k - c, z[j], sc);
        }
    } else {
        float ignored = 0.0f;
        for (int c = 8 * t; c < k; c += 8 * TPR) {
            row_values<DT, NORM, 1>(x, res_in, weight, res, c, k, z[0], ignored);
            store_codes(codes + c, k - c, z[0], sc);
        }
    }
}

template <int DT, int NORM, int TPR, int CH>
int launch_rows(const RowArgs& p, hipStream_t s) {
    constexpr int ROWS = kThreads / TPR;
    const int64_t groups = (int64_t(p.m) + ROWS - 1) / ROWS;
    hipLaunchKernelGGL((quantize_kernel<DT, NORM, TPR, CH>), dim3(static_cast<uint32_t>(groups)), dim3(kThreads), 0, s,
                       p.x, p.r, p.w, p.ldx, p.ldr, p.res, p.codes, p.scales, p.eps, p.m, p.k);
    return check_launch(NORM ? "add_rmsnorm_quantize" : "quantize_rows");
}

template <int DT, int NORM>
int launch_typed(const RowArgs& p, hipStream_t s) {
    if (p.k <= 128) return launch_rows<DT, NORM, 16, 1>(p, s);
    if (p.k <= 512) return launch_rows<DT, NORM, 64, 1>(p, s);
    if (p.k <= 1024) return launch_rows<DT, NORM, 64, 2>(p, s);
    if (p.k <= 2048) return launch_rows<DT, NORM, 64, 4>(p, s);
    if (p.k <= 4096) return launch_rows<DT, NORM, 256, 2>(p, s);
    if (p.k <= 8192) return launch_rows<DT, NORM, 256, 4>(p, s);
    if (p.k <= 16384) return launch_rows<DT, NORM, 256, 8>(p, s);
    return launch_rows<DT, NORM, 256, 0>(p, s);
}

}  // namespace

int launch_quantize_rows(const void* x, int64_t ldx, int8_t* codes, float* scales, int64_t m, int64_t k, int dtype,
                         hipStream_t s) {
    const RowArgs p{static_cast<const char*>(x), nullptr, nullptr, ldx, 0, nullptr, codes, scales, 0.0f,
                    static_cast<int32_t>(m), static_cast<int32_t>(k)};
    if (dtype == NANOVLLM_GEMM_F32) return launch_typed<NANOVLLM_GEMM_F32, 0>(p, s);
    if (dtype == NANOVLLM_GEMM_F16) return launch_typed<NANOVLLM_GEMM_F16, 0>(p, s);
    return launch_typed<NANOVLLM_GEMM_BF16, 0>(p, s);
}

int launch_add_rmsnorm_quantize(const void* h, int64_t ldh, const void* r, int64_t ldr, const void* w, float eps,
                                int8_t* codes, float* scales, void* res, int64_t m, int64_t k, int dtype,
                                hipStream_t s) {
    const RowArgs p{static_cast<const char*>(h), static_cast<const char*>(r), static_cast<const char*>(w), ldh, ldr,
                    static_cast<char*>(res), codes, scales, eps, static_cast<int32_t>(m), static_cast<int32_t>(k)};
    if (dtype == NANOVLLM_GEMM_F16) return launch_typed<NANOVLLM_GEMM_F16, 1>(p, s);
    return launch_typed<NANOVLLM_GEMM_BF16, 1>(p, s);
}

}  // namespace nvg
