// sample_logits: a token a row by temperature, top-k, top-p and min-p from a
// given random number (the definition is in nanovllm_sampling.h).
//
// The three filters each keep a run from the front of the row's order (largest
// logit first, lowest index first among equals), so what is kept is given by one
// border: the pair (logit, index) of the last token that all of them keep.  No
// row is sorted.  With c = 16 log2(e) / T a token's weight is 2^((l c) / 16), and
// floor(l c) puts it into one of 1024 bins of 1/16 octave below the largest
// logit's; within a bin weights differ by less than 2^(1/16), and the exponent's
// fraction is a short polynomial.  A histogram of counts and weights by bin
// finds the bin of a border, and only that bin's members are put in order.
//
// Numerics: l c is held as a product and its remainder in 64 bits, so its
// fraction is exact at any size of l c; a weight within its bin is rounded to a
// multiple of 2^-40 and summed as an integer.  Sums do not depend on the order
// of atomics, and a border falls where 64-bit arithmetic puts it.  The last bin
// holds everything from 2^-63.9 of the largest weight down, which counts as 0.
#include "int8_common.hpp"

namespace nvg {
namespace {

constexpr int kThreads = 1024;
constexpr int kBins = 1024;
constexpr int kRest = kBins - 1;      // bin of the tokens without weight
constexpr int kPer = 8;               // logits a thread takes at once
constexpr int kTile = kThreads * kPer;
constexpr int kList = 4096;           // members of a bin that are put in order at once
constexpr uint32_t kNanKey = 0xFFC00000u;

// Logits as integers of the same order (argmax_order), and back.
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __builtin_bit_cast(float, (key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

// A token's place in the order: larger is earlier.
__device__ __forceinline__ uint64_t place_of(uint32_t key, int index) {
    return (uint64_t(key) << 32) | uint64_t(0xFFFFFFFFu - uint32_t(index));
}

struct Weight {
    int bin;
    double part;   // weight within its bin, 0.97 .. 1.03, a multiple of 2^-40
};

// How a row weighs its logits.
struct Scale {
    double c;      // 16 log2(e) / T
    double top;    // floor(c * largest logit)
    float largest;
    bool flat;     // the largest logit is an infinity: its holders share the row
};

__device__ __forceinline__ Scale scale_of(float largest, float t) {
    Scale s;
    s.c = 16.0 * 1.4426950408889634074 / double(t);
    s.top = __builtin_floor(double(largest) * s.c);
    s.largest = largest;
    s.flat = !(__builtin_fabsf(largest) < __builtin_inff());
    return s;
}

// 1 unit is 2^-40: 2^12 * 1.5 plus a part is rounded to a multiple of it.
constexpr double kRound = 6144.0;

__device__ __forceinline__ Weight weigh(float l, const Scale& s) {
#pragma clang fp contract(off)   // hi - f below is of the rounded product
    if (s.flat) return Weight{l == s.largest ? 0 : kRest, 1.0};
    const double hi = double(l) * s.c, lo = __builtin_fma(double(l), s.c, -hi), f = __builtin_floor(hi);
    const double down = s.top - f;
    // -inf, and 0 * inf at T = inf, are not below kRest either.
    const int bin = down < double(kRest) ? int(down) : kRest;
    // 2^(x / 16) around the middle of the bin: e^(x ln2 / 16) to the 6th power
    // is off by less than 2^-51.  Beyond 2^53 a product has no fraction, and its
    // remainder, the same for all tokens that can share its bin, is cut.
    double x = (hi - f) + lo - 0.5;
    x = __builtin_fmin(__builtin_fmax(x, -1.0), 1.0);
    constexpr double a = 0.69314718055994530942 / 16.0;
    double p = a * a * a * a * a * a / 720.0;
    p = __builtin_fma(p, x, a * a * a * a * a / 120.0);
    p = __builtin_fma(p, x, a * a * a * a / 24.0);
    p = __builtin_fma(p, x, a * a * a / 6.0);
    p = __builtin_fma(p, x, a * a / 2.0);
    p = __builtin_fma(p, x, a);
    p = __builtin_fma(p, x, 1.0);
    return Weight{bin, (p + kRound) - kRound};
}

// A part in units of 2^-40.
__device__ __forceinline__ uint64_t units_of(double part) {
    return __builtin_bit_cast(uint64_t, part + kRound) - __builtin_bit_cast(uint64_t, kRound);
}

// 2^(-bin / 16).
__device__ __forceinline__ double bin_scale(int bin) {
    constexpr double root[16] = {1.0,
                                 0.95760328069857364694, 0.91700404320467123174, 0.87812608018664974156,
                                 0.84089641525371454303, 0.80524516597462715411, 0.77110541270397041180,
                                 0.73841307296974965571, 0.70710678118654752440, 0.67712777346844636414,
                                 0.64841977732550483296, 0.62092890603674202431, 0.59460355750136053336,
                                 0.56939431737834582684, 0.54525386633262882960, 0.52213689121370692017};
    return __builtin_ldexp(root[bin & 15], -(bin >> 4));
}

template <int DT>
__device__ __forceinline__ float logit_at(const char* row, int i) {
    if constexpr (DT == NANOVLLM_GEMM_F32) return reinterpret_cast<const float*>(row)[i];
    else return half_to_f32<DT>(reinterpret_cast<const uint16_t*>(row)[i]);
}

// Logits i .. i + 7 of a row of n (-inf past its end; they are told apart by their index).
template <int DT>
__device__ __forceinline__ void load_logits(const char* row, int i, int n, float (&l)[kPer]) {
    if (i + kPer <= n) {
        if constexpr (DT == NANOVLLM_GEMM_F32) {
            f32x4_t v[2];
            __builtin_memcpy(v, row + int64_t(i) * 4, 32);
#pragma unroll
            for (int e = 0; e < kPer; ++e) l[e] = v[e >> 2][e & 3];
        } else {
            u32x4_t v;
            __builtin_memcpy(&v, row + int64_t(i) * 2, 16);
#pragma unroll
            for (int e = 0; e < kPer; ++e) l[e] = half_to_f32<DT>(uint16_t(v[e >> 1] >> (16 * (e & 1))));
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) l[e] = i + e < n ? logit_at<DT>(row, i + e) : -__builtin_inff();
}

// ---------------------------------------------------------------------------
// Sums over the workgroup.
// ---------------------------------------------------------------------------
struct Shared {
    uint32_t count[kBins];     // tokens of a bin, then of the bins up to it
    uint64_t units[kBins];     // weight of a bin in units
    double mass[kBins];        // weight of the bins up to it
    union {
        uint64_t list[kList];
        struct { uint32_t count[kBins]; uint64_t units[kBins]; } sub;
        double tile[kBins];    // kept weight of the row's tiles
    };
    uint64_t part64[kThreads / 64];
    double partd[kThreads / 64];
    uint32_t part32[kThreads / 64];
    int pick;
    int fill;
    uint64_t border;
};

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int off) {
    return (uint64_t(uint32_t(__shfl_xor(int(v >> 32), off))) << 32) | uint32_t(__shfl_xor(int(uint32_t(v)), off));
}

__device__ __forceinline__ uint64_t max_all(uint64_t v, Shared& sh) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        const uint64_t o = shfl_xor64(v, off);
        v = o > v ? o : v;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.part64[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) v = sh.part64[w] > v ? sh.part64[w] : v;
    return v;
}

__device__ __forceinline__ double sum_all(double v, Shared& sh) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.partd[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) v += sh.partd[w];
    return v;
}

// Inclusive sums over the threads in order.
__device__ __forceinline__ double scan(double v, Shared& sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const double o = __shfl_up(v, off);
        if (lane >= off) v += o;
    }
    __syncthreads();
    if (lane == 63) sh.partd[wave] = v;
    __syncthreads();
    double before = 0.0;
    for (int w = 0; w < wave; ++w) before += sh.partd[w];
    return before + v;
}

__device__ __forceinline__ uint32_t scan(uint32_t v, Shared& sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t o = static_cast<uint32_t>(__shfl_up(static_cast<int>(v), off));
        if (lane >= off) v += o;
    }
    __syncthreads();
    if (lane == 63) sh.part32[wave] = v;
    __syncthreads();
    uint32_t before = 0;
    for (int w = 0; w < wave; ++w) before += sh.part32[w];
    return before + v;
}

// The first number for which a thread says yes (`none` if none does).
__device__ __forceinline__ int first_of(bool yes, int number, int none, Shared& sh) {
    __syncthreads();
    if (threadIdx.x == 0) sh.pick = none;
    __syncthreads();
    if (yes) atomicMin(&sh.pick, number);
    __syncthreads();
    return sh.pick;
}

__device__ __forceinline__ int last_of(bool yes, int number, int none, Shared& sh) {
    __syncthreads();
    if (threadIdx.x == 0) sh.pick = none;
    __syncthreads();
    if (yes) atomicMax(&sh.pick, number);
    __syncthreads();
    return sh.pick;
}

// ---------------------------------------------------------------------------
// The border within a bin: the place of its need-th member (by_mass false), or
// of the member at which the running weight, in parts, reaches `want` (true),
// and the weight up to and with it, in parts.
// ---------------------------------------------------------------------------
struct Border {
    uint64_t place;
    double mass;
};

// Calls f(index, logit) for every logit of the row.
template <int DT, typename F>
__device__ __forceinline__ void each_logit(const char* row, int vocab, F f) {
    for (int i = threadIdx.x * kPer; i < vocab; i += kTile) {
        float l[kPer];
        load_logits<DT>(row, i, vocab, l);
#pragma unroll
        for (int e = 0; e < kPer; ++e)
            if (i + e < vocab) f(i + e, l[e]);
    }
}

template <int DT>
__device__ Border border_in(const char* row, int vocab, const Scale& sc, int bin, uint32_t members, bool by_mass,
                            uint32_t need, double want, Shared& sh) {
    // Keys of the members still in question, lo .. hi; need and want go down by
    // what lies above them.
    uint32_t lo = 0, hi = 0xFFFFFFFFu;
    double above = 0.0;
    auto inside = [&](float l, uint32_t key) { return key >= lo && key <= hi && weigh(l, sc).bin == bin; };
    if (members > uint32_t(kList)) {
        uint32_t low = 0xFFFFFFFFu, high = 0;
        each_logit<DT>(row, vocab, [&](int, float l) {
            if (weigh(l, sc).bin != bin) return;
            const uint32_t key = argmax_order(l);
            low = key < low ? key : low;
            high = key > high ? key : high;
        });
        hi = uint32_t(max_all(high, sh));
        lo = 0xFFFFFFFFu - uint32_t(max_all(0xFFFFFFFFu - low, sh));
    }
    while (members > uint32_t(kList) && lo < hi) {
        const uint32_t width = (hi - lo) / kBins + 1;
        __syncthreads();
        sh.sub.count[threadIdx.x] = 0;
        sh.sub.units[threadIdx.x] = 0;
        __syncthreads();
        each_logit<DT>(row, vocab, [&](int, float l) {
            const uint32_t key = argmax_order(l);
            if (!inside(l, key)) return;
            const uint32_t b = (hi - key) / width;
            atomicAdd(&sh.sub.count[b], 1u);
            atomicAdd(reinterpret_cast<unsigned long long*>(&sh.sub.units[b]),
                      static_cast<unsigned long long>(units_of(weigh(l, sc).part)));
        });
        __syncthreads();
        const uint32_t n = sh.sub.count[threadIdx.x];
        const double m = double(sh.sub.units[threadIdx.x]) * 0x1p-40;
        const uint32_t counts = scan(n, sh);
        const double masses = scan(m, sh);
        const int at = first_of(n > 0 && (by_mass ? masses >= want : counts >= need), threadIdx.x, kBins, sh);
        // Rounding may leave the whole a little short: then its last member.
        const int b = at < kBins ? at : last_of(n > 0, threadIdx.x, 0, sh);
        __syncthreads();
        if (int(threadIdx.x) == b) {
            sh.part32[0] = n;
            sh.part32[1] = counts - n;
            sh.partd[0] = masses - m;
        }
        __syncthreads();
        members = sh.part32[0];
        need -= sh.part32[1] < need ? sh.part32[1] : need - 1;
        want -= sh.partd[0];
        above += sh.partd[0];
        hi -= uint32_t(b) * width;
        lo = hi - lo >= width ? hi - (width - 1) : lo;
    }
    if (members > uint32_t(kList)) {
        // Equals: the c-th of them by index.
        const double part = weigh(logit_of(hi), sc).part;
        uint32_t c = need;
        if (by_mass) {
            c = want > 0.0 ? uint32_t(__builtin_ceil(want / part)) : 1u;
            c = c < 1u ? 1u : c > members ? members : c;
        }
        uint32_t seen = 0;
        for (int base = 0; base < vocab; base += kTile) {
            const int i = base + int(threadIdx.x) * kPer;
            uint32_t here = 0;
            float l[kPer];
            load_logits<DT>(row, i, vocab, l);
#pragma unroll
            for (int e = 0; e < kPer; ++e) here += i + e < vocab && argmax_order(l[e]) == hi;
            const uint32_t upto = scan(here, sh);
            __syncthreads();
            if (threadIdx.x == kThreads - 1) sh.part32[0] = upto;
            __syncthreads();
            const uint32_t all = sh.part32[0];
            if (seen + all >= c) {   // uniform
                uint32_t k = seen + upto - here;
                if (k < c && seen + upto >= c) {
#pragma unroll
                    for (int e = 0; e < kPer; ++e)
                        if (i + e < vocab && argmax_order(l[e]) == hi && ++k == c) sh.border = place_of(hi, i + e);
                }
                __syncthreads();
                return Border{sh.border, above + double(c) * part};
            }
            seen += all;
        }
        return Border{place_of(hi, vocab - 1), above + double(members) * part};   // not reached
    }
    // A list in order.
    __syncthreads();
    if (threadIdx.x == 0) sh.fill = 0;
    int size = 64;
    while (size < int(members)) size *= 2;
    for (int i = threadIdx.x; i < size; i += kThreads) sh.list[i] = 0;
    __syncthreads();
    each_logit<DT>(row, vocab, [&](int i, float l) {
        const uint32_t key = argmax_order(l);
        if (inside(l, key)) sh.list[atomicAdd(&sh.fill, 1) & (kList - 1)] = place_of(key, i);
    });
    for (int span = 2; span <= size; span *= 2) {
        for (int step = span / 2; step >= 1; step /= 2) {
            __syncthreads();
            for (int t = threadIdx.x; t < size / 2; t += kThreads) {
                const int i = 2 * t - (t & (step - 1)), j = i + step;
                const uint64_t x = sh.list[i], y = sh.list[j];
                if ((x < y) == ((i & span) == 0)) {   // descending runs first
                    sh.list[i] = y;
                    sh.list[j] = x;
                }
            }
        }
    }
    __syncthreads();
    constexpr int kEach = kList / kThreads;
    uint64_t place[kEach];
    double part[kEach], mine = 0.0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const int i = int(threadIdx.x) * kEach + e;
        place[e] = i < int(members) ? sh.list[i] : 0;
        part[e] = i < int(members) ? weigh(logit_of(uint32_t(place[e] >> 32)), sc).part : 0.0;
        mine += part[e];
    }
    double run = scan(mine, sh) - mine;   // exact: at most 2^12 parts of 2^-40
    int at = kList;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const int i = int(threadIdx.x) * kEach + e;
        run += part[e];
        part[e] = run;
        if (at == kList && i < int(members) && (by_mass ? run >= want : i + 1 >= int(need))) at = i;
    }
    at = first_of(at < kList, at, int(members) - 1, sh);
#pragma unroll
    for (int e = 0; e < kEach; ++e)
        if (int(threadIdx.x) * kEach + e == at) {
            sh.border = place[e];
            sh.partd[0] = part[e];
        }
    __syncthreads();
    const Border b{sh.border, above + sh.partd[0]};
    __syncthreads();
    return b;
}

struct RowArgs {
    const char* logits;
    const float *temperatures, *uniforms;
    const int32_t* top_k;
    const float *top_p, *min_p;
    int64_t* tokens;
    float* logprobs;
    int64_t ld;
    int32_t vocab;
};

// One workgroup a row.
template <int DT>
__global__ __launch_bounds__(kThreads) void sample_row_kernel(RowArgs p) {
    __shared__ Shared sh;
    const int64_t r = blockIdx.x;
    const int vocab = p.vocab;
    const char* row = p.logits + r * p.ld * (DT == NANOVLLM_GEMM_F32 ? 4 : 2);
    const float t = p.temperatures[r];

    uint64_t best = 0;
    each_logit<DT>(row, vocab, [&](int i, float l) {
        const uint64_t place = place_of(argmax_order(l), i);
        best = place > best ? place : best;
    });
    best = max_all(best, sh);
    const uint32_t best_key = uint32_t(best >> 32);
    const int best_index = int(0xFFFFFFFFu - uint32_t(best));
    if (!(t > 1e-10f) || best_key == kNanKey) {
        if (threadIdx.x == 0) {
            p.tokens[r] = best_index;
            p.logprobs[r] = best_key == kNanKey ? __builtin_nanf("") : 0.0f;
        }
        return;
    }
    const Scale sc = scale_of(logit_of(best_key), t);

    sh.count[threadIdx.x] = 0;
    sh.units[threadIdx.x] = 0;
    __syncthreads();
    each_logit<DT>(row, vocab, [&](int, float l) {
        const Weight w = weigh(l, sc);
        atomicAdd(&sh.count[w.bin], 1u);
        if (w.bin < kRest)
            atomicAdd(reinterpret_cast<unsigned long long*>(&sh.units[w.bin]),
                      static_cast<unsigned long long>(units_of(w.part)));
    });
    __syncthreads();
    {
        const uint32_t counts = scan(sh.count[threadIdx.x], sh);
        const double masses = scan(double(sh.units[threadIdx.x]) * 0x1p-40 * bin_scale(threadIdx.x), sh);
        sh.count[threadIdx.x] = counts;
        sh.mass[threadIdx.x] = masses;
    }
    __syncthreads();
    auto members = [&](int b) { return b ? sh.count[b] - sh.count[b - 1] : sh.count[0]; };
    auto mass_before = [&](int b) { return b ? sh.mass[b - 1] : 0.0; };

    uint64_t border = 0;   // places from here on are kept
    double total = sh.mass[kRest];
    const int32_t k = p.top_k != nullptr ? p.top_k[r] : 0;
    if (k > 0 && k < vocab) {
        const int b = first_of(sh.count[threadIdx.x] >= uint32_t(k), threadIdx.x, kRest, sh);
        if (b < kRest) {
            const Border at = border_in<DT>(row, vocab, sc, b, members(b), false,
                                            uint32_t(k) - (b ? sh.count[b - 1] : 0u), 0.0, sh);
            border = at.place;
            total = mass_before(b) + at.mass * bin_scale(b);
        }
    }
    const float top_p = p.top_p != nullptr ? p.top_p[r] : 1.0f;
    if (top_p < 1.0f) {
        const double want = double(top_p) * total;
        const int b = first_of(sh.mass[threadIdx.x] >= want, threadIdx.x, kRest - 1, sh);
        const Border at = border_in<DT>(row, vocab, sc, b, members(b), true, 0u,
                                        (want - mass_before(b)) / bin_scale(b), sh);
        border = at.place > border ? at.place : border;
    }
    const float min_p = p.min_p != nullptr ? p.min_p[r] : 0.0f;
    if (min_p > 0.0f) {
        // The least logit whose weight is min_p or more.
        const double least = min_p >= 1.0f ? double(sc.largest) : double(sc.largest) + double(t) * log(double(min_p));
        const float near = float(least);
        const uint64_t at = uint64_t(argmax_order(near) + (double(near) < least ? 1u : 0u)) << 32;
        border = at > border ? at : border;
        if (min_p > 1.0f) border = best;
    }
    border = border < best ? border : best;

    auto kept = [&](int i, float l) {
        const uint32_t key = argmax_order(l);
        if (place_of(key, i) < border) return 0.0;
        const Weight w = weigh(l, sc);
        return w.bin < kRest ? w.part * bin_scale(w.bin) : 0.0;
    };
    // Kept weight tile by tile, then the tile in which the running sum passes
    // u times the total, then the token.
    __syncthreads();
    sh.tile[threadIdx.x] = 0.0;
    for (int base = 0; base < vocab; base += kTile) {
        const int i = base + int(threadIdx.x) * kPer;
        double mine = 0.0;
        if (i < vocab) {
            float l[kPer];
            load_logits<DT>(row, i, vocab, l);
#pragma unroll
            for (int e = 0; e < kPer; ++e)
                if (i + e < vocab) mine += kept(i + e, l[e]);
        }
        const double all = sum_all(mine, sh);
        if (threadIdx.x == 0) sh.tile[base / kTile] = all;
    }
    __syncthreads();
    const double here = sh.tile[threadIdx.x];
    const double upto = scan(here, sh);
    __syncthreads();
    if (threadIdx.x == kThreads - 1) sh.partd[0] = upto;
    __syncthreads();
    total = sh.partd[0];
    const float u = p.uniforms[r];
    const double target = u > 0.0f ? double(u) * total : 0.0;
    int tile = first_of(here > 0.0 && upto > target, threadIdx.x, kBins, sh);
    if (tile == kBins) tile = last_of(here > 0.0, threadIdx.x, 0, sh);
    __syncthreads();
    if (int(threadIdx.x) == tile) sh.partd[0] = upto - here;
    __syncthreads();
    const double before = sh.partd[0];
    const int i = tile * kTile + int(threadIdx.x) * kPer;
    double w[kPer], mine = 0.0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) w[e] = 0.0;
    if (i < vocab) {
        float l[kPer];
        load_logits<DT>(row, i, vocab, l);
#pragma unroll
        for (int e = 0; e < kPer; ++e) w[e] = i + e < vocab ? kept(i + e, l[e]) : 0.0;
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) mine += w[e];
    double run = before + (scan(mine, sh) - mine);
    int found = INT32_MAX, last = -1;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        run += w[e];
        if (w[e] > 0.0) {
            if (found == INT32_MAX && run > target) found = i + e;
            last = i + e;
        }
    }
    int token = first_of(found != INT32_MAX, found, INT32_MAX, sh);
    if (token == INT32_MAX) token = last_of(last >= 0, last, 0, sh);
#pragma unroll
    for (int e = 0; e < kPer; ++e)
        if (i + e == token) {
            p.tokens[r] = token;
            p.logprobs[r] = static_cast<float>(log(w[e] / total));
        }
}

}  // namespace

int64_t sample_logits_workspace(int64_t, int64_t, int) { return 0; }

int launch_sample_logits(const SampleLogitsArgs& p, hipStream_t s) {
    const RowArgs a{static_cast<const char*>(p.logits), p.temperatures, p.uniforms, p.top_k, p.top_p, p.min_p, p.tokens,
                    p.logprobs, p.ld, static_cast<int32_t>(p.vocab)};
    const dim3 grid(static_cast<uint32_t>(p.m)), block(kThreads);
    if (p.dtype == NANOVLLM_GEMM_F32) hipLaunchKernelGGL(sample_row_kernel<NANOVLLM_GEMM_F32>, grid, block, 0, s, a);
    else if (p.dtype == NANOVLLM_GEMM_F16) hipLaunchKernelGGL(sample_row_kernel<NANOVLLM_GEMM_F16>, grid, block, 0, s, a);
    else hipLaunchKernelGGL(sample_row_kernel<NANOVLLM_GEMM_BF16>, grid, block, 0, s, a);
    return check_launch("sample_logits");
}

}  // namespace nvg
