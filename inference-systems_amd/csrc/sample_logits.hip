// sample_logits: a token a row by temperature, top-k, top-p and min-p from a
// given random number (the definition is in nanovllm_sampling.h).
//
// The three filters each keep a run from the front of the row's order (largest
// logit first, lowest index first among equals), so what is kept is given by one
// border: the pair (logit, index) of the last token that all of them keep.  No
// row is sorted.  With c = 16 log2(e) / T a token's weight is 2^((l c) / 16), and
// the whole number next to l c puts it into one of 1024 bins of 1/16 octave below
// the largest logit's; within a bin weights differ by less than 2^(1/16), and
// what is left of l c is the argument of a short polynomial.  A histogram of
// counts and weights by bin finds the bin of a border, and only that bin's
// members are put in order.
//
// Workgroups keep slices of the rows in LDS, bin them below their own largest logit
// (the whole number is the same whatever it is counted from, so slices are joined
// by a shift) and leave their histogram and their first few members, 1/128 of a
// slice.  One workgroup a row joins the histograms; where all that is kept is
// among the listed members (usual: a top-k, or a distribution with peaks), it puts
// those in order and draws, and the row is read once.  Otherwise it looks the
// members of the border's bin up in the row, and draws in the slice in which the
// running sum passes u times the total, which it reads again.
//
// What bounds it: with many rows the instructions of a weight (23 a logit, 33 with
// its bin, half of the slices' time; the histogram's atomics run beside them for
// nothing), a slice's list (a fifth) and its fixed steps; with few the join, a chain of short steps whose code is fetched as it runs:
// loops are left rolled and what a step shares with another is a call.
//
// Measured: 1 x 151936 bf16, top-k 50 and top-p 0.9: 25 us, of which the slices 8
// and the join 15.  256 x 151936 fp32 (156 MB), top-p and min-p by row: 120 us; the
// slices 71 (2.2 TB/s; reading alone takes 25), the join 50, which is the time of
// the rows that look their border up (others 15).  One workgroup a row for all of
// it: 176 and 231 us.  Slices by 512 threads instead of 1024: 82 us for 78.
//
// Numerics: l c is held as a product and its remainder; a weight within its bin
// is a whole number of 2^-36, off by less than 8 of them (sample_weights.hpp), and
// summed as one, in one 64-bit word with the count.  Sums over bins are in 64 bits and do not depend
// on the order of atomics.  The last bin holds everything from 2^-63.9 of the
// largest weight down, which counts as 0.
#include "int8_common.hpp"
#include "sample_weights.hpp"

#include <type_traits>

namespace nvg {
namespace {

constexpr int kThreads = 1024;
constexpr int kPer = 8;               // logits a thread takes at once
constexpr int kTile = kThreads * kPer;
constexpr int kList = 512;           // members of a bin that are put in order at once
constexpr uint32_t kNanKey = 0xFFC00000u;

// A token's place in the order: larger is earlier.
__device__ __forceinline__ uint64_t place_of(uint32_t key, int index) {
    return (uint64_t(key) << 32) | uint64_t(0xFFFFFFFFu - uint32_t(index));
}

// A bin's count and weight in one word: the count from bit 48 up, and below it
// off + kOff of its members, each below 2^32, so 2^15 members fit.
constexpr int32_t kOff = 1600000000;
constexpr int kCountBit = 48;
constexpr int kMostSlice = 1 << 15;

__device__ __forceinline__ uint64_t packed(int32_t off) {
    return (uint64_t(1) << kCountBit) | uint32_t(off + kOff);
}
__device__ __forceinline__ uint32_t count_of(uint64_t word) { return uint32_t(word >> kCountBit); }
__device__ __forceinline__ uint64_t sum_of(uint64_t word) {
    return (word & ((uint64_t(1) << kCountBit) - 1)) + count_of(word) * ((uint64_t(1) << 36) - uint64_t(kOff));
}

// weigh_finite and log as calls, for where they run once.
__device__ __attribute__((noinline)) Weight weigh_once(float l, Scale s) { return weigh_finite(l, s); }
__device__ __attribute__((noinline)) double log_once(double x) { return log(x); }

template <int DT>
__device__ __forceinline__ float logit_at(const char* row, int i) {
    if constexpr (DT == NANOVLLM_GEMM_F32) return reinterpret_cast<const float*>(row)[i];
    else return half_to_f32<DT>(reinterpret_cast<const uint16_t*>(row)[i]);
}

// Logits i .. i + C - 1 (4 or 8) of a row of n; NaN past its end.
template <int DT, int C>
__device__ __forceinline__ void load_logits(const char* row, int i, int n, float* l) {
    if (i + C <= n) {
        if constexpr (DT == NANOVLLM_GEMM_F32) {
            f32x4_t v[C / 4];
            __builtin_memcpy(v, row + int64_t(i) * 4, C * 4);
#pragma unroll
            for (int e = 0; e < C; ++e) l[e] = v[e >> 2][e & 3];
        } else {
            u32x2_t v[C / 4];
            __builtin_memcpy(v, row + int64_t(i) * 2, C * 2);
#pragma unroll
            for (int e = 0; e < C; ++e) l[e] = half_to_f32<DT>(uint16_t(v[e >> 2][(e >> 1) & 1] >> (16 * (e & 1))));
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < C; ++e) l[e] = i + e < n ? logit_at<DT>(row, i + e) : __builtin_nanf("");
}

// ---------------------------------------------------------------------------
// Sums over the workgroup.
// ---------------------------------------------------------------------------
constexpr int kMostSlices = 256;
constexpr int kFew = 2 * kThreads;    // listed members that decide: two a thread

// Where a bin is cut.
struct Border {
    uint64_t place;   // the last member in front of the cut
    double mass;      // weight up to and with it, in parts
};

struct Shared {
    uint32_t count[kBins];     // tokens of the bins up to one
    uint64_t words[kBins];     // the histogram (packed) while a slice is binned
    double mass[kBins];        // weight of the bins up to one
    union {
        struct { uint64_t list[kList], units[kList], front[kList]; uint32_t rank[kList]; };
        struct { uint32_t count[kBins]; uint64_t units[kBins]; } sub;
        double scale_of[kBins];   // of the bins' weights
    };
    uint64_t few[kFew];    // listed members of a row of one slice, by index; a bin's members
    uint64_t part64[kThreads / 64];
    double partd[kThreads / 64];
    uint32_t part32[kThreads / 64];
    int listed[kMostSlices];         // members a slice lists
    int shift[kMostSlices];          // bins from the row's largest logit down to a slice's
    uint64_t slice[kMostSlices];     // kept members of the border's bin by slice, in units
    uint32_t some[kThreads / 64];
    int fill;
    Scale scale;
    Border border;
};

// Moves between lanes as DPP: rows are 16 lanes; kShr + n takes the value n lanes
// down the row, kBcast15 and kBcast31 give a row's last lane to the next row, and
// lane 31 to the upper half.  Lanes that get none keep `old`.
constexpr int kShr = 0x110, kBcast15 = 0x142, kBcast31 = 0x143;

template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T moved(T old, T v) {
    if constexpr (sizeof(T) == 8) {
        const uint64_t o = __builtin_bit_cast(uint64_t, old), b = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = uint32_t(__builtin_amdgcn_update_dpp(int(uint32_t(o)), int(uint32_t(b)), CTRL, ROWS, 15, false));
        const uint32_t hi =
            uint32_t(__builtin_amdgcn_update_dpp(int(uint32_t(o >> 32)), int(uint32_t(b >> 32)), CTRL, ROWS, 15, false));
        return __builtin_bit_cast(T, (uint64_t(hi) << 32) | lo);
    } else {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, old), __builtin_bit_cast(int, v),
                                                                 CTRL, ROWS, 15, false));
    }
}

// What lane `lane` (the same in all) holds.
template <typename T>
__device__ __forceinline__ T from_lane(T v, int lane) {
    if constexpr (sizeof(T) == 8) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(b)), lane));
        const uint32_t hi = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(b >> 32)), lane));
        return __builtin_bit_cast(T, (uint64_t(hi) << 32) | lo);
    } else {
        return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
    }
}

constexpr int kWaves = kThreads / 64;
static_assert(kWaves == 16, "a wave's partial sums fill a row");

struct Add {
    template <typename T>
    __device__ __forceinline__ T operator()(T x, T y) const { return x + y; }
};
struct Max {
    template <typename T>
    __device__ __forceinline__ T operator()(T x, T y) const { return x > y ? x : y; }
};

// Inclusive over the lanes of a row, and over those of a wave (0 is neutral).
template <typename F, typename T>
__device__ __forceinline__ T row_scan(T v, F f) {
    v = f(v, moved<kShr + 1, 15>(T(0), v));
    v = f(v, moved<kShr + 2, 15>(T(0), v));
    v = f(v, moved<kShr + 4, 15>(T(0), v));
    return f(v, moved<kShr + 8, 15>(T(0), v));
}
template <typename F, typename T>
__device__ __forceinline__ T wave_scan(T v, F f) {
    v = row_scan(v, f);
    v = f(v, moved<kBcast15, 10>(T(0), v));
    return f(v, moved<kBcast31, 12>(T(0), v));
}

template <typename T>
__device__ __attribute__((noinline)) T max_over(T v, T* part) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_scan(v, Max{});
    __syncthreads();
    if (lane == 63) part[wave] = v;
    __syncthreads();
    return from_lane(row_scan(part[lane & (kWaves - 1)], Max{}), kWaves - 1);
}

// Inclusive sums over the threads in order, and the sum over all.
template <typename T>
struct Sums {
    T upto, all;
    __device__ __forceinline__ operator T() const { return upto; }
};
template <typename T>
__device__ __attribute__((noinline)) Sums<T> scan_over(T v, T* part) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    v = wave_scan(v, Add{});
    __syncthreads();
    if (lane == 63) part[wave] = v;
    __syncthreads();
    const T upto = row_scan(part[lane & (kWaves - 1)], Add{});
    return Sums<T>{wave > 0 ? from_lane(upto, wave - 1) + v : v, from_lane(upto, kWaves - 1)};
}

// The number of the first (or last) thread that says yes; `none` if none does.
__device__ __attribute__((noinline)) int pick(bool yes, int number, int none, bool last, uint32_t* part, uint32_t* some) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t all = __ballot(yes);
    int at = last ? 63 - __builtin_clzll(all | 1) : __builtin_ctzll(all | (uint64_t(1) << 63));
    const int mine = from_lane(number, __builtin_amdgcn_readfirstlane(at));
    __syncthreads();
    if (lane == 0) {
        part[wave] = uint32_t(mine);
        some[wave] = all != 0;
    }
    __syncthreads();
    const uint32_t theirs = part[lane & (kWaves - 1)];
    all = __ballot(lane < kWaves && some[lane & (kWaves - 1)] != 0);
    at = last ? 63 - __builtin_clzll(all | 1) : __builtin_ctzll(all | (uint64_t(1) << 63));
    const int found = int(from_lane(theirs, __builtin_amdgcn_readfirstlane(at) & (kWaves - 1)));
    return all != 0 ? found : none;
}

template <typename S>
__device__ __forceinline__ uint64_t max_all(uint64_t v, S& sh) { return max_over<uint64_t>(v, sh.part64); }
template <typename S>
__device__ __forceinline__ uint32_t max_all(uint32_t v, S& sh) { return max_over<uint32_t>(v, sh.part32); }
__device__ __forceinline__ Sums<double> scan(double v, Shared& sh) { return scan_over<double>(v, sh.partd); }
template <typename S>
__device__ __forceinline__ Sums<uint32_t> scan(uint32_t v, S& sh) { return scan_over<uint32_t>(v, sh.part32); }
template <typename S>
__device__ __forceinline__ Sums<uint64_t> scan(uint64_t v, S& sh) { return scan_over<uint64_t>(v, sh.part64); }
template <typename S>
__device__ __forceinline__ int first_of(bool yes, int number, int none, S& sh) {
    return pick(yes, number, none, false, sh.part32, sh.some);
}
__device__ __forceinline__ int last_of(bool yes, int number, int none, Shared& sh) {
    return pick(yes, number, none, true, sh.part32, sh.some);
}

// What thread `from` holds, in every thread.
template <typename T>
__device__ __forceinline__ T given_by(int from, T v, T* part) {
    __syncthreads();
    if (int(threadIdx.x) == from) part[0] = v;
    __syncthreads();
    return part[0];
}

// Calls f(index, logit) for the logits of the row from `low` to `high`.  Few are
// expected: they are marked first, at four instructions a logit.
template <int DT, typename F>
__device__ __forceinline__ void each_between(const char* row, int vocab, float low, float high, F f) {
    constexpr int kAhead = 2;   // loads in flight
    for (int base = threadIdx.x * kPer; base < vocab; base += kAhead * kTile) {
        float l[kAhead][kPer];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            if (a == 0 || base + a * kTile < vocab) {
                load_logits<DT, kPer>(row, base + a * kTile, vocab, l[a]);
            } else {
#pragma unroll
                for (int e = 0; e < kPer; ++e) l[a][e] = __builtin_nanf("");
            }
        }
        uint32_t hits = 0;
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
#pragma unroll
            for (int e = 0; e < kPer; ++e) hits |= l[a][e] >= low && l[a][e] <= high ? 1u << (a * kPer + e) : 0u;
#pragma unroll 1
        for (; hits; hits &= hits - 1) {
            const int at = __builtin_ctz(hits);
            float v = 0.0f;
#pragma unroll
            for (int e = 0; e < kAhead * kPer; ++e) v = at == e ? l[e / kPer][e % kPer] : v;
            f(base + at / kPer * kTile + at % kPer, v);
        }
    }
}

// A key's logit as a bound; keys below that of -inf are of no logit.
__device__ __forceinline__ float bound_of(uint32_t key) {
    return key > 0x007FFFFFu ? logit_of(key) : -__builtin_inff();
}

// ---------------------------------------------------------------------------
// The border within a bin, in sh.border: its need-th member (kByCount), or the
// member at which the running weight, in parts, reaches `want` (kByMass).
// ---------------------------------------------------------------------------
enum { kByCount, kByMass };

// The border among the `members` places in sh.list, which are of one bin.  The
// threads of a member, 1024 / members of them, count the places in front of it
// and sum their weights (whole numbers, in any order).
__device__ __attribute__((noinline)) void border_of_list(int members, int mode, uint32_t need, double want, double above,
                                                         Shared& sh) {
    int size = 64;
    while (size < members) size *= 2;
    const int i = threadIdx.x & (size - 1), part = threadIdx.x / size, parts = kThreads / size;
    __syncthreads();
    const uint64_t place = i < members ? sh.list[i] : 0;
    const uint64_t units = i < members ? units_of(weigh(logit_of(uint32_t(place >> 32)), sh.scale).off) : 0;
    if (part == 0) {
        sh.units[i] = units;
        sh.front[i] = 0;
        sh.rank[i] = 0;
    }
    __syncthreads();
    uint32_t rank = 0;
    uint64_t front = 0;
#pragma unroll 4
    for (int j = part; j < members; j += parts) {
        const bool ahead = sh.list[j] > place;
        rank += ahead;
        front += ahead ? sh.units[j] : 0;
    }
    if (i < members) {
        atomicAdd(&sh.rank[i], rank);
        atomicAdd(reinterpret_cast<unsigned long long*>(&sh.front[i]), static_cast<unsigned long long>(front));
    }
    __syncthreads();
    // The one that the cut lies behind; the last where rounding leaves the whole
    // a little short.
    if (part == 0 && i < members) {
        rank = sh.rank[i];
        const double before = double(sh.front[i]) * kUnit, upto = double(sh.front[i] + units) * kUnit;
        const bool cut = mode == kByMass ? (upto >= want || rank + 1 == uint32_t(members)) && (before < want || rank == 0)
                                         : rank + 1 == need;
        if (cut) sh.border = Border{place, above + upto};
    }
    __syncthreads();
}

template <int DT>
__device__ __forceinline__ void border_in(const char* row, int vocab, const Scale& sc, int bin, uint32_t members,
                                          int mode, uint32_t need, double want, Shared& sh) {
    const bool by_mass = mode == kByMass;
    // Keys of the members still in question, lo .. hi; need and want go down by
    // what lies above them.
    uint32_t hi = key_ceiling(bin, sc), lo = sc.flat ? hi : key_floor(bin, sc);
    double above = 0.0;
    auto inside = [&](float l, uint32_t key) { return key >= lo && key <= hi && weigh(l, sc).bin == bin; };
    // The row is read once where sh.few holds the bin's members.
    const uint32_t all = members;
    const bool whole = all <= uint32_t(kFew);
    if (whole) {
        __syncthreads();
        if (threadIdx.x == 0) sh.fill = 0;
        __syncthreads();
        each_between<DT>(row, vocab, bound_of(lo), bound_of(hi), [&](int i, float l) {
            const uint32_t key = argmax_order(l);
            if (inside(l, key)) sh.few[atomicAdd(&sh.fill, 1) & (kFew - 1)] = place_of(key, i);
        });
        __syncthreads();
    }
    auto each = [&](auto f) {
        if (whole) {
#pragma unroll 1
            for (uint32_t j = threadIdx.x; j < all; j += kThreads) {
                const uint64_t place = sh.few[j];
                const uint32_t key = uint32_t(place >> 32);
                if (key >= lo && key <= hi) f(place, key);
            }
        } else {
            each_between<DT>(row, vocab, bound_of(lo), bound_of(hi), [&](int i, float l) {
                const uint32_t key = argmax_order(l);
                if (inside(l, key)) f(place_of(key, i), key);
            });
        }
    };
    // Fewer are compared with each other (members^2 comparisons).
    const uint32_t most = whole ? 64 : kList;
    while (members > most && lo < hi) {
        const uint32_t width = (hi - lo) / kBins + 1;
        __syncthreads();
        sh.sub.count[threadIdx.x] = 0;
        sh.sub.units[threadIdx.x] = 0;
        __syncthreads();
        each([&](uint64_t, uint32_t key) {
            const uint32_t b = (hi - key) / width;
            atomicAdd(&sh.sub.count[b], 1u);
            atomicAdd(reinterpret_cast<unsigned long long*>(&sh.sub.units[b]),
                      static_cast<unsigned long long>(units_of(weigh_once(logit_of(key), sc).off)));
        });
        __syncthreads();
        const uint32_t n = sh.sub.count[threadIdx.x];
        const double m = double(sh.sub.units[threadIdx.x]) * kUnit;
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
        const double part = part_of(weigh(logit_of(hi), sc).off);
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
            load_logits<DT, kPer>(row, i, vocab, l);
#pragma unroll
            for (int e = 0; e < kPer; ++e) here += i + e < vocab && argmax_order(l[e]) == hi;
            const Sums<uint32_t> sums = scan(here, sh);
            const uint32_t upto = sums.upto, all = sums.all;
            if (seen + all >= c) {   // uniform
                uint32_t k = seen + upto - here;
                if (k < c && seen + upto >= c) {
#pragma unroll
                    for (int e = 0; e < kPer; ++e)
                        if (i + e < vocab && argmax_order(l[e]) == hi && ++k == c)
                            sh.border = Border{place_of(hi, i + e), above + double(c) * part};
                }
                __syncthreads();
                return;
            }
            seen += all;
        }
        return;   // not reached: there are c of them
    }
    // The members, in any order; each finds what lies in front of it.
    __syncthreads();
    if (threadIdx.x == 0) sh.fill = 0;
    __syncthreads();
    each([&](uint64_t place, uint32_t) { sh.list[atomicAdd(&sh.fill, 1) & (kList - 1)] = place; });
    border_of_list(int(members), mode, need, want, above, sh);
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
    // What slices leave: `slices` of `step` logits a row.
    char* work;
    int32_t slices, step;
};

// A slice's record in the workspace.
struct Record {
    uint64_t best;       // its first place
    int32_t listed;      // members listed
    int32_t last;        // its last bin (counted from its own largest) all of whose members are listed; -1: none
    uint64_t words[kBins];
    // then the listed places, by index, list_room of them at most
};

// Members a slice lists: a few of its tokens, and of a row kFew at most.  Even, so
// that a thread of the join takes two next to each other.
__host__ __device__ inline int list_room(int step, int slices) {
    const int share = kFew / (slices > 0 ? slices : 1) & ~1;
    return step / 128 < share ? step / 128 : share;
}
__host__ __device__ inline int64_t record_bytes(int step, int slices) {
    return int64_t(sizeof(Record)) + list_room(step, slices) * 8;
}

template <int STEP>
struct SliceShared {
    uint64_t words[kBins];
    uint64_t part64[kWaves];
    uint32_t part32[kWaves], some[kWaves];
};

// A slice of up to STEP logits from `begin` on, kept in LDS as they are given;
// NaN past the end.  Thread t has logits 8 t .. 8 t + 7 of every 8192.
template <int DT, int STEP>
struct Slice {
    static constexpr int B = DT == NANOVLLM_GEMM_F32 ? 4 : 2, E = 16 / B, G = STEP / kTile;
    static_assert(G * kTile == STEP && G <= 4, "a count of 16 bits a group");
    char* kept;      // STEP * B bytes
    int begin, n;
    uint64_t best;   // its first place
    Scale sc;

    __device__ __forceinline__ int first(int g) const { return g * kTile + int(threadIdx.x) * kPer; }

    static constexpr int R = G * kPer / E;   // 16-byte loads a thread
    // Whole runs of 8 logits of the slice from `from` on (of size logits).
    static __device__ __forceinline__ void request(const char* row, int from, int size, u32x4_t (&v)[R]) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int i = g * kTile + int(threadIdx.x) * kPer;
            if (i + kPer <= size) {
#pragma unroll
                for (int h = 0; h < kPer / E; ++h)
                    __builtin_memcpy(&v[g * (kPer / E) + h], row + int64_t(from + i + h * E) * B, 16);
            }
        }
    }

    // Puts it into LDS and finds its first place: the largest key, then the first
    // index that holds it.
    template <typename S>
    __device__ __forceinline__ void take(const char* row, const u32x4_t (&v)[R], S& sh) {
        float top = -__builtin_inff();
        bool nan = false;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int i = first(g);
            if (i + kPer <= n) {
#pragma unroll
                for (int h = 0; h < kPer / E; ++h) {
                    chunk(i + h * E) = v[g * (kPer / E) + h];
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float l = element(v[g * (kPer / E) + h], e);
                        top = __builtin_fmaxf(top, l);
                        nan |= l != l;
                    }
                }
            } else if (i < n) {
#pragma unroll 1
                for (int e = 0; e < kPer; ++e) {
                    uint32_t bits = DT == NANOVLLM_GEMM_F32 ? 0x7FC00000u : DT == NANOVLLM_GEMM_F16 ? 0x7E00u : 0x7FC0u;
                    if (i + e < n) {
                        const float l = logit_at<DT>(row, begin + i + e);
                        top = __builtin_fmaxf(top, l);
                        nan |= l != l;
                        if constexpr (B == 4) bits = reinterpret_cast<const uint32_t*>(row)[begin + i + e];
                        else bits = reinterpret_cast<const uint16_t*>(row)[begin + i + e];
                    }
                    if constexpr (B == 4) reinterpret_cast<uint32_t*>(kept)[i + e] = bits;
                    else reinterpret_cast<uint16_t*>(kept)[i + e] = uint16_t(bits);
                }
            }
        }
        const uint32_t mine = nan ? kNanKey : argmax_order(top), key = max_all(mine, sh);
        uint32_t at = 0;   // all bits less the index
        if (mine == key) {
#pragma unroll 1
            for (int g = 0; g < G && at == 0; ++g)
#pragma unroll 1
                for (int e = 0; e < kPer && at == 0; ++e)
                    if (first(g) + e < n && argmax_order(at_index(first(g) + e)) == key)
                        at = 0xFFFFFFFFu - uint32_t(begin + first(g) + e);
        }
        best = (uint64_t(key) << 32) | max_all(at, sh);
    }

    // Element e of 16 bytes of logits, and the 16 bytes from logit i on.
    static __device__ __forceinline__ float element(u32x4_t v, int e) {
        if constexpr (B == 4) {
            const uint32_t bits = v[e];   // of a vector's element the cast takes the first
            return __builtin_bit_cast(float, bits);
        }
        else return half_to_f32<DT>(uint16_t(v[e >> 1] >> (16 * (e & 1))));
    }
    __device__ __forceinline__ u32x4_t& chunk(int i) const { return *reinterpret_cast<u32x4_t*>(kept + i * B); }

    __device__ __forceinline__ float at_index(int i) const {
        if constexpr (B == 4) return __builtin_bit_cast(float, reinterpret_cast<const uint32_t*>(kept)[i]);
        else return logit_at<DT>(kept, i);
    }

    template <bool NEAR, typename S>
    __device__ __forceinline__ void bins_of(S& sh) {
#pragma unroll 1
        for (int i = int(threadIdx.x) * kPer; i < n; i += (i & 4) ? kTile - 4 : 4) {
            float l[4];
            if constexpr (B == 4) {
                const u32x4_t v = chunk(i);
#pragma unroll
                for (int e = 0; e < 4; ++e) l[e] = element(v, e);
            } else {
                const u32x2_t v = *reinterpret_cast<const u32x2_t*>(kept + i * B);
#pragma unroll
                for (int e = 0; e < 4; ++e) l[e] = half_to_f32<DT>(uint16_t(v[e >> 1] >> (16 * (e & 1))));
            }
            Weight w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = weigh_finite<NEAR>(l[e], sc);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (w[e].bin < kRest)
                    atomicAdd(reinterpret_cast<unsigned long long*>(&sh.words[w[e].bin]),
                              static_cast<unsigned long long>(packed(w[e].off)));
        }
    }

    // Its histogram in sh.words, four logits side by side.  A slice of infinities
    // leaves none.
    template <typename S>
    __device__ __forceinline__ void bins(S& sh) {
        sh.words[threadIdx.x] = 0;
        __syncthreads();
        if (is_near(sc) && !sc.flat) bins_of<true>(sh);
        else if (!sc.flat) bins_of<false>(sh);
        __syncthreads();
    }

    // Calls put(at, index, key) for the logits from `least` on, at = 0, 1, ... by
    // index; returns how many there are.  16 bits of a word count the logits of
    // one of its groups.
    template <typename S, typename F>
    __device__ __forceinline__ uint32_t list(float least, S& sh, F put) {
        using Counts = std::conditional_t<(G > 2), uint64_t, uint32_t>;
        uint32_t hits = 0;   // bit 8 g + e: logit e of group g is listed
        Counts mine = 0;
#pragma unroll 1
        for (int g = 0; g < G; ++g) {
            if (first(g) >= n) break;
            uint32_t here = 0;
#pragma unroll
            for (int h = 0; h < kPer / E; ++h) {
                const u32x4_t v = chunk(first(g) + h * E);
#pragma unroll
                for (int e = 0; e < E; ++e) here |= element(v, e) >= least ? 1u << (h * E + e) : 0u;
            }
            hits |= here << (kPer * g);
            mine |= Counts(__builtin_popcount(here)) << (16 * g);
        }
        const Sums<Counts> upto = scan(mine, sh);
        const Counts at = upto.upto - mine;   // by group, its groups' starts to come
        uint32_t start = 0;
#pragma unroll 1
        for (int g = 0; g < G; ++g) {
            uint32_t where = start + uint32_t(at >> (16 * g) & 0xFFFFu);
            for (uint32_t here = hits >> (kPer * g) & 0xFFu; here; here &= here - 1) {
                const int i = first(g) + __builtin_ctz(here);
                put(where++, begin + i, argmax_order(at_index(i)));
            }
            start += uint32_t(upto.all >> (16 * g) & 0xFFFFu);
        }
        return start;
    }
};

__device__ __forceinline__ bool draws(float t, uint64_t best) {
    return t > 1e-10f && uint32_t(best >> 32) != kNanKey;
}

// The least logit that may be in bin `last` or above.
__device__ __forceinline__ float least_of(int last, const Scale& s) { return bound_of(key_floor(last, s)); }

// Workgroups take slice after slice, the logits of the next one on their way
// while this one is binned.
template <int DT, int STEP>
__global__ __launch_bounds__(kThreads, STEP <= 2 * kTile ? 8 : 4) void sample_slices_kernel(
    RowArgs p, int64_t rows) {
    using S = Slice<DT, STEP>;
    __shared__ SliceShared<STEP> sh;
    __shared__ u32x4_t kept[STEP * S::B / 16];
    const int64_t total = rows * p.slices;
    const uint32_t cap = list_room(p.step, p.slices);
    S slice;
    slice.kept = reinterpret_cast<char*>(kept);
    u32x4_t next[S::R];
    auto row_of = [&](int64_t r) { return p.logits + r * p.ld * S::B; };
    auto size_of = [&](int s) { return (s + 1) * p.step < p.vocab ? p.step : p.vocab - s * p.step; };
    int64_t r = blockIdx.x / p.slices;
    int s = int(blockIdx.x - r * p.slices);
    S::request(row_of(r), s * p.step, size_of(s), next);
    for (int64_t at = blockIdx.x; at < total;) {
        const float t = p.temperatures[r];
        Record* out = reinterpret_cast<Record*>(p.work + at * record_bytes(p.step, p.slices));
        slice.begin = s * p.step;
        slice.n = size_of(s);
        slice.take(row_of(r), next, sh);
        at += gridDim.x;
        r = at / p.slices;
        s = int(at - r * p.slices);
        if (at < total) S::request(row_of(r), s * p.step, size_of(s), next);
        if (threadIdx.x == 0) out->best = slice.best;
        if (draws(t, slice.best)) {
            slice.sc = scale_of(logit_of(uint32_t(slice.best >> 32)), t);
            slice.bins(sh);
            const uint64_t word = sh.words[threadIdx.x];
            out->words[threadIdx.x] = word;
            const uint32_t upto = scan(count_of(word), sh);
            const int last = first_of(upto > cap, threadIdx.x, kRest, sh) - 1;
            // Listed is what a logit's size may put into the bins up to `last`; the
            // join looks again.  Where that is more than there is room for (equals
            // next to the bin's end), none counts as listed.
            uint64_t* list = reinterpret_cast<uint64_t*>(out + 1);
            uint32_t listed = cap + 1;
            if (last >= 0)
                listed = slice.list(least_of(last, slice.sc), sh, [&](uint32_t i, int index, uint32_t key) {
                    if (i < cap) list[i] = place_of(key, index);
                });
            if (threadIdx.x == 0) {
                out->listed = listed <= cap ? int(listed) : 0;
                out->last = listed <= cap ? last : -1;
            }
        }
        __syncthreads();   // the slice in LDS has been read
    }
}

// One workgroup a row.  STEP 0: behind sample_slices_kernel; otherwise the row is
// one slice of its own.
template <int DT, int STEP>
__global__ __launch_bounds__(kThreads) void sample_row_kernel(RowArgs p) {
    __shared__ Shared sh;
    __shared__ u32x4_t kept_logits[STEP > 0 ? STEP * Slice<DT, kTile>::B / 16 : 1];
    const int64_t r = blockIdx.x;
    const int vocab = p.vocab, tid = threadIdx.x;
    const char* row = p.logits + r * p.ld * (DT == NANOVLLM_GEMM_F32 ? 4 : 2);
    const float t = p.temperatures[r], u = p.uniforms[r];
    const int32_t k = p.top_k != nullptr ? p.top_k[r] : 0;
    const float top_p = p.top_p != nullptr ? p.top_p[r] : 1.0f;
    const float min_p = p.min_p != nullptr ? p.min_p[r] : 0.0f;
    const int64_t record = record_bytes(p.step, p.slices);
    const char* records = p.work + r * p.slices * record;
    auto record_of = [&](int s) { return reinterpret_cast<const Record*>(records + s * record); };

    Slice<DT, STEP == 0 ? kTile : STEP> slice;
    uint64_t best = 0, its_best = 0;   // of the row, and of slice `tid`
    int its_last = 0, its_listed = 0;
    uint64_t place[2] = {0, 0};        // two of the row's listed members, by index
    if constexpr (STEP > 0) {
        u32x4_t v[Slice<DT, STEP>::R];
        Slice<DT, STEP>::request(row, 0, vocab, v);
        slice.kept = reinterpret_cast<char*>(kept_logits);
        slice.begin = 0;
        slice.n = vocab;
        slice.take(row, v, sh);
        best = slice.best;
    } else {
        if (tid < p.slices) {
            const Record* rec = record_of(tid);
            its_best = rec->best;
            its_last = rec->last;
            its_listed = rec->listed;
        }
        const int cap = list_room(p.step, p.slices), s = 2 * tid / cap, i = 2 * tid - s * cap;
        if (s < p.slices) __builtin_memcpy(place, reinterpret_cast<const uint64_t*>(record_of(s) + 1) + i, 16);
        best = max_all(its_best, sh);
    }
    const uint32_t best_key = uint32_t(best >> 32);
    // The largest logit's token alone: a row that draws none, and what is left of
    // one where no kept token should have weight, so that every token written is
    // one of the row's.
    auto take_best = [&] {
        if (tid == 0) {
            p.tokens[r] = int(0xFFFFFFFFu - uint32_t(best));
            p.logprobs[r] = best_key == kNanKey ? __builtin_nanf("") : 0.0f;
        }
    };
    if (!draws(t, best)) return take_best();
    const Scale sc = scale_of(logit_of(best_key), t);
    if (tid == 0) sh.scale = sc;   // read behind the barriers of what follows

    // The row's histogram, and the last bin whose members are all listed.
    int covered = kRest;
    uint32_t count = 0;
    uint64_t units = 0;
    if (sc.flat) {
        // The holders of an infinity share the row.
        each_between<DT>(row, vocab, sc.largest, sc.largest, [&](int, float) { ++count; });
        count = scan(count, sh).all;
        count = tid == 0 ? count : 0;
        units = uint64_t(count) << 36;
        covered = -1;
    } else if constexpr (STEP > 0) {
        slice.sc = sc;
        slice.bins(sh);
        count = count_of(sh.words[tid]);
        units = sum_of(sh.words[tid]);
    } else {
        int mine = kRest;
        if (tid < p.slices) {
            const float largest = logit_of(uint32_t(its_best >> 32));
            const double down = sc.top - top_of(largest, sc);
            const bool some = __builtin_fabsf(largest) < __builtin_inff() && down < double(kRest);
            sh.shift[tid] = some ? int(down) : kRest;
            sh.listed[tid] = some ? its_listed : 0;
            if (some && int(down) + its_last < mine) mine = int(down) + its_last;
        }
        // The least of them, as the largest of what they are below kRest.
        covered = kRest - int(max_all(uint32_t(kRest - mine), sh));
        constexpr int kBatch = 24;   // loads in flight
        for (int first = 0; first < p.slices; first += kBatch) {
            uint64_t word[kBatch];
#pragma unroll
            for (int e = 0; e < kBatch; ++e) {
                const int s = first + e, b = s < p.slices ? tid - sh.shift[s] : -1;
                word[e] = b >= 0 && tid < kRest ? record_of(s)->words[b] : 0;
            }
#pragma unroll
            for (int e = 0; e < kBatch; ++e) {
                count += count_of(word[e]);
                units += sum_of(word[e]);
            }
        }
    }
    sh.count[tid] = scan(count, sh);
    sh.mass[tid] = scan(double(units) * kUnit * bin_scale(tid), sh);
    __syncthreads();
    auto members = [&](int b) { return b ? sh.count[b] - sh.count[b - 1] : sh.count[0]; };
    auto mass_before = [&](int b) { return b ? sh.mass[b - 1] : 0.0; };
    // The first bin with members at which the running mass reaches `want`; the last
    // one where rounding leaves the whole a little short.  A bin without members is
    // none: its sum is that of the bins before it in another order, which may pass
    // `want` in the last bit alone.
    const bool some = members(tid) > 0;
    auto bin_reaching = [&](double want) {
        const int b = first_of(some && sh.mass[tid] >= want, tid, -1, sh);
        return b >= 0 ? b : last_of(some, tid, 0, sh);
    };

    // The least logit whose weight is min_p or more, as a key.
    uint32_t least = 0;
    int least_bin = kRest;   // no member of a lower one has that weight
    if (min_p > 0.0f) {
        // At T = inf every finite logit weighs 1 (and the logarithm's product is no number).
        double l = double(sc.largest);
        if (t == __builtin_inff() && min_p <= 1.0f && !sc.flat) l = -__builtin_inf();
        else if (min_p < 1.0f) l += double(t) * log_once(double(min_p));
        const float near = float(l);
        least = argmax_order(near) + (double(near) < l ? 1u : 0u);
        if (min_p > 1.0f || least > best_key) least = best_key;
        least_bin = sc.flat ? 0 : weigh_once(logit_of(least), sc).bin;
    }
    const int k_bin = k > 0 && k < vocab ? first_of(sh.count[tid] >= uint32_t(k), tid, kRest, sh) : kRest;
    const double whole = sh.mass[kRest];
    // From 1 on no running sum is above it, whose last bits may pass the total's.
    const double share = u >= 1.0f ? __builtin_inf() : u > 0.0f ? double(u) : 0.0;

    // Where everything up to the border is listed, and not too many, the listed
    // members decide.  With a top-k in front of the top-p its whole bin is needed.
    int last = k_bin;
    if (top_p < 1.0f && k_bin == kRest) last = bin_reaching(double(top_p) * whole);
    const int p_bin = last;   // of the top-p where there is no top-k
    if (!(top_p < 1.0f && k_bin < kRest)) last = least_bin < last ? least_bin : last;
    if (last >= kRest) last = kRest - 1;
    bool few = covered >= last && sh.count[last] <= uint32_t(kFew);
    if constexpr (STEP > 0) {
        if (few) {
            const uint32_t n = slice.list(least_of(last, sc), sh, [&](uint32_t at, int i, uint32_t key) {
                if (at < uint32_t(kFew)) sh.few[at] = place_of(key, i);
            });
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 2; ++e) place[e] = 2 * uint32_t(tid) + e < n ? sh.few[2 * tid + e] : 0;
            few = n <= uint32_t(kFew);
        }
    } else {
        const int cap = list_room(p.step, p.slices), s = 2 * tid / cap, i = 2 * tid - s * cap;
        const int there = s < p.slices ? sh.listed[s] - i : 0;
#pragma unroll
        for (int e = 0; e < 2; ++e) place[e] = e < there ? place[e] : 0;
    }
    if (few) {
        Weight mine[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            mine[e] = Weight{kRest, 0};
            if (place[e] != 0) mine[e] = weigh_once(logit_of(uint32_t(place[e] >> 32)), sc);
        }
        uint64_t border = uint64_t(least) << 32;
        double total = whole;
#pragma unroll 1
        for (int mode = kByCount; mode <= kByMass; ++mode) {
            int b = k_bin;
            double want = 0.0;
            if (mode == kByCount) {
                if (k_bin > last) continue;
            } else {
                if (!(top_p < 1.0f)) continue;
                want = double(top_p) * total;
                b = bin_reaching(want);
                if (b > last) continue;
            }
            const int n = int(members(b));
            if (n > kList) {   // uniform: more than are put in order at once
                few = false;
                break;
            }
            __syncthreads();
            if (tid == 0) sh.fill = 0;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (mine[e].bin == b) sh.list[atomicAdd(&sh.fill, 1) & (kList - 1)] = place[e];
            border_of_list(n, mode, mode == kByMass ? 0u : uint32_t(k) - (b ? sh.count[b - 1] : 0u),
                           (want - mass_before(b)) / bin_scale(b), 0.0, sh);
            const Border at = sh.border;
            if (mode == kByCount) total = mass_before(b) + at.mass * bin_scale(b);
            border = at.place > border ? at.place : border;
        }
        border = border > best || min_p > 1.0f ? best : border;
        double w[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
            w[e] = place[e] >= border && mine[e].bin <= last ? part_of(mine[e].off) * bin_scale(mine[e].bin) : 0.0;
        if (few) {
            const Sums<double> sums = scan(w[0] + w[1], sh);
            const double sum = sums.upto;
            total = sums.all;
            const double target = share * total;
            // At u = 0 the first weight decides, also one that is lost in the sum with the other.
            const bool first = sum - w[1] > target || !(target > 0.0);
            const int one = w[0] > 0.0 && first ? 0 : w[1] > 0.0 && sum > target ? 1 : -1;
            int at = first_of(one >= 0, 2 * tid + one, -1, sh);
            if (at < 0) at = last_of(w[0] + w[1] > 0.0, 2 * tid + (w[1] > 0.0), -1, sh);
            if (at < 0) return take_best();
            if (tid == at >> 1) {
                p.tokens[r] = int64_t(0xFFFFFFFFu - uint32_t(place[at & 1]));
                p.logprobs[r] = static_cast<float>(log_once(w[at & 1] / total));
            }
            return;
        }
    }

    // The borders one after the other, from the bins' members in the row: the
    // top-k's, the top-p's of what that keeps, the min-p's.
    uint64_t border = 0;   // places from here on are kept
    double total = whole;
    bool listed = false;   // sh.few holds the members of the border's bin
    int border_bin = kRest;
#pragma unroll 1
    for (int mode = kByCount; mode <= kByMass; ++mode) {
        int b = k_bin;
        double want = 0.0;
        uint32_t need = 0;
        if (mode == kByCount) {
            // Without a top-p behind it a lower border than the min-p's is none.
            if (k_bin == kRest || (!(top_p < 1.0f) && least_bin < k_bin)) continue;
            need = uint32_t(k) - (b ? sh.count[b - 1] : 0u);
        } else {
            if (!(top_p < 1.0f) || (k_bin == kRest && least_bin < p_bin)) continue;
            want = double(top_p) * total;
            b = bin_reaching(want);
            if (b > border_bin) continue;   // rounding alone: the top-k's border stands
        }
        border_in<DT>(row, vocab, sc, b, members(b), mode, need, (want - mass_before(b)) / bin_scale(b), sh);
        const Border at = sh.border;
        // sh.few is of bin b now, where the border lies already or comes to lie.
        listed = members(b) <= uint32_t(kFew);
        if (at.place > border) {
            border = at.place;
            border_bin = b;
            if (mode == kByCount) total = mass_before(b) + at.mass * bin_scale(b);
        }
    }
    if (uint64_t(least) << 32 > border && least_bin < kRest) {
        border = uint64_t(least) << 32;
        border_bin = least_bin;
        listed = false;
    }
    if (border > best || min_p > 1.0f) {
        border = best;
        border_bin = 0;
        listed = false;
    }

    // Kept weight slice by slice, from the histograms and the members of the
    // border's bin; then the slice, and in it the thread's run, in which the running
    // sum passes u times the total.
    int from = 0, to = vocab;
    double ahead = 0.0;
    const bool by_slice = STEP == 0 && !sc.flat;
    if (by_slice) {
        __syncthreads();
        if (tid < p.slices) sh.slice[tid] = 0;
        __syncthreads();
        auto add = [&](int i, Weight w) {
            atomicAdd(reinterpret_cast<unsigned long long*>(&sh.slice[i / p.step]),
                      static_cast<unsigned long long>(units_of(w.off)));
        };
        if (border_bin < kRest && listed) {
            for (int i = tid; i < int(members(border_bin)); i += kThreads) {
                const uint64_t at = sh.few[i];
                if (at >= border) add(int(0xFFFFFFFFu - uint32_t(at)), weigh_once(logit_of(uint32_t(at >> 32)), sc));
            }
        } else if (border_bin < kRest) {
            const uint32_t least_key = uint32_t(border >> 32);
            each_between<DT>(row, vocab, bound_of(least_key), bound_of(key_ceiling(border_bin, sc)), [&](int i, float l) {
                if (place_of(argmax_order(l), i) < border) return;
                const Weight w = weigh_once(l, sc);
                if (w.bin == border_bin) add(i, w);
            });
        }
        __syncthreads();
        const int wave = tid >> 6, lane = tid & 63;
        for (int s = wave; s < p.slices; s += kThreads / 64) {
            const Record* rec = record_of(s);
            const int shift = sh.shift[s];
            uint64_t words[kBins / 64];
#pragma unroll
            for (int e = 0; e < kBins / 64; ++e) {   // the whole bins that are kept
                const int b = e * 64 + lane;
                words[e] = b < kRest && b + shift < border_bin ? rec->words[b] : 0;
            }
            double sum = 0.0;   // 64 bins are four octaves
#pragma unroll
            for (int e = kBins / 64 - 1; e >= 0; --e) sum = __builtin_fma(sum, 0x1p-4, double(sum_of(words[e])));
            sum *= kUnit * bin_scale(lane + shift);
#pragma unroll
            for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off);
            if (border_bin < kRest) sum += double(sh.slice[s]) * kUnit * bin_scale(border_bin);
            if (lane == 0) sh.mass[s] = sum;
        }
        __syncthreads();
        const double here = tid < p.slices ? sh.mass[tid] : 0.0;
        const Sums<double> sums = scan(here, sh);
        const double upto = sums.upto;
        total = sums.all;
        int s = first_of(here > 0.0 && upto > share * total, tid, kBins, sh);
        if (s == kBins) s = last_of(here > 0.0, tid, 0, sh);
        ahead = given_by(s, upto - here, sh.partd);
        from = s * p.step;
        to = from + p.step < vocab ? from + p.step : vocab;
    }
    __syncthreads();
    sh.scale_of[tid] = bin_scale(tid);
    __syncthreads();
    auto kept = [&](int i, float l) {
        const uint32_t key = argmax_order(l);
        if (place_of(key, i) < border) return 0.0;
        const Weight w = weigh(l, sc);
        return w.bin < kRest ? part_of(w.off) * sh.scale_of[w.bin] : 0.0;
    };
    // A run of logits a thread.
    const int run = ((to - from + kThreads - 1) / kThreads + kPer - 1) / kPer * kPer;
    const int begin = from + tid * run < to ? from + tid * run : to, end = to - begin < run ? to : begin + run;
    const float bound = bound_of(uint32_t(border >> 32));
    double mine = 0.0;
#pragma unroll 1
    for (int i = begin; i < end; i += kPer) {
        float l[kPer];
        load_logits<DT, kPer>(row, i, end, l);
        uint32_t hits = 0;
#pragma unroll
        for (int e = 0; e < kPer; ++e) hits |= l[e] >= bound ? 1u << e : 0u;
#pragma unroll 1
        for (; hits; hits &= hits - 1) {
            const int at = __builtin_ctz(hits);
            float v = l[0];
#pragma unroll
            for (int e = 1; e < kPer; ++e) v = at == e ? l[e] : v;
            mine += kept(i + at, v);
        }
    }
    const Sums<double> sums = scan(mine, sh);
    const double upto = sums.upto;
    if (!by_slice) total = sums.all;
    const double target = share * total - ahead;
    int at = first_of(mine > 0.0 && upto > target, tid, kThreads, sh);
    if (at == kThreads) at = last_of(mine > 0.0, tid, -1, sh);
    if (at < 0) return take_best();
    if (tid != at) return;
    double sum = upto - mine, its = 0.0;
    int token = begin;
#pragma unroll 1
    for (int i = begin; i < end && !(its > 0.0 && sum > target); ++i) {
        const double w = kept(i, logit_at<DT>(row, i));
        sum += w;
        if (w > 0.0) {
            token = i;
            its = w;
        }
    }
    p.tokens[r] = token;
    p.logprobs[r] = static_cast<float>(log_once(its / total));
}

// Logits of a slice: the whole row (0) where 64 KiB of LDS hold it; otherwise 8192
// while that makes no more than two rounds of workgroups, then 16384, and 32768,
// the most that a histogram counts, where a row has more slices than are joined.
int slice_step(int64_t m, int64_t vocab, int dtype) {
    constexpr int64_t kCus = 256;
    if (vocab <= (dtype == NANOVLLM_GEMM_F32 ? 2 * kTile : 4 * kTile)) return 0;
    const int64_t tiles = (vocab + kTile - 1) / kTile;
    if (tiles <= kMostSlices && m * tiles <= 4 * kCus) return kTile;
    return (tiles + 1) / 2 <= kMostSlices ? 2 * kTile : kMostSlice;
}

template <int DT>
int launch_typed(RowArgs a, int64_t m, hipStream_t s) {
    constexpr int B = DT == NANOVLLM_GEMM_F32 ? 4 : 2, kMost = B == 4 ? 2 * kTile : 4 * kTile;
    const dim3 rows(static_cast<uint32_t>(m)), block(kThreads);
    a.step = slice_step(m, a.vocab, DT);
    if (a.step == 0) {
        hipLaunchKernelGGL((sample_row_kernel<DT, kMost>), rows, block, 0, s, a);
        return check_launch("sample_logits");
    }
    a.slices = (a.vocab + a.step - 1) / a.step;
    // Two workgroups to a CU, one of the largest slices.
    const int64_t total = m * a.slices, room = a.step > 2 * kTile ? 256 : 512;
    const dim3 grid(static_cast<uint32_t>(total < room ? total : room));
    if (a.step == kTile) hipLaunchKernelGGL((sample_slices_kernel<DT, kTile>), grid, block, 0, s, a, m);
    else if (a.step == 2 * kTile) hipLaunchKernelGGL((sample_slices_kernel<DT, 2 * kTile>), grid, block, 0, s, a, m);
    else hipLaunchKernelGGL((sample_slices_kernel<DT, 4 * kTile>), grid, block, 0, s, a, m);
    const int rc = check_launch("sample_logits");
    if (rc != NANOVLLM_GEMM_OK) return rc;
    hipLaunchKernelGGL((sample_row_kernel<DT, 0>), rows, block, 0, s, a);
    return check_launch("sample_logits");
}

}  // namespace

int64_t sample_logits_workspace(int64_t m, int64_t vocab, int dtype) {
    const int step = slice_step(m, vocab, dtype);
    if (step == 0) return 0;
    const int64_t slices = (vocab + step - 1) / step;
    return m * slices * record_bytes(step, static_cast<int>(slices));
}

int launch_sample_logits(const SampleLogitsArgs& p, hipStream_t s) {
    const RowArgs a{static_cast<const char*>(p.logits), p.temperatures, p.uniforms, p.top_k, p.top_p, p.min_p, p.tokens,
                    p.logprobs, p.ld, static_cast<int32_t>(p.vocab), p.workspace, 0, 0};
    if (p.dtype == NANOVLLM_GEMM_F32) return launch_typed<NANOVLLM_GEMM_F32>(a, p.m, s);
    if (p.dtype == NANOVLLM_GEMM_F16) return launch_typed<NANOVLLM_GEMM_F16>(a, p.m, s);
    return launch_typed<NANOVLLM_GEMM_BF16>(a, p.m, s);
}

}  // namespace nvg
