// The weights of the sampler on logits, for device and host: which bin below the
// largest logit a token falls into, and what its weight is within it.  With
// c = 16 log2(e) / T a token's weight is 2^((l c) / 16); the whole number next to l c
// gives the bin, and what is left of l c is the argument of a short polynomial.
#pragma once

#include "gemm_common.hpp"

namespace nvg {

constexpr int kBins = 1024;
constexpr int kRest = kBins - 1;      // bin of the tokens without weight

// Logits as integers of the same order (argmax_order), and back.
__host__ __device__ __forceinline__ float logit_of(uint32_t key) {
    return __builtin_bit_cast(float, (key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

// A token's weight: 2^(-bin / 16) * (1 + off * 2^-36).
struct Weight {
    int bin;
    int32_t off;   // within 1.6e9 of 0
};
constexpr double kUnit = 0x1p-36;

__host__ __device__ __forceinline__ double part_of(int32_t off) { return 1.0 + double(off) * kUnit; }
// A part in units.
__host__ __device__ __forceinline__ uint64_t units_of(int32_t off) { return (uint64_t(1) << 36) + int64_t(off); }

// How a row weighs its logits.
struct Scale {
    double c;        // 16 log2(e) / T
    float ch, cl;    // the same as a sum
    double top;      // the largest logit's rounded product with it
    float topf;
    float floor;     // products in 32 bits below it are of bin kRest; NaN or -inf where topf is no number
    float largest;
    bool flat;       // the largest logit is an infinity: its holders share the row
};

// A logit's product with c, rounded to a whole number: in 32 bits where it is at
// most kNear, beyond that in 64 (never nearer to 0 than kNear, so that it does
// not fall with the logit).
constexpr float kNear = 16384.0f;

__host__ __device__ __forceinline__ double far_product(float l, const Scale& s, double& rest) {
#pragma clang fp contract(off)   // hi - f below is of the rounded product
    const double hi = double(l) * s.c, lo = __builtin_fma(double(l), s.c, -hi);
    double f = __builtin_rint(hi);
    f = f > 0.0 ? __builtin_fmax(f, double(kNear)) : __builtin_fmin(f, -double(kNear));
    // Beyond 2^53 a product has no fraction, and its remainder, the same for all
    // tokens that can share its bin, is cut.
    rest = __builtin_fmin(__builtin_fmax((hi - f) + lo, -0.5), 0.5);
    return f;
}

// A logit's product as a whole number.
__host__ __device__ __forceinline__ double top_of(float l, const Scale& s) {
    const float hi = l * s.ch;
    double rest;
    return __builtin_fabsf(hi) <= kNear ? double(__builtin_rintf(hi)) : far_product(l, s, rest);
}

__host__ __device__ __forceinline__ Scale scale_of(float largest, float t) {
    Scale s;
    s.c = 16.0 * 1.4426950408889634074 / double(t);
    s.ch = float(s.c);
    s.cl = float(s.c - double(s.ch));
    s.top = top_of(largest, s);
    s.topf = float(s.top);
    // A product in 32 bits is off by 2^-23 of itself (c and the product round),
    // topf by 2^-24, so what is in a bin lies within 1024 and 3 * 2^-24 |topf| of it.
    s.floor = s.topf - (2048.0f + 0x1p-21f * __builtin_fabsf(s.topf));
    s.largest = largest;
    s.flat = !(__builtin_fabsf(largest) < __builtin_inff());
    return s;
}

// Of a row whose largest logit is finite.  y, the product in 32 bits less its whole
// number, is exact; low is what that product leaves of l c.  2^(y / 16) - 1 in units
// of 2^-36: the linear term of y as a float and its remainder, the others, to the
// 5th power, with the remainder.
//
// Off by less than 8 units, at a product up to 2^14: less than 1 each for the cuts of
// both terms to whole numbers; 0.17 for low's rounding and 0.25 for its term's; 1 for
// that of the sum r, which may pass 2^24; of the square term, up to 1.7e7 units, 0.5
// each from its coefficient and the polynomial q, 1 from z * z and 1.95 from z; 0.02
// for the 6th power.  4.4 is the most in 4e7 random products.  A weight is 0.978 of its bin's
// or more, so as a share of the largest logit's it is good to 2^-32 (above T = 2^100,
// where cl is denormal, to 2^-25).
//
// A vector instruction in 64 bits takes as long as four in 32 here, and the
// sum of both terms as integers takes the place of a wider type.  NEAR: all products
// down to the last bin's are within kNear.
template <bool NEAR = false>
__host__ __device__ __forceinline__ Weight weigh_finite(float l, const Scale& s) {
#pragma clang fp contract(off)
    constexpr double a = 0.69314718055994530942 / 16.0, unit = 0x1p36;
    constexpr float ah = float(a * unit), al = float(a * unit - double(float(a * unit)));
    const float hi = l * s.ch;
    float y, low, down;
    if (!NEAR && __builtin_fabsf(hi) > kNear && !(hi < s.floor)) {
        double rest;
        down = float(s.top - far_product(l, s, rest));
        y = float(rest);
        low = float(rest - double(y));
    } else {
        const float f = __builtin_rintf(hi);
        y = hi - f;
        low = __builtin_fmaf(l, s.cl, __builtin_fmaf(l, s.ch, -hi));
        down = s.topf - f;
    }
    const float z = y + low;   // of the terms from the 2nd power on
    float q = __builtin_fmaf(float(a * a * a * a * a / 120.0 * unit), z, float(a * a * a * a / 24.0 * unit));
    q = __builtin_fmaf(q, z, float(a * a * a / 6.0 * unit));
    q = __builtin_fmaf(q, z, float(a * a / 2.0 * unit));
    const float p = ah * y;
    float r = __builtin_fmaf(al, y, __builtin_fmaf(ah, y, -p));
    r = __builtin_fmaf(ah, low, r);
    r = __builtin_fmaf(q, z * z, r);
    // -inf is as far down as there is, and so is 0 * inf at T = inf (a NaN).
    return Weight{int(__builtin_fminf(down, float(kRest))), int32_t(p) + int32_t(r)};
}

__host__ __device__ __forceinline__ Weight weigh(float l, const Scale& s) {
    if (s.flat) return Weight{l == s.largest ? 0 : kRest, 0};
    return weigh_finite(l, s);
}

// A key no larger than that of any logit of bin `last` or above: what its bound
// in 64 bits says, with room for the roundings.  0 where that says nothing.
__host__ __device__ __forceinline__ uint32_t key_floor(int last, const Scale& s) {
    const double l = (s.top - double(last) - 0.5) / s.c;
    if (s.flat || last >= kRest || !(__builtin_fabs(l) < 3.0e38)) return 0;
    const uint32_t key = argmax_order(float(l));
    return key > 4 ? key - 4 : 0;
}

// The same from above: no smaller than any key of bin `first` or below.
__host__ __device__ __forceinline__ uint32_t key_ceiling(int first, const Scale& s) {
    const uint32_t most = argmax_order(s.largest);
    const double l = (s.top - double(first) + 0.5) / s.c;
    if (s.flat || !(__builtin_fabs(l) < 3.0e38)) return most;
    const uint32_t key = argmax_order(float(l)) + 4;
    return key < most ? key : most;
}

__host__ __device__ __forceinline__ bool is_near(const Scale& s) { return __builtin_fabsf(s.topf) < kNear - 2.0f * kBins; }

// 2^(-bin / 16), by the bits of bin.
__host__ __device__ __forceinline__ double bin_scale(int bin) {
    double x = bin & 1 ? 0.95760328069857364694 : 1.0;
    x *= bin & 2 ? 0.91700404320467123174 : 1.0;
    x *= bin & 4 ? 0.84089641525371454303 : 1.0;
    x *= bin & 8 ? 0.70710678118654752440 : 1.0;
    return __builtin_ldexp(x, -(bin >> 4));
}

}  // namespace nvg
