// Rows brought to 8 bits, shared by the kernels that write or multiply them (qlinear.hip, block_norm.hip).
//
//   amax = max_k |x[k]|,  scale = amax / 127,  q[k] = rint(127 x[k] / amax)   (ties to even, |q| <= 127)
//
// A row of zeros gets scale 0 and zeros; a row that holds a NaN or an infinity gets scale NaN and zeros, so all of
// its products come out as NaN and no other row's do.
#pragma once
#include <type_traits>

#include "sox_device.h"

typedef int int4v __attribute__((ext_vector_type(4)));
typedef int int16v __attribute__((ext_vector_type(16)));

// The activation of an output stored as T. A NaN (of a row that is not finite) stays one; sox_act's maxima drop it.
template <typename T> SOX_DEV float q_act(float v, int act) {
    if (act == SOX_ACT_NONE || v != v) return v;
    return sizeof(T) == 4 ? sox_act(v, act) : act_fast(v, act);
}

// |v| as bits: they order like the magnitudes, an infinity above every finite value and a NaN above that, so one
// unsigned maximum finds the row's largest magnitude and whether the row is finite
SOX_DEV uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

template <int LANES> SOX_DEV uint32_t wave_max(uint32_t v) {
#pragma unroll
    for (int d = LANES / 2; d; d >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d));
    return v;
}
template <int LANES> SOX_DEV float wave_sum(float v) {
#pragma unroll
    for (int d = LANES / 2; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// The rounding of one row. For 16-bit x (T half_t / bf16_t) 127 x is exact in fp32 and the quotient, correctly rounded
// by one residual step (its reciprocal is), lies on the same side of every half as the exact one: 254 x - (2 j + 1)
// amax is a multiple of x's last place or 0, which keeps a quotient that is no half at least 2^-12 of x's last
// place over amax's away from it, where its rounding error is below 2^-16 of that. So q is the exact rounding,
// whatever computes it; a plain product with 127 / amax puts halves (amax / 2 always is one) on either side. Powers
// of two keep the steps out of the subnormals and of overflow. Full precision x takes the same steps in 64 bits.
template <typename T> struct RowQuant {
    typedef typename std::conditional<sizeof(T) == 4, double, float>::type F;
    F mul, amax, inv;
    float scale;
    SOX_DEV RowQuant make(uint32_t bits) {
        RowQuant r;
        const float a = __uint_as_float(bits);
        const bool some = bits != 0 && bits < 0x7f800000u;
        r.scale = bits < 0x7f800000u ? a / 127.0f : __uint_as_float(0x7fc00000u);
        if constexpr (sizeof(T) == 4) {
            r.mul = some ? 127.0 : 0.0;
            r.amax = some ? (double)a : 1.0;
            r.inv = 1.0 / r.amax;
        } else {
            const float s = a < 0x1p-60f ? 0x1p64f : a > 0x1p60f ? 0x1p-64f : 1.0f;
            r.mul = some ? 127.0f * s : 0.0f;
            r.amax = some ? a * s : 1.0f;
            r.inv = 1.0f / r.amax;
        }
        return r;
    }
    SOX_DEV int q(float x, const RowQuant& r) {
        x = r.mul != 0 ? x : 0.0f;  // (one that is not finite would stay a NaN)
        if constexpr (sizeof(T) == 4) {
            const double t = (double)x * r.mul, v = t * r.inv;
            return (int)rint(__builtin_fma(__builtin_fma(-v, r.amax, t), r.inv, v));
        } else {
            const float t = x * r.mul, v = t * r.inv;
            return (int)rintf(__builtin_fmaf(__builtin_fmaf(-v, r.amax, t), r.inv, v));
        }
    }
};
