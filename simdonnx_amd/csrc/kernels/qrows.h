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

// The activation of an output stored as T: ACT as known at compile time, Q_ACT_GATES for the runtime one of sigmoid,
// hardswish and swish, Q_ACT_ANY for any runtime one, by branches. A NaN (of a row that
// is not finite) stays one; sox_act's maxima would drop it.
enum { Q_ACT_ANY = -1, Q_ACT_GATES = -2 };
template <typename T, int ACT> SOX_DEV float q_out(float v, int act = 0) {
    if constexpr (ACT == SOX_ACT_RELU) {
        return __builtin_elementwise_maximum(v, 0.0f);
    } else if constexpr (ACT == SOX_ACT_GELU) {
        if constexpr (sizeof(T) == 2) return gelu_fast(v);  // (these two keep a NaN by themselves)
        const float g = sox_gelu(v);
        return v != v ? v : g;
    } else if constexpr (ACT == Q_ACT_GATES) {
        const float hard = fminf(fmaxf(__builtin_fmaf(v, 1.0f / 6.0f, 0.5f), 0.0f), 1.0f);
        const float gate = act == SOX_ACT_HARDSWISH ? hard : sox_sigmoid(v), r = act == SOX_ACT_SIGMOID ? gate : v * gate;
        return v != v ? v : r;
    } else {
        static_assert(ACT == Q_ACT_ANY, "activation");
        if (act == SOX_ACT_NONE) return v;
        if (act == SOX_ACT_RELU) return q_out<T, SOX_ACT_RELU>(v);
        if (act == SOX_ACT_GELU) return q_out<T, SOX_ACT_GELU>(v);
        return q_out<T, Q_ACT_GATES>(v, act);
    }
}

// |v| as bits: they order like the magnitudes, an infinity above every finite value and a NaN above that, so one
// unsigned maximum finds the row's largest magnitude and whether the row is finite
SOX_DEV uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Sum and maximum over a wave by DPP moves, in the order of a tree (lanes 1, 2, 4, 8, 16, 32 apart), given to every lane:
// six additions of a few cycles each where lane shuffles through LDS take about 60.
template <int CTRL, int ROWS> SOX_DEV float dpp_moved(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xf, true));
}
template <int CTRL, int ROWS> SOX_DEV uint32_t dpp_moved(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, true);
}
template <class V, class F> SOX_DEV V wave_fold(V v, F&& f) {
    v = f(v, dpp_moved<0x111, 0xf>(v));  // row_shr 1, 2, 4, 8: lane 15 of each row of 16 holds the row's
    v = f(v, dpp_moved<0x112, 0xf>(v));
    v = f(v, dpp_moved<0x114, 0xf>(v));
    v = f(v, dpp_moved<0x118, 0xf>(v));
    v = f(v, dpp_moved<0x142, 0xa>(v));  // row_bcast 15 into rows 1 and 3, row_bcast 31 into rows 2 and 3
    v = f(v, dpp_moved<0x143, 0xc>(v));
    return v;  // lane 63
}
SOX_DEV float wave_sum(float v) {
    v = wave_fold(v, [](float a, float b) { return a + b; });
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
SOX_DEV uint32_t wave_max(uint32_t v) {
    v = wave_fold(v, [](uint32_t a, uint32_t b) { return max(a, b); });
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
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
    // four consecutive values, a byte each
    SOX_DEV uint32_t q4(const float* x, const RowQuant& r) {
        uint32_t b[4];
#pragma unroll
        for (int e = 0; e < 4; e++) b[e] = (uint32_t)q(x[e], r);
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400), __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400),
                                     0x05040100);
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
