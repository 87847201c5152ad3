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
        // (v + 3 is exact near its zero, where v / 6 + 1 / 2 would be left with the quotient's rounding)
        const float hard = fminf(fmaxf((v + 3.0f) * (1.0f / 6.0f), 0.0f), 1.0f);
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

// Sum and maximum over a wave or its halves by DPP moves, in the order of a tree (lanes 1, 2, 4, 8, 16, 32 apart), given to
// every lane:
// six additions of a few cycles each where lane shuffles through LDS take about 60.
template <int CTRL, int ROWS> SOX_DEV float dpp_moved(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xf, true));
}
template <int CTRL, int ROWS> SOX_DEV uint32_t dpp_moved(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, true);
}
template <int LANES, class V, class F> SOX_DEV V lanes_fold(V v, F&& f) {
    static_assert(LANES == 32 || LANES == 64, "half a wave or a wave");
    v = f(v, dpp_moved<0x111, 0xf>(v));  // row_shr 1, 2, 4, 8: lane 15 of each row of 16 holds the row's
    v = f(v, dpp_moved<0x112, 0xf>(v));
    v = f(v, dpp_moved<0x114, 0xf>(v));
    v = f(v, dpp_moved<0x118, 0xf>(v));
    v = f(v, dpp_moved<0x142, 0xa>(v));  // row_bcast 15 into rows 1 and 3: lanes 31 and 63 hold the halves'
    if constexpr (LANES == 64) v = f(v, dpp_moved<0x143, 0xc>(v));  // row_bcast 31 into rows 2 and 3: lane 63
    const int top = __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63);
    if constexpr (LANES == 64) return __builtin_bit_cast(V, top);
    const int low = __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 31);
    return __builtin_bit_cast(V, (threadIdx.x & 32) ? top : low);
}
template <int LANES = 64> SOX_DEV float wave_sum(float v) {
    return lanes_fold<LANES>(v, [](float a, float b) { return a + b; });
}
template <int LANES = 64> SOX_DEV uint32_t wave_max(uint32_t v) {
    return lanes_fold<LANES>(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}

// Maximum over each row of 16 lanes, given to its lanes
SOX_DEV uint32_t row16_max(uint32_t v) {
    v = max(v, dpp_moved<0x111, 0xf>(v));
    v = max(v, dpp_moved<0x112, 0xf>(v));
    v = max(v, dpp_moved<0x114, 0xf>(v));
    v = max(v, dpp_moved<0x118, 0xf>(v));
    return dpp_moved<0x15f, 0xf>(v);  // row_newbcast 15
}

// 16 bytes of a row, which may stand on any element: the compiler takes such a vector with one instruction all the same. (By
// single elements, 8192 x 2304 norms of bf16 rows off 16-byte boundaries took 109 us, so 45,
// on boundaries 41.)
template <typename T> struct Chunk16 {
    typedef vec_t<T, 16 / sizeof(T)> V;
    typedef V At __attribute__((aligned(sizeof(T))));
};

// E consecutive values of a row as they stand in memory, zeros past its end.
template <typename T, int E> struct RawValues {
    static constexpr int V = 16 / sizeof(T);
    static_assert(E % V == 0, "whole 16-byte chunks");
    typedef vec_t<T, V> TV;
    TV r[E / V];
    // from column k on of a row of K
    __device__ __forceinline__ void load(const T* __restrict__ row, int k, int K) {
        if (k + E <= K) {
#pragma unroll
            for (int c = 0; c < E / V; c++) r[c] = *(const typename Chunk16<T>::At*)(row + k + c * V);
        } else {
#pragma unroll
            for (int c = 0; c < E / V; c++)
#pragma unroll
                for (int e = 0; e < V; e++) r[c][e] = k + c * V + e < K ? row[k + c * V + e] : (T)0.0f;
        }
    }
    __device__ __forceinline__ float operator[](int i) const { return (float)r[i / V][i % V]; }
};

// The largest magnitude of a row's values, as an unsigned number: two 16-bit values to an instruction. row_bits gives the
// fp32 bits of |v| of the one that a row's lanes agreed on.
template <typename T> struct AbsMax {
    typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));
    ushort2v m16 = {0, 0};
    uint32_t m32 = 0;
    template <int E> __device__ __forceinline__ void add(const RawValues<T, E>& v) {
        typedef vec_t<uint32_t, 4> U4;
#pragma unroll
        for (int c = 0; c < E / RawValues<T, E>::V; c++) {
            const U4 w = __builtin_bit_cast(U4, v.r[c]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if constexpr (sizeof(T) == 2)
                    m16 = __builtin_elementwise_max(m16, __builtin_bit_cast(ushort2v, w[i] & 0x7fff7fffu));
                else
                    m32 = max(m32, w[i] & 0x7fffffffu);
            }
        }
    }
    __device__ __forceinline__ uint32_t lane() const { return sizeof(T) == 2 ? (uint32_t)max(m16[0], m16[1]) : m32; }
    SOX_DEV uint32_t row_bits(uint32_t folded) {
        if constexpr (sizeof(T) == 4)
            return folded;
        else
            return abs_bits((float)__builtin_bit_cast(T, (unsigned short)folded));
    }
};

// The rounding of one row. For 16-bit x (T half_t / bf16_t) 127 x is exact in fp32 and the quotient, correctly rounded
// by one residual step (its reciprocal is), lies on the same side of every half as the exact one: 254 x - (2 j + 1)
// amax is a multiple of x's last place or 0, which keeps a quotient that is no half at least 2^-12 of x's last
// place over amax's away from it, where its rounding error is below 2^-16 of that. So q is the exact rounding,
// whatever computes it; a plain product with 127 / amax puts halves (amax / 2 always is one) on either side. Powers
// of two keep the steps out of the subnormals and of overflow. Full precision x takes the same steps in 64 bits.
// The integer comes from the sum with 3 * 2^22, whose last byte is it (ties to even, as the sum rounds).
template <typename T> struct RowQuant {
    typedef typename std::conditional<sizeof(T) == 4, double, float>::type F;
    F mul, amax, inv;
    float scale;
    uint32_t keep;  // 0 for a row that is not finite: its values give zeros
    SOX_DEV RowQuant make(uint32_t bits) {
        RowQuant r;
        const float a = __uint_as_float(bits);
        const bool some = bits != 0 && bits < 0x7f800000u;
        r.scale = bits < 0x7f800000u ? a / 127.0f : __uint_as_float(0x7fc00000u);
        r.keep = some ? ~0u : 0;
        if constexpr (sizeof(T) == 4) {
            r.mul = 127.0;
            r.amax = some ? (double)a : 1.0;
            r.inv = 1.0 / r.amax;
        } else {
            const float s = a < 0x1p-60f ? 0x1p64f : a > 0x1p60f ? 0x1p-64f : 1.0f;
            r.mul = 127.0f * s;
            r.amax = some ? a * s : 1.0f;
            r.inv = 1.0f / r.amax;
        }
        return r;
    }
    // a value's integer in the last byte
    SOX_DEV uint32_t low(float x, const RowQuant& r) {
        float v;
        if constexpr (sizeof(T) == 4) {
            const double t = (double)x * r.mul, d = t * r.inv;
            v = (float)rint(__builtin_fma(__builtin_fma(-d, r.amax, t), r.inv, d));
        } else {
            const float t = x * r.mul;
            v = t * r.inv;
            v = __builtin_fmaf(__builtin_fmaf(-v, r.amax, t), r.inv, v);
        }
        return __float_as_uint(v + 12582912.0f);
    }
    SOX_DEV int8_t q(float x, const RowQuant& r) { return (int8_t)(low(x, r) & r.keep); }
    // four consecutive values, a byte each
    SOX_DEV uint32_t q4(float x0, float x1, float x2, float x3, const RowQuant& r) {
        const uint32_t a = __builtin_amdgcn_perm(low(x1, r), low(x0, r), 0x0c0c0400), b = __builtin_amdgcn_perm(low(x3, r), low(x2, r), 0x04000c0c);
        return (a | b) & r.keep;
    }
    template <int E> SOX_DEV uint32_t q4(const RawValues<T, E>& v, int i, const RowQuant& r) {
        return q4(v[i], v[i + 1], v[i + 2], v[i + 3], r);
    }
};
