// The norms before and after a transformer block, with its gate and residual scale, in one pass over the rows:
//   h = res_scale * residual + act(gate) * (post(x) * scale),   y = pre(h)
//   rms(v) = v / sqrt(mean(v^2) + eps) * gamma,   layer(v) = (v - mean v) / sqrt(mean((v - mean v)^2) + eps) * gamma + beta
// y leaves in the storage type or as 8-bit rows with their scales for the product that reads them (qlinear.hip).
//
// Bound by memory: x, residual and gate are read once, h and y written once, and a row stays in registers in between.
// All sums and norms in fp32, a variance as the mean square about the mean (a second sum over the registers, so a large
// mean costs no digits); y is computed from h as summed in fp32, not from its rounded copy. TPR threads share a row; a
// workgroup walks its rows with the parameter vectors in registers, since reading up to four fp32 vectors per row again
// would move as much from L2 as the 16-bit rows do from memory.
#include "qrows.h"

enum { NORM_NONE = 0, NORM_RMS = 1, NORM_LAYER = 2 };

// CH chunks of E values per thread; VEC: chunk j of thread t is columns (j TPR + t) E .. + E - 1 as one 16-byte access
// (rows on 16-byte boundaries, c a multiple of E), else value e of it is column (j E + e) TPR + t on its own
template <typename T, int TPR, int CH, bool VEC> struct Row {
    static constexpr int E = 16 / sizeof(T), N = CH * E;
    typedef vec_t<T, E> TV;
    SOX_DEV int col(int t, int i) { return VEC ? (i / E * TPR + t) * E + i % E : i * TPR + t; }
    SOX_DEV void load(const T* __restrict__ p, int t, int c, float (&v)[N]) {
        if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < CH; j++) {
                const int k = (j * TPR + t) * E;
                const TV x = k < c ? *(const TV*)(p + k) : TV{};
#pragma unroll
                for (int e = 0; e < E; e++) v[j * E + e] = (float)x[e];
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) v[i] = col(t, i) < c ? (float)p[col(t, i)] : 0.0f;
        }
    }
    SOX_DEV void store(T* __restrict__ p, int t, int c, const float (&v)[N]) {
        if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < CH; j++) {
                const int k = (j * TPR + t) * E;
                TV x;
#pragma unroll
                for (int e = 0; e < E; e++) x[e] = (T)v[j * E + e];
                if (k < c) *(TV*)(p + k) = x;
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i++)
                if (col(t, i) < c) p[col(t, i)] = (T)v[i];
        }
    }
    SOX_DEV void param(const float* __restrict__ p, int t, int c, float (&v)[N]) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = col(t, i) < c ? p[col(t, i)] : 0.0f;
    }
    // columns c .. round_up(c, 16) - 1 hold zeros (v is 0 there)
    SOX_DEV void store8(int8_t* __restrict__ p, int t, int c, const float (&v)[N], const RowQuant<half_t>& rq) {
        const int c16 = (c + 15) & ~15;
        if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < CH; j++) {
                const int k = (j * TPR + t) * E;
#pragma unroll
                for (int w = 0; w < E / 4; w++) {
                    uint32_t b = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) b |= (uint32_t)(RowQuant<half_t>::q(v[j * E + 4 * w + e], rq) & 255) << (8 * e);
                    if (k + 4 * w < c16) *(uint32_t*)(p + k + 4 * w) = b;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i++)
                if (col(t, i) < c16) p[col(t, i)] = (int8_t)RowQuant<half_t>::q(v[i], rq);
        }
    }
};

// Sum (maximum) over the TPR threads of a row. Each reduction over several waves has an LDS row of its own, two sets
// in turn per row walked, so one barrier per reduction is enough: a set is written again only after the barriers of
// the row in between.
template <int TPR> SOX_DEV float row_sum(float v, float* lds) {
    v = wave_sum<64>(v);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) v += lds[w];
    }
    return v;
}
template <int TPR> SOX_DEV uint32_t row_max(uint32_t v, uint32_t* lds) {
    v = wave_max<64>(v);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int w = 0; w < W; w++) v = max(v, lds[w]);
    }
    return v;
}

// KEEP: the parameter vectors stay in registers for all rows (where they fit; else they come from L2 row by row)
template <typename T, int TPR, int CH, bool VEC, bool KEEP> SOX_DEV void bnorm_body(const sox_bnorm_args& p) {
    typedef Row<T, TPR, CH, VEC> R;
    constexpr int N = R::N, BLOCK = TPR < 256 ? 256 : TPR, RPB = BLOCK / TPR;
    __shared__ float lds[2][5][BLOCK / 64];
    const int t = threadIdx.x % TPR, c = p.c;
    const float inv_c = 1.0f / (float)c;
    constexpr int NK = KEEP ? N : 1;
    float pg[NK], pb[NK], g[NK], b[NK];
    if constexpr (KEEP) {
        R::param(p.pg, t, c, pg);
        R::param(p.pb, t, c, pb);
        R::param(p.g, t, c, g);
        R::param(p.b, t, c, b);
    }
    // (the empty asm: without it the loads are moved out of the row loop, into registers that are not there)
    auto fresh = [&](const float* vec) {
        if constexpr (!KEEP) asm volatile("" : "+s"(vec));
        return vec;
    };
    auto at = [&](const float* vec, const float (&kept)[NK], int i) {
        if constexpr (KEEP) return kept[i];
        return R::col(t, i) < c ? vec[R::col(t, i)] : 0.0f;
    };
    auto norm = [&](float (&v)[N], int kind, float eps, const float* gp, const float (&ga)[NK], const float* bp,
                    const float (&be)[NK], float* l0, float* l1) __attribute__((always_inline)) {
        float s = 0.0f;
        if (kind == NORM_LAYER) {
#pragma unroll
            for (int i = 0; i < N; i++) s += v[i];
            const float mean = row_sum<TPR>(s, l0) * inv_c;
#pragma unroll
            for (int i = 0; i < N; i++) v[i] = R::col(t, i) < c ? v[i] - mean : 0.0f;
            s = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < N; i++) s = __builtin_fmaf(v[i], v[i], s);
        const float r = 1.0f / sqrtf(row_sum<TPR>(s, l1) * inv_c + eps);
#pragma unroll
        for (int i = 0; i < N; i++) {
            v[i] = __builtin_fmaf(v[i] * r, at(gp, ga, i), at(bp, be, i));
            if constexpr (!KEEP)
                if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // a few parameters at a time
        }
    };
    int set = 0;
    for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; row < p.rows; row += (int64_t)gridDim.x * RPB, set ^= 1) {
        float h[N], a[N];
        if (p.x) {
            R::load((const T*)p.x + row * p.ldx, t, c, a);
            float ga[KEEP ? N : 1];
            // all of a row's loads go out together where registers allow
            if constexpr (KEEP) {
                if (p.gate) R::load((const T*)p.gate + row / p.gate_group * p.ldg, t, c, ga);
                if (p.residual) R::load((const T*)p.residual + row * p.ldr, t, c, h);
            }
            if (p.post != NORM_NONE) {
                norm(a, p.post, p.post_eps, fresh(p.pg), pg, fresh(p.pb), pb, lds[set][0], lds[set][1]);
            } else {
                const float* sc = fresh(p.pg);
#pragma unroll
                for (int i = 0; i < N; i++) a[i] *= at(sc, pg, i);
            }
            if constexpr (KEEP) {
                if (p.gate)
#pragma unroll
                    for (int i = 0; i < N; i++) a[i] *= q_act<float>(ga[i], p.gate_act);
#pragma unroll
                for (int i = 0; i < N; i++) h[i] = p.residual ? __builtin_fmaf(p.res_scale, h[i], a[i]) : a[i];
            } else {
                __builtin_amdgcn_sched_barrier(0);
                if (p.gate) {
                    R::load((const T*)p.gate + row / p.gate_group * p.ldg, t, c, h);
#pragma unroll
                    for (int i = 0; i < N; i++) a[i] *= q_act<float>(h[i], p.gate_act);
                }
                __builtin_amdgcn_sched_barrier(0);
                if (p.residual) R::load((const T*)p.residual + row * p.ldr, t, c, h);
#pragma unroll
                for (int i = 0; i < N; i++) h[i] = p.residual ? __builtin_fmaf(p.res_scale, h[i], a[i]) : a[i];
            }
        } else {
            R::load((const T*)p.residual + row * p.ldr, t, c, h);
#pragma unroll
            for (int i = 0; i < N; i++) h[i] *= p.res_scale;
        }
        if (p.h) R::store((T*)p.h + row * p.ldh, t, c, h);
        if (!p.y && !p.q) continue;
        if (p.pre != NORM_NONE) norm(h, p.pre, p.pre_eps, fresh(p.g), g, fresh(p.b), b, lds[set][2], lds[set][3]);
        if (p.y) R::store((T*)p.y + row * p.ldy, t, c, h);
        if (p.q) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < N; i++) m = max(m, abs_bits(h[i]));
            const RowQuant<half_t> rq = RowQuant<half_t>::make(row_max<TPR>(m, (uint32_t*)lds[set][4]));
            R::store8(p.q + row * p.ldq, t, c, h, rq);
            if (t == 0) p.qs[row] = rq.scale;
        }
    }
}

#define SOX_BNORM_V(NAME, T, TPR, CH, SUFFIX, VEC, KEEP)                                                                  \
    extern "C" __global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) sox_bnorm_##NAME##_t##TPR##c##CH##SUFFIX(sox_bnorm_args p) { \
        bnorm_body<T, TPR, CH, VEC, KEEP>(p);                                                                               \
    }
#define SOX_BNORM(NAME, T, TPR, CH, KEEP) \
    SOX_BNORM_V(NAME, T, TPR, CH, v, true, KEEP) SOX_BNORM_V(NAME, T, TPR, CH, s, false, KEEP)
// threads of a row and chunks of a thread: 16-bit rows of up to 512, 1024, 2048, 4096, 8192, 16384 columns ...
#define SOX_BNORM_16(NAME, T)                                                                                             \
    SOX_BNORM(NAME, T, 64, 1, true) SOX_BNORM(NAME, T, 64, 2, true) SOX_BNORM(NAME, T, 256, 1, true)                      \
    SOX_BNORM(NAME, T, 256, 2, true) SOX_BNORM(NAME, T, 1024, 1, true) SOX_BNORM(NAME, T, 512, 4, false)
SOX_BNORM_16(f16, half_t)
SOX_BNORM_16(bf16, bf16_t)
// ... and the same in fp32, twice the chunks
SOX_BNORM(f32, float, 64, 2, true) SOX_BNORM(f32, float, 64, 4, true) SOX_BNORM(f32, float, 256, 2, true)
SOX_BNORM(f32, float, 256, 4, true) SOX_BNORM(f32, float, 1024, 2, true) SOX_BNORM(f32, float, 512, 8, false)
