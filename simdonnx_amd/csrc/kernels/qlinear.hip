// The 8-bit product's other kernels: floating rows to 8 bits (sox_qrows_*) and products of few rows (sox_qfew_*).
#include "qgemm_ring.h"

// E consecutive values of a row from column k on, zeros past column K
template <typename T, int E> SOX_DEV void load_values(const T* __restrict__ row, int k, int K, bool vec, float (&v)[E]) {
    constexpr int V = 16 / sizeof(T);
    static_assert(E % V == 0, "whole 16-byte chunks");
    typedef vec_t<T, V> TV;
    if (vec && k + E <= K) {
#pragma unroll
        for (int c = 0; c < E / V; c++) {
            const TV t = *(const TV*)(row + k + c * V);
#pragma unroll
            for (int e = 0; e < V; e++) v[c * V + e] = (float)t[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = k + e < K ? (float)row[k + e] : 0.0f;
    }
}

// ---- rows to 8 bits ----
// TPR threads per row (a wave, or the workgroup for long rows). A thread keeps its first CH chunks of 16 bytes in
// registers between the maximum and the rounding; what is past them (rows of more than CH * TPR * 16 bytes) is read
// again, from L2. One read of x and one write of q: bound by memory.
template <typename T, int TPR> SOX_DEV void qrows_body(const sox_qrows_args& p) {
    constexpr int E = 16 / sizeof(T), CH = 4, RPW = 256 / TPR;
    __shared__ uint32_t wmax[4];
    const int t = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * RPW + threadIdx.x / TPR;
    if (row >= p.rows) return;  // (whole waves; with the workgroup per row the grid has no such row)
    const T* x = (const T*)p.x + row * p.ldx;
    int8_t* q = p.q + row * p.ldq;
    const int chunks = ((p.k + 15) / 16 * 16) / E;
    float v[CH][E];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < CH; j++)
        if (t + j * TPR < chunks) load_values<T, E>(x, (t + j * TPR) * E, p.k, p.vec, v[j]);
#pragma unroll
    for (int j = 0; j < CH; j++)
        if (t + j * TPR < chunks)
#pragma unroll
            for (int e = 0; e < E; e++) m = max(m, abs_bits(v[j][e]));
    for (int c = t + CH * TPR; c < chunks; c += TPR) {
        float u[E];
        load_values<T, E>(x, c * E, p.k, p.vec, u);
#pragma unroll
        for (int e = 0; e < E; e++) m = max(m, abs_bits(u[e]));
    }
    m = wave_max(m);
    if constexpr (TPR == 256) {
        if ((threadIdx.x & 63) == 0) wmax[threadIdx.x >> 6] = m;
        __syncthreads();
        m = max(max(wmax[0], wmax[1]), max(wmax[2], wmax[3]));
    }
    typedef RowQuant<T> Q;
    const Q rq = Q::make(m);
    auto put = [&](int c, const float (&u)[E]) {
        uint32_t w[E / 4];
#pragma unroll
        for (int i = 0; i < E / 4; i++) w[i] = Q::q4(&u[4 * i], rq);
        if constexpr (E == 8)
            *(uint2*)(q + c * 8) = make_uint2(w[0], w[1]);
        else
            *(uint32_t*)(q + c * 4) = w[0];
    };
#pragma unroll
    for (int j = 0; j < CH; j++)
        if (t + j * TPR < chunks) put(t + j * TPR, v[j]);
    for (int c = t + CH * TPR; c < chunks; c += TPR) {
        float u[E];
        load_values<T, E>(x, c * E, p.k, p.vec, u);
        put(c, u);
    }
    if (t == 0) p.scale[row] = rq.scale;
}

#define SOX_QROWS(NAME, T)                                                                                               \
    extern "C" __global__ void __launch_bounds__(256) sox_qrows_##NAME(sox_qrows_args p) { qrows_body<T, 64>(p); }      \
    extern "C" __global__ void __launch_bounds__(256) sox_qrows_##NAME##_wide(sox_qrows_args p) { qrows_body<T, 256>(p); }
SOX_QROWS(f16, half_t)
SOX_QROWS(bf16, bf16_t)
SOX_QROWS(f32, float)

// ---- products of few rows ----
// Up to 16 * RB rows: the weights are read once and nothing else is worth counting, so a workgroup takes 16 columns
// of all rows and its waves split K. v_mfma_i32_16x16x64_i8, W the row operand: lane l multiplies k 16 (l / 16) .. + 15
// of a 64-deep step for column l % 16 and row l % 16. Both operands go straight from memory to registers: a W fragment
// is four 256-byte pieces of two packed blocks, a row fragment 16 consecutive values of a row. A wave's S steps are
// all in flight before the first is used. The waves' int32 sums meet in LDS.
// FUSED: the rows are floating ones, of which a wave brings its own steps' values to 8 bits in registers once the row
// maxima of all waves have met in LDS; one launch then does a token's whole product. Every workgroup repeats that
// rounding, which hides behind the weights' loads; K is at most 64 S * waves.
template <typename T, bool FUSED, int S, int RB> SOX_DEV void qfew_body(const sox_qgemm_args& p) {
    static_assert(!FUSED || RB == 1, "16 floating rows at most");
    constexpr int WMAX = FUSED ? 16 : 8;
    __shared__ uint32_t wmax[16][16];
    __shared__ float xscale[16];
    __shared__ int red[WMAX][RB][16 * 17];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int r16 = lane & 15, kq = lane >> 4;
    const int n0 = blockIdx.x * 16;
    const int steps = (p.k + 63) / 64;
    const int8_t* wcol = p.w + (int64_t)(n0 / 32) * p.kb * 1024 + (n0 % 32 + r16) * 16 + (kq >> 1) * 1024 + (kq & 1) * 512;
    int4v acc[RB];
#pragma unroll
    for (int b = 0; b < RB; b++) acc[b] = (int4v)0;
    for (int base = wave * S; base < steps; base += waves * S) {
        int4v wf[S], xf[S][RB];
#pragma unroll
        for (int s = 0; s < S; s++)  // (kb is even: a step's two blocks exist; steps past the last are not loaded)
            wf[s] = base + s < steps ? *(const int4v*)(wcol + (int64_t)(base + s) * 2048) : (int4v)0;
        if constexpr (FUSED) {
            float v[S][16];
            const T* x = (const T*)p.x + min(r16, p.m - 1) * p.ldx;
#pragma unroll
            for (int s = 0; s < S; s++) load_values<T, 16>(x, (base + s) * 64 + kq * 16, p.k, p.vec & 2, v[s]);
            uint32_t m = 0;
#pragma unroll
            for (int s = 0; s < S; s++)
#pragma unroll
                for (int e = 0; e < 16; e++) m = max(m, abs_bits(v[s][e]));
            m = max(m, (uint32_t)__shfl_xor((int)m, 16));
            m = max(m, (uint32_t)__shfl_xor((int)m, 32));
            if (lane < 16) wmax[wave][lane] = m;
            __syncthreads();  // (one round: every wave has steps, the launcher sees to it)
            m = 0;
            for (int w = 0; w < waves; w++) m = max(m, wmax[w][r16]);
            typedef RowQuant<T> Q;
            const Q rq = Q::make(m);
            if (wave == 0 && lane < 16) xscale[lane] = rq.scale;
#pragma unroll
            for (int s = 0; s < S; s++)
#pragma unroll
                for (int c = 0; c < 4; c++)
                    xf[s][0][c] = (int)Q::q4(&v[s][4 * c], rq);
        } else {
#pragma unroll
            for (int b = 0; b < RB; b++) {
                const int8_t* a = p.a + min(b * 16 + r16, p.m - 1) * p.lda + kq * 16;
#pragma unroll
                for (int s = 0; s < S; s++)
                    xf[s][b] = (base + s) * 64 + kq * 16 < p.k16 ? *(const int4v*)(a + (int64_t)(base + s) * 64) : (int4v)0;
            }
        }
#pragma unroll
        for (int s = 0; s < S; s++)
#pragma unroll
            for (int b = 0; b < RB; b++) acc[b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[s], xf[s][b], acc[b], 0, 0, 0);
    }
#pragma unroll
    for (int b = 0; b < RB; b++)
#pragma unroll
        for (int e = 0; e < 4; e++) red[wave][b][(4 * kq + e) * 17 + r16] = acc[b][e];
    __syncthreads();
    for (int o = threadIdx.x; o < RB * 256; o += blockDim.x) {
        const int c = o % 16, r = o / 16 % 16, b = o / 256, row = b * 16 + r, n = n0 + c;
        if (row >= p.m || n >= p.n) continue;
        int sum = 0;
        for (int w = 0; w < waves; w++) sum += red[w][b][c * 17 + r];
        float v = __builtin_fmaf((float)sum * p.ws[n], FUSED ? xscale[r] : p.xs[row], p.bias[n]);
        if (p.add) v += (float)((const T*)p.add)[row * p.ldr + n];
        ((T*)p.y)[row * p.ldy + n] = (T)q_out<T, Q_ACT_ANY>(v, p.act);
    }
}

#define SOX_QFEW(NAME, T, S)                                                                                                   \
    extern "C" __global__ void __launch_bounds__(1024) sox_qfewx_##NAME##_s##S(sox_qgemm_args p) { qfew_body<T, true, S, 1>(p); }
#define SOX_QFEW_RB(NAME, T, RB)                                                                                               \
    extern "C" __global__ void __launch_bounds__(512) sox_qfew_##NAME##_r##RB(sox_qgemm_args p) { qfew_body<T, false, 8 / RB, RB>(p); }
#define SOX_QFEW_ALL(NAME, T) \
    SOX_QFEW(NAME, T, 1) SOX_QFEW(NAME, T, 2) SOX_QFEW(NAME, T, 4) SOX_QFEW_RB(NAME, T, 1) SOX_QFEW_RB(NAME, T, 2) SOX_QFEW_RB(NAME, T, 4)
SOX_QFEW_ALL(f16, half_t)
SOX_QFEW_ALL(bf16, bf16_t)
SOX_QFEW_ALL(f32, float)
