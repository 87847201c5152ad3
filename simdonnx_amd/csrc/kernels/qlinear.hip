// The 8-bit product's other kernels (the ring of qgemm_ring.h aside): floating rows to 8 bits (sox_qrows_*), products of few
// rows, 8-bit (sox_qfew_*) or floating (sox_qfewx_*), and of a moderate number of floating rows (sox_qpanel_*).
#include "qgemm_ring.h"

// ---- rows to 8 bits ----
// TPR threads per row (half a wave, a wave, or the workgroup for long rows). A thread keeps its first CH chunks of 16 bytes in
// registers between the maximum and the rounding; what is past them (rows of more than CH * TPR * 16 bytes) is read
// again, from L2. One read of x and one write of q: bound by memory, 8192 x 1024 fp16 in 10.4 us with its launch.
template <typename T, int TPR> SOX_DEV void qrows_body(const sox_qrows_args& p) {
    constexpr int E = 16 / sizeof(T), CH = 4, RPW = 256 / TPR;
    typedef RawValues<T, E> Chunk;
    typedef RowQuant<T> Q;
    __shared__ uint32_t wmax[4];
    const int t = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * RPW + threadIdx.x / TPR;
    if (TPR < 256 && row >= p.rows) return;  // (with the workgroup per row the grid has no such row)
    const T* x = (const T*)p.x + row * p.ldx;
    int8_t* q = p.q + row * p.ldq;
    const int chunks = ((p.k + 15) / 16 * 16) / E;
    Chunk v[CH];
    AbsMax<T> top;
#pragma unroll
    for (int j = 0; j < CH; j++)
        if (t + j * TPR < chunks) v[j].load(x, (t + j * TPR) * E, p.k);
#pragma unroll
    for (int j = 0; j < CH; j++)
        if (t + j * TPR < chunks) top.add(v[j]);
    for (int c = t + CH * TPR; c < chunks; c += TPR) {
        Chunk u;
        u.load(x, c * E, p.k);
        top.add(u);
    }
    uint32_t m = wave_max<TPR == 32 ? 32 : 64>(top.lane());
    if constexpr (TPR == 256) {
        if ((threadIdx.x & 63) == 0) wmax[threadIdx.x >> 6] = m;
        __syncthreads();
        m = max(max(wmax[0], wmax[1]), max(wmax[2], wmax[3]));
    }
    const Q rq = Q::make(AbsMax<T>::row_bits(m));
    auto put = [&](int c, const Chunk& u) {
        if constexpr (E == 8)
            *(uint2*)(q + c * 8) = make_uint2(Q::q4(u, 0, rq), Q::q4(u, 4, rq));
        else
            *(uint32_t*)(q + c * 4) = Q::q4(u, 0, rq);
    };
#pragma unroll
    for (int j = 0; j < CH; j++)
        if (t + j * TPR < chunks) put(t + j * TPR, v[j]);
    for (int c = t + CH * TPR; c < chunks; c += TPR) {
        Chunk u;
        u.load(x, c * E, p.k);
        put(c, u);
    }
    if (t == 0) p.scale[row] = rq.scale;
}

#define SOX_QROWS_T(NAME, T, TPR) \
    extern "C" __global__ void __launch_bounds__(256) sox_qrows_##NAME##_t##TPR(sox_qrows_args p) { qrows_body<T, TPR>(p); }
#define SOX_QROWS(NAME, T) SOX_QROWS_T(NAME, T, 32) SOX_QROWS_T(NAME, T, 64) SOX_QROWS_T(NAME, T, 256)
SOX_QROWS(f16, half_t)
SOX_QROWS(bf16, bf16_t)
SOX_QROWS(f32, float)

// ---- products of few rows ----
// Up to 16 * RB rows: the weights are read once and nothing else is worth counting, so a workgroup takes 16 columns
// of all rows and its waves split K. v_mfma_i32_16x16x64_i8, W the row operand: lane l multiplies k 16 (l / 16) .. + 15
// of a 64-deep step for column l % 16 and row l % 16. A W fragment goes straight from memory to registers, four 256-byte
// pieces of two packed blocks, and a wave's S steps are all in flight before the first is used. The waves' int32 sums
// meet in LDS. Bound by one trip to memory and the sums' meeting: 64 x 1024 -> 8192 6.9 us, 64 x 4096 -> 4096 10.8.
SOX_DEV const int8_t* few_weights(const sox_qgemm_args& p, int n0) {  // of step 0; a step is 2 KiB on (kb is even)
    const int lane = threadIdx.x & 63, r16 = lane & 15, kq = lane >> 4;
    return p.w + (int64_t)(n0 / 32) * p.kb * 1024 + (n0 % 32 + r16) * 16 + (kq >> 1) * 1024 + (kq & 1) * 512;
}
// the sums of `waves` waves to outputs; red[w][b] holds column c of row r of 16 rows b at c * 17 + r
template <typename T, int RB, class X>
SOX_DEV void few_outputs(const sox_qgemm_args& p, const int (*red)[RB][16 * 17], int waves, int n0, X&& row_scale) {
    for (int o = threadIdx.x; o < RB * 256; o += blockDim.x) {
        const int c = o % 16, r = o / 16 % 16, b = o / 256, row = b * 16 + r, n = n0 + c;
        if (row >= p.m || n >= p.n) continue;
        int sum = 0;
        for (int w = 0; w < waves; w++) sum += red[w][b][c * 17 + r];
        float v = __builtin_fmaf((float)sum * p.ws[n], row_scale(row), p.bias[n]);
        if (p.add) v += (float)((const T*)p.add)[row * p.ldr + n];
        ((T*)p.y)[row * p.ldy + n] = (T)q_out<T, Q_ACT_ANY>(v, p.act);
    }
}

// 8-bit rows: a row fragment is 16 consecutive bytes of a row.
template <typename T, int S, int RB> SOX_DEV void qfew_body(const sox_qgemm_args& p) {
    __shared__ int red[8][RB][16 * 17];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int r16 = lane & 15, kq = lane >> 4, n0 = blockIdx.x * 16, steps = (p.k + 63) / 64;
    const int8_t* w = few_weights(p, n0);
    int4v acc[RB];
#pragma unroll
    for (int b = 0; b < RB; b++) acc[b] = (int4v)0;
    for (int base = wave * S; base < steps; base += waves * S) {
        int4v wf[S], xf[S][RB];
#pragma unroll
        for (int s = 0; s < S; s++) wf[s] = base + s < steps ? *(const int4v*)(w + (int64_t)(base + s) * 2048) : (int4v)0;
#pragma unroll
        for (int b = 0; b < RB; b++) {
            const int8_t* a = p.a + min(b * 16 + r16, p.m - 1) * p.lda + kq * 16;
#pragma unroll
            for (int s = 0; s < S; s++)
                xf[s][b] = (base + s) * 64 + kq * 16 < p.k16 ? *(const int4v*)(a + (int64_t)(base + s) * 64) : (int4v)0;
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
    few_outputs<T, RB>(p, red, waves, n0, [&](int row) { return p.xs[row]; });
}

// Floating rows, up to 16 of at most 4096 values: the workgroup brings them to 8 bits in LDS while its weights are on their
// way, so a token's product is one launch. A wave's item is 1024 values of a row, 16 to a lane; the rows' maxima meet in
// LDS. Every workgroup repeats that rounding, beside the weights' trip from memory. At most 64 items for 16 waves (the
// launcher takes min(16, max(steps, items)) waves), and S >= steps / waves. Bound by latency: 1 x 768 -> 768 3.9 us, of which
// an empty launch is about 2; 7 x 4096 -> 4096 7.8.
template <typename T, int S> SOX_DEV void qfewx_body(const sox_qgemm_args& p) {
    typedef RawValues<T, 16> Chunk;
    typedef RowQuant<T> Q;
    constexpr int ITEMS = 4;
    extern __shared__ __attribute__((aligned(16))) unsigned char qrow[];  // [m][pitch]
    __shared__ uint32_t tops[16][4];
    __shared__ float xscale[16];
    __shared__ int red[16][1][16 * 17];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int r16 = lane & 15, kq = lane >> 4, n0 = blockIdx.x * 16, steps = (p.k + 63) / 64;
    const int segs = (p.k + 1023) / 1024, items = p.m * segs;
    const int pitch = (p.k + 255) / 256 * 256 + 16;  // a row's fragments start in a bank group of their own
    const int8_t* w = few_weights(p, n0);
    int4v wf[S];
#pragma unroll
    for (int s = 0; s < S; s++)
        wf[s] = wave * S + s < steps ? *(const int4v*)(w + (int64_t)(wave * S + s) * 2048) : (int4v)0;
    Chunk v[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        const int it = wave + i * waves, row = it / segs;
        if (it < items) v[i].load((const T*)p.x + row * p.ldx, ((it - row * segs) * 64 + lane) * 16, p.k);
    }
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        const int it = wave + i * waves, row = it / segs;
        if (it < items) {
            AbsMax<T> top;
            top.add(v[i]);
            const uint32_t m = wave_max(top.lane());
            if (lane == 0) tops[row][it - row * segs] = m;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        const int it = wave + i * waves, row = it / segs, ch = (it - row * segs) * 64 + lane;  // 16 k of the row
        if (it < items) {
            uint32_t m = tops[row][0];
            for (int s = 1; s < segs; s++) m = max(m, tops[row][s]);
            const Q rq = Q::make(AbsMax<T>::row_bits(m));
            if (ch == 0) xscale[row] = rq.scale;
            if (ch < steps * 4)
                *(int4v*)(qrow + row * pitch + ch * 16) =
                    int4v{(int)Q::q4(v[i], 0, rq), (int)Q::q4(v[i], 4, rq), (int)Q::q4(v[i], 8, rq), (int)Q::q4(v[i], 12, rq)};
        }
    }
    __syncthreads();
    int4v acc = (int4v)0;
#pragma unroll
    for (int s = 0; s < S; s++) {
        const int step = min(wave * S + s, steps - 1);  // (past the last: its weights are zeros)
        const int4v xf = *(const int4v*)(qrow + min(r16, p.m - 1) * pitch + step * 64 + kq * 16);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[s], xf, acc, 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < 4; e++) red[wave][0][(4 * kq + e) * 17 + r16] = acc[e];
    __syncthreads();
    few_outputs<T, 1>(p, red, min(waves, (steps + S - 1) / S), n0, [&](int row) { return xscale[row]; });
}

#define SOX_QFEWX(NAME, T, S)                                                                                                  \
    extern "C" __global__ void __launch_bounds__(1024) sox_qfewx_##NAME##_s##S(sox_qgemm_args p) { qfewx_body<T, S>(p); }
#define SOX_QFEW(NAME, T, RB)                                                                                                  \
    extern "C" __global__ void __launch_bounds__(512) sox_qfew_##NAME##_r##RB(sox_qgemm_args p) { qfew_body<T, 8 / RB, RB>(p); }
#define SOX_QFEW_ALL(NAME, T) \
    SOX_QFEWX(NAME, T, 1) SOX_QFEWX(NAME, T, 2) SOX_QFEWX(NAME, T, 4) SOX_QFEW(NAME, T, 1) SOX_QFEW(NAME, T, 2) SOX_QFEW(NAME, T, 4)
SOX_QFEW_ALL(f16, half_t)
SOX_QFEW_ALL(bf16, bf16_t)
SOX_QFEW_ALL(f32, float)

// ---- products of a moderate number of floating rows, in one launch ----
// A workgroup of 8 waves takes 32 rows x 128 columns: it brings its rows to 8 bits itself, into LDS in fragment order, while
// its weights are already on their way to registers; wave w then multiplies column block w % 4 over half w / 4 of K and
// the halves meet in LDS. A wave rounds 4 rows side by side, 16 lanes to a row and 16 values of K to a lane and chunk.
// LDS, block kb of 32 k: slot (k % 32 / 16 * 32 + row) ^ (k / 16 % 16) of 16 bytes, so the writers (a lane per 16 k of a row)
// spread over the banks, and a fragment read stays a permutation of one KiB. Bound by the chain load, maximum, round, barrier,
// multiply: 786 x 768 -> 760 7.3 us, and 9.4 with a rounding launch ahead of the ring.
constexpr int QP_ROWS = 32;
template <typename T, int CH> SOX_DEV void qpanel_body(const sox_qgemm_args& p) {
    typedef RowQuant<T> Q;
    extern __shared__ __attribute__((aligned(1024))) unsigned char panel[];  // [kb][1 KiB]
    __shared__ __attribute__((aligned(1024))) unsigned char stage[4][STG_BYTES];
    __shared__ int4v half_sums[4][4][64];
    __shared__ float xscale[QP_ROWS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nbk = (p.k + 31) / 32, per = (nbk + 1) / 2;  // blocks of K, of a half
    const int cb = blockIdx.x * 4 + wave % 4, k0 = wave / 4 * per, k1 = min(k0 + per, nbk);
    const int m0 = blockIdx.y * QP_ROWS;
    const bool live = cb < p.nb;  // (uniform per wave)
    const int8_t* w = p.w + (int64_t)min(cb, p.nb - 1) * p.kb * 1024 + lane * 16;
    int4v wf[4 * CH];  // the wave's weights, all of them (K <= 256 CH)
#pragma unroll
    for (int i = 0; i < 4 * CH; i++) wf[i] = k0 + i < k1 ? *(const int4v*)(w + (int64_t)(k0 + i) * 1024) : (int4v)0;
    {
        const int row = wave * 4 + lane / 16, i16 = lane % 16;
        const T* x = (const T*)p.x + (int64_t)min(m0 + row, p.m - 1) * p.ldx;
        RawValues<T, 16> v[CH];
#pragma unroll
        for (int c = 0; c < CH; c++) v[c].load(x, (c * 16 + i16) * 16, p.k);
        AbsMax<T> top;
#pragma unroll
        for (int c = 0; c < CH; c++) top.add(v[c]);
        const Q rq = Q::make(AbsMax<T>::row_bits(row16_max(top.lane())));
        if (i16 == 0) xscale[row] = rq.scale;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int ch = c * 16 + i16;  // 16 k of the row
            if (ch < 2 * nbk)
                *(int4v*)(panel + ch / 2 * 1024 + (((ch % 2 * 32 + row) ^ i16) << 4)) =
                    int4v{(int)Q::q4(v[c], 0, rq), (int)Q::q4(v[c], 4, rq), (int)Q::q4(v[c], 8, rq), (int)Q::q4(v[c], 12, rq)};
        }
    }
    __syncthreads();
    int16v acc = (int16v)0;
#pragma unroll
    for (int i = 0; i < 4 * CH; i++) {
        const int kb = min(k0 + i, nbk - 1);  // (past the wave's last: its weights are zeros)
        const int4v xf = *(const int4v*)(panel + kb * 1024 + ((lane ^ ((2 * kb + lane / 32) % 16)) << 4));
        acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[i], xf, acc, 0, 0, 0);
    }
    if (wave >= 4)
#pragma unroll
        for (int q = 0; q < 4; q++) half_sums[wave - 4][q][lane] = int4v{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
    __syncthreads();
    if (wave >= 4 || !live) return;
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const int4v o = half_sums[wave][q][lane];
#pragma unroll
        for (int e = 0; e < 4; e++) acc[4 * q + e] += o[e];
    }
    finish_block<T>(p, acc, xscale[lane & 31], p.ws + cb * 32, p.bias + cb * 32, stage[wave], m0, cb * 32, lane);
}

#define SOX_QPANEL(NAME, T, CH)                                                                                              \
    extern "C" __global__ void __launch_bounds__(512) sox_qpanel_##NAME##_c##CH(sox_qgemm_args p) { qpanel_body<T, CH>(p); }
#define SOX_QPANEL_ALL(NAME, T) SOX_QPANEL(NAME, T, 1) SOX_QPANEL(NAME, T, 2) SOX_QPANEL(NAME, T, 3) SOX_QPANEL(NAME, T, 4)
SOX_QPANEL_ALL(f16, half_t)
SOX_QPANEL_ALL(bf16, bf16_t)
SOX_QPANEL_ALL(f32, float)
