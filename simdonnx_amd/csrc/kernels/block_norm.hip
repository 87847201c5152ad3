// The norms before and after a transformer block, with its gate and residual scale, in one pass over the rows:
//   h = res_scale * residual + act(gate) * (post(x) * scale),   y = pre(h)
//   rms(v) = v / sqrt(mean(v^2) + eps) * gamma,   layer(v) = (v - mean v) / sqrt(mean((v - mean v)^2) + eps) * gamma + beta
// y leaves in the storage type or as 8-bit rows with their scales for the product that reads them (qlinear.hip).
//
// Bound by memory: x, residual and gate are read once, h and y written once, and a row stays in registers in between.
// All sums and norms in fp32, a variance as the mean square about the mean (a second sum over the registers, so a large
// mean costs no digits); y is computed from h as summed in fp32, not from its rounded copy.
//
// How a row is held, by how many rows there are and how long:
//  * many rows of up to 1024 columns: a wave per row (half a wave up to 256), no barriers; the parameter vectors, which
//    would move as much from L2 per row as the row itself moves from memory, stand in LDS for all rows the workgroup walks.
//  * few rows, or longer ones: TPR threads per row, which shortens the one row's chain of loads, sums and stores; the
//    parameters stay in registers (or, for the longest rows, are read where they are used).
// A workgroup walks rows a whole grid apart; the grid is held to what the rows' streams run best with: 16384 x 4096 bf16 in
// 95 to 100 us by box (5.7 to 5.4 TB/s) on 2 workgroups per CU, 122 with one row each, and 135 to 300 with a wave per row.
// Registers decide how many waves there are: 8192 x 768 with a gate 13.8 us (100 registers, 4 waves on a SIMD), 17.5 when it took 144.
#include "qrows.h"

enum { NORM_NONE = 0, NORM_RMS = 1, NORM_LAYER = 2 };
enum { PAR_LDS, PAR_REG, PAR_MEM };  // where the parameter vectors are

// CH chunks of E values per thread: chunk j of thread t is columns (j TPR + t) E .. + E - 1 as one 16-byte access
template <typename T, int TPR, int CH> struct Row {
    static constexpr int E = 16 / sizeof(T), N = CH * E;
    typedef typename Chunk16<T>::V TE;
    typedef typename Chunk16<T>::At At;
    TE v[CH];
    SOX_DEV int col(int t, int j) { return (j * TPR + t) * E; }
    // value e of chunk j is inside the row (a compare with a constant: the columns themselves would be held in registers)
    SOX_DEV bool in(int t, int j, int e, int c) { return e < c - col(t, j); }
    __device__ __forceinline__ void load(const T* __restrict__ p, int t, int c) {
#pragma unroll
        for (int j = 0; j < CH; j++) {
            const int k = col(t, j);
            v[j] = TE{};
            if (k + E <= c) {
                v[j] = *(const At*)(p + k);
            } else if (k < c) {  // the row's end inside a chunk
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (in(t, j, e, c)) v[j][e] = p[k + e];
            }
        }
    }
    SOX_DEV void store(T* __restrict__ p, int t, int c, const float (&f)[N]) {
#pragma unroll
        for (int j = 0; j < CH; j++) {
            TE o;
#pragma unroll
            for (int e = 0; e < E; e++) o[e] = (T)f[j * E + e];
            const int k = col(t, j);
            if (k + E <= c) {
                *(At*)(p + k) = o;
            } else if (k < c) {
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (in(t, j, e, c)) p[k + e] = o[e];
            }
        }
    }
    // columns c .. round_up(c, 16) - 1 hold zeros (f is 0 there)
    SOX_DEV void store8(int8_t* __restrict__ p, int t, int c, const float (&f)[N], const RowQuant<half_t>& rq) {
        const int c16 = (c + 15) & ~15;
#pragma unroll
        for (int j = 0; j < CH; j++) {
            uint32_t w[E / 4];
#pragma unroll
            for (int i = 0; i < E / 4; i++) {
                const float* g = &f[j * E + 4 * i];
                w[i] = RowQuant<half_t>::q4(g[0], g[1], g[2], g[3], rq);
            }
            if (col(t, j) < c16) {
                if constexpr (E == 8)
                    *(uint2*)(p + col(t, j)) = make_uint2(w[0], w[1]);
                else
                    *(uint32_t*)(p + col(t, j)) = w[0];
            }
        }
    }
};

// Sum (maximum) over the TPR threads of a row. Each reduction over several waves has an LDS row of its own, two sets
// in turn per row walked, so one barrier per reduction is enough: a set is written again only after the barriers of
// the row in between.
template <int TPR, class V, class F> SOX_DEV V row_fold(V v, V* lds, F&& f) {
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int w = 1; w < W; w++) v = f(v, lds[w]);
    }
    return v;
}
template <int TPR> SOX_DEV float row_sum(float v, float* lds) {
    return row_fold<TPR>(wave_sum<TPR == 32 ? 32 : 64>(v), lds, [](float a, float b) { return a + b; });
}
template <int TPR> SOX_DEV uint32_t row_max(uint32_t v, uint32_t* lds) {
    return row_fold<TPR>(wave_max<TPR == 32 ? 32 : 64>(v), lds, [](uint32_t a, uint32_t b) { return max(a, b); });
}

template <typename T, int TPR, int CH, int PAR> SOX_DEV void bnorm_body(const sox_bnorm_args& p) {
    typedef Row<T, TPR, CH> R;
    constexpr int E = R::E, N = R::N, BLOCK = TPR <= 64 ? 256 : TPR, RPB = BLOCK / TPR, CAP = TPR * N;
    static_assert((PAR == PAR_LDS) == (TPR <= 64), "a wave or half of one per row");
    __shared__ float lds[2][5][BLOCK / 64];
    extern __shared__ float par_lds[];  // PAR_LDS: the vectors there are, CAP floats each
    const int t = threadIdx.x % TPR, c = p.c;
    const float inv_c = 1.0f / (float)c;

    // The parameter vectors: k = 0 post gamma * scale, 1 post beta * scale, 2 pre gamma, 3 pre beta (null: 1, 0, 1, 0)
    const float* const vec[4] = {p.pg, p.pb, p.g, p.b};
    int slot[4];
    float kept[PAR == PAR_REG ? 4 : 1][PAR == PAR_REG ? N : 1];
    auto from_memory = [&](const float* v, int j, float (&o)[E]) __attribute__((always_inline)) {
        const bool in = R::col(t, j) < c;
#pragma unroll
        for (int i = 0; i < E / 4; i++) {
            float4v f = {};
            if (in) f = *(const float4v*)(v + R::col(t, j) + 4 * i);
#pragma unroll
            for (int e = 0; e < 4; e++) o[4 * i + e] = f[e];
        }
    };
    if constexpr (PAR == PAR_REG) {
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (vec[k])
#pragma unroll
                for (int j = 0; j < CH; j++) {
                    float o[E];
                    from_memory(vec[k], j, o);
#pragma unroll
                    for (int e = 0; e < E; e++) kept[k][j * E + e] = o[e];
                }
    }
    if constexpr (PAR == PAR_LDS) {
        // The chunks' first four values of all chunks, then their second four, so 16-byte reads of consecutive lanes are
        // consecutive
        int n = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            slot[k] = n * CAP;
            if (!vec[k]) continue;
            n++;
            for (int i = threadIdx.x; i < CAP; i += BLOCK) {
                const int at = i % E / 4 * (CAP / (E / 4)) + i / E * 4 + i % 4;
                par_lds[slot[k] + at] = i < c ? vec[k][i] : 0.0f;
            }
        }
        __syncthreads();
    }
    // the values of chunk j of vector k
    auto par = [&](int k, int j, float (&o)[E]) __attribute__((always_inline)) {
        if constexpr (PAR == PAR_REG) {
#pragma unroll
            for (int e = 0; e < E; e++) o[e] = kept[k][j * E + e];
        } else if constexpr (PAR == PAR_LDS) {
#pragma unroll
            for (int i = 0; i < E / 4; i++) {
                const float4v f = *(const float4v*)(par_lds + slot[k] + i * (CAP / (E / 4)) + (j * TPR + t) * 4);
#pragma unroll
                for (int e = 0; e < 4; e++) o[4 * i + e] = f[e];
            }
        } else {
            const float* v = vec[k];
            asm volatile("" : "+s"(v));  // (read here, not ahead of the rows into registers that are not there)
            from_memory(v, j, o);
        }
    };
    // v (zeros past column c) normed in place; the vectors k and k + 1
    auto norm = [&](float (&v)[N], int kind, float eps, int k, float* l0, float* l1) __attribute__((always_inline)) {
        if (kind == NORM_LAYER) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < N; i++) s += v[i];
            const float mean = row_sum<TPR>(s, l0) * inv_c;
#pragma unroll
            for (int i = 0; i < N; i++) v[i] = R::in(t, i / E, i % E, c) ? v[i] - mean : 0.0f;
        }
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) s = __builtin_fmaf(v[i], v[i], s);
        const float r = 1.0f / sqrtf(row_sum<TPR>(s, l1) * inv_c + eps);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] *= r;
    };
    // v * gamma (+ beta), the vectors k and k + 1
    auto affine = [&](float (&v)[N], int k) __attribute__((always_inline)) {
        if (vec[k])
#pragma unroll
            for (int j = 0; j < CH; j++) {
                float o[E];
                par(k, j, o);
#pragma unroll
                for (int e = 0; e < E; e++) v[j * E + e] *= o[e];
                if constexpr (PAR == PAR_MEM) __builtin_amdgcn_sched_barrier(0);
            }
        if (vec[k + 1])
#pragma unroll
            for (int j = 0; j < CH; j++) {
                float o[E];
                par(k + 1, j, o);
#pragma unroll
                for (int e = 0; e < E; e++) v[j * E + e] += o[e];
                if constexpr (PAR == PAR_MEM) __builtin_amdgcn_sched_barrier(0);
            }
    };
    int set = 0;
    // (a wave's row is one number: its addresses stay in scalar registers. With 256 threads and up to two chunks it fits as it
    // is, and lanes' own addresses are faster: 16384 x 4096 95.9 us, 99.5 with scalar ones)
    const int sub = TPR == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / TPR) : BLOCK == TPR && (TPR != 256 || N > 16) ? 0 : threadIdx.x / TPR;
    // Where a workgroup fills a CU (512 threads a row), the next row's values come while the row before is worked on; smaller
    // ones have each other's loads for that, and fewer registers: 4096 x 8192 bf16 55 us, 64 without; 40000 x 192 19.4, 14.8
    // without.
    constexpr bool AHEAD = TPR == 512 && PAR == PAR_REG;
    struct Rows {
        R x, r, g;
    };
    std::conditional_t<AHEAD, Rows, char> next;
    auto load_x = [&](R& x, int64_t row) __attribute__((always_inline)) { x.load((const T*)p.x + row * p.ldx, t, c); };
    auto load_r = [&](R& r, int64_t row) __attribute__((always_inline)) { r.load((const T*)p.residual + row * p.ldr, t, c); };
    auto load_g = [&](R& g, int64_t row) __attribute__((always_inline)) {
        g.load((const T*)p.gate + (int64_t)((uint32_t)row / (uint32_t)p.gate_group) * p.ldg, t, c);
    };
    auto fetch = [&](int64_t row) __attribute__((always_inline)) {
        if constexpr (AHEAD) {
            if (row >= p.rows) return;
            if (p.x) load_x(next.x, row);
            if (p.residual) load_r(next.r, row);
            if (p.gate) load_g(next.g, row);
        }
    };
    int64_t row = (int64_t)blockIdx.x * RPB + sub;
    fetch(row);
    for (; row < p.rows; row += (int64_t)gridDim.x * RPB, set ^= 1) {
        R rr, gr;
        float h[N];
        if (p.x) {
            R xr;
            if constexpr (AHEAD) {
                xr = next.x, rr = next.r, gr = next.g;
                fetch(row + (int64_t)gridDim.x * RPB);
            } else {  // all of a row's loads go out together
                load_x(xr, row);
                if (p.residual) load_r(rr, row);
                if (p.gate) load_g(gr, row);
            }
#pragma unroll
            for (int i = 0; i < N; i++) h[i] = (float)xr.v[i / E][i % E];
            if (p.post != NORM_NONE) norm(h, p.post, p.post_eps, 0, lds[set][0], lds[set][1]);
            affine(h, 0);
            if (p.gate) {
                // (one choice per row, each a straight line)
                auto gated = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
                    for (int i = 0; i < N; i++) h[i] *= f((float)gr.v[i / E][i % E]);
                };
                if (p.gate_act == SOX_ACT_NONE)
                    gated([](float g) { return g; });
                else if (p.gate_act == SOX_ACT_RELU)
                    gated([](float g) { return q_out<float, SOX_ACT_RELU>(g); });
                else if (p.gate_act == SOX_ACT_GELU)
                    gated([](float g) { return q_out<float, SOX_ACT_GELU>(g); });
                else
                    gated([&](float g) { return q_out<float, Q_ACT_GATES>(g, p.gate_act); });
            }
            if (p.residual)
#pragma unroll
                for (int i = 0; i < N; i++) h[i] = __builtin_fmaf(p.res_scale, (float)rr.v[i / E][i % E], h[i]);
        } else {
            if constexpr (AHEAD) {
                rr = next.r;
                fetch(row + (int64_t)gridDim.x * RPB);
            } else {
                load_r(rr, row);
            }
#pragma unroll
            for (int i = 0; i < N; i++) h[i] = p.res_scale * (float)rr.v[i / E][i % E];
        }
        if (p.h) R::store((T*)p.h + row * p.ldh, t, c, h);
        if (!p.y && !p.q) continue;
        if (p.pre != NORM_NONE) {
            norm(h, p.pre, p.pre_eps, 2, lds[set][2], lds[set][3]);
            affine(h, 2);
        }
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

#define SOX_BNORM(NAME, T, TPR, CH, PAR)                                                                                   \
    extern "C" __global__ void __launch_bounds__(TPR <= 64 ? 256 : TPR, TPR <= 64 ? 4 : TPR <= 256 ? 2 : 1)                \
        sox_bnorm_##NAME##_t##TPR##c##CH(sox_bnorm_args p) {                                                               \
        bnorm_body<T, TPR, CH, PAR>(p);                                                                                    \
    }
// threads of a row and chunks of a thread: 16-bit rows of up to 256, 512, 1024 columns for many rows, and of up to 2048, 4096,
// 8192, 16384 and one and a half times 2048 and 4096 for few or long ones ...
#define SOX_BNORM_16(NAME, T)                                                                                             \
    SOX_BNORM(NAME, T, 32, 1, PAR_LDS) SOX_BNORM(NAME, T, 64, 1, PAR_LDS) SOX_BNORM(NAME, T, 64, 2, PAR_LDS)              \
    SOX_BNORM(NAME, T, 256, 1, PAR_REG) SOX_BNORM(NAME, T, 128, 3, PAR_REG) SOX_BNORM(NAME, T, 256, 2, PAR_REG) SOX_BNORM(NAME, T, 256, 3, PAR_REG) SOX_BNORM(NAME, T, 512, 2, PAR_REG)           \
    SOX_BNORM(NAME, T, 512, 4, PAR_MEM)
SOX_BNORM_16(f16, half_t)
SOX_BNORM_16(bf16, bf16_t)
// ... and the same in fp32, twice the chunks
SOX_BNORM(f32, float, 32, 2, PAR_LDS) SOX_BNORM(f32, float, 64, 2, PAR_LDS) SOX_BNORM(f32, float, 64, 4, PAR_LDS)
SOX_BNORM(f32, float, 256, 2, PAR_REG) SOX_BNORM(f32, float, 128, 6, PAR_REG) SOX_BNORM(f32, float, 256, 4, PAR_REG) SOX_BNORM(f32, float, 256, 6, PAR_REG) SOX_BNORM(f32, float, 512, 4, PAR_REG)
SOX_BNORM(f32, float, 512, 8, PAR_MEM)
