// Products in 8-bit integers with a scale for each row and each column on the CDNA4 matrix cores:
//   Y[M,N] = act((A[M,K] . W[K,N]) * xs[M] * ws[N] + bias[N] (+ R[M,N])),  A and W int8, int32 sums
//
// The int32 sums are exact (K <= 131071: |sum| < 2^31), so tiles, splits and orders never change a result; one
// conversion to fp32, two scale products and the bias fma follow, and one rounding to the output type.
//
// A ring of K slices in LDS as the 16-bit Gemm's (gemm_ring.h), BM x BN tiles, NW waves, STAGES slices of BK bytes
// of each row, one barrier per slice:
//  * v_mfma_i32_32x32x32_i8: twice the 16-bit instruction's products in the same cycles from the same 16 operand
//    bytes per lane, so a slice has the 16-bit ring's bytes, fragments and LDS traffic at twice the work. W is the
//    row operand: lane l holds Y^T[n = 8 q + 4 (l / 32) + e][m = l % 32].
//  * A rows go global -> LDS by DMA, 16-byte chunks XOR-swizzled on the load side (bank-conflict-free reads); the
//    chunks past k16 come from a zero block.
//  * W is packed at creation in fragment order: a 32 x 32 block is the one KiB that a wave's fragment read takes,
//    lane by lane. Its DMA is one contiguous KiB from a uniform address, its LDS reads need no swizzle, and all
//    blocks of a stage are immediate offsets from one register.
//  * The tile's scales and bias ride into LDS with its first slice.
//  * Persistent: each workgroup walks its tiles as one ring, the next tile's slices load during the epilogue.
//    Workgroups are numbered XCD-major, so the tiles in flight on one XCD share rows and columns in its L2.
//  * Epilogue per 32 x 32 block through 4 KiB of LDS per wave: scaled fp32 values in, rows out, so residual loads
//    and output stores are whole row segments and one code path serves every storage type.
#pragma once
#include "qrows.h"

#define LDS_PTR(p) ((__attribute__((address_space(3))) void*)(p))

template <int I, int N, class F> SOX_DEV void static_for(F&& f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        static_for<I + 1, N>(f);
    }
}

// s_waitcnt with only vmcnt constrained (gfx9 encoding: vmcnt[3:0] | expcnt[6:4] | lgkmcnt[11:8] | vmcnt_hi[15:14])
template <int N> SOX_DEV void wait_vmcnt() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}
SOX_DEV void wait_lgkmcnt0() { __builtin_amdgcn_s_waitcnt(0xc07f); }

// LDS chunk swizzle for rows of CPR 16-byte chunks: 16 consecutive rows read at one chunk hit 16 distinct bank groups
template <int CPR> SOX_DEV int swz(int r) { return (r / (16 / CPR)) % CPR; }

// One 32 x 32 block of scaled sums from a wave's LDS stage to memory. The stage holds 32 rows of 8 16-byte chunks of
// fp32, chunk c of row r at slot c ^ r / 2 % 8: the writers (a row per lane) and the readers (a row per 4 or 8 lanes)
// both spread over all banks.
SOX_DEV int stage_at(int r, int c) { return r * 128 + ((c ^ ((r >> 1) & 7)) << 4); }

template <typename T>
SOX_DEV void store_block(const sox_qgemm_args& p, const unsigned char* stg, int m0, int n0) {
    const int lane = threadIdx.x & 63;
    T* __restrict__ Y = (T*)p.y;
    const T* __restrict__ R = (const T*)p.add;
    if (p.vec & 1) {  // uniform: 16-byte row chunks
        constexpr int E = 16 / sizeof(T), PER = 32 / E;  // elements of a chunk, chunks of a row
        typedef vec_t<T, E> TE;
#pragma unroll
        for (int t = 0; t < 32 * PER / 64; t++) {
            const int idx = t * 64 + lane, r = idx / PER, u = idx % PER;
            const int m = m0 + r, n = n0 + u * E;
            const bool in = m < p.m && n < p.n;
            float v[E];
#pragma unroll
            for (int c = 0; c < E / 4; c++) {
                const float4v f = *(const float4v*)(stg + stage_at(r, u * (E / 4) + c));
#pragma unroll
                for (int e = 0; e < 4; e++) v[4 * c + e] = f[e];
            }
            if (R) {
                const TE rv = in ? *(const TE*)(R + (int64_t)m * p.ldr + n) : TE{};
#pragma unroll
                for (int e = 0; e < E; e++) v[e] += (float)rv[e];
            }
            TE o;
#pragma unroll
            for (int e = 0; e < E; e++) o[e] = (T)q_act<T>(v[e], p.act);
            if (in) *(TE*)(Y + (int64_t)m * p.ldy + n) = o;
        }
    } else {
#pragma unroll 4
        for (int t = 0; t < 16; t++) {
            const int idx = t * 64 + lane, r = idx / 32, c = idx % 32;
            const int m = m0 + r, n = n0 + c;
            if (m < p.m && n < p.n) {
                float v = *(const float*)(stg + stage_at(r, c / 4) + (c % 4) * 4);
                if (R) v += (float)R[(int64_t)m * p.ldr + n];
                Y[(int64_t)m * p.ldy + n] = (T)q_act<T>(v, p.act);
            }
        }
    }
}

template <typename T, int BM, int BN, int BK, int WM, int WN, int STAGES, int NW, int GM>
__device__ __forceinline__ void qgemm_body(const sox_qgemm_args& p) {
    constexpr int CPR = BK / 16, KS = BK / 32;
    constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK, STAGE_BYTES = A_BYTES + B_BYTES;
    constexpr int A_IT = A_BYTES / 1024 / NW, B_IT = B_BYTES / 1024 / NW, LOADS = A_IT + B_IT;
    constexpr int TI = WM / 32, TJ = WN / 32, WAVES_N = BN / WN;
    // scales and bias of the tiles in flight: a tile's first slice may be issued STAGES tiles ahead (K of one slice)
    constexpr int SC_BYTES = BM * 4 + BN * 8, SCB = STAGES + 1;
    static_assert(CPR == 4 || CPR == 8, "64 or 128 bytes of K per slice");
    static_assert(KS % 2 == 0, "fragment sets alternate per k-step and must realign per slice");
    static_assert((BM / WM) * (BN / WN) == NW && WM % 32 == 0 && WN % 32 == 0, "tiling");
    static_assert(A_IT * 1024 * NW == A_BYTES && B_IT * 1024 * NW == B_BYTES, "DMA split");
    static_assert(BM % 64 == 0 && BN <= 256 && NW >= 2, "scale DMA split");
    static_assert(STAGES >= 2 && (STAGES - 1) * LOADS < 64, "vmcnt range");
    __shared__ __attribute__((aligned(1024))) unsigned char smem[STAGE_BYTES * STAGES + SC_BYTES * SCB + NW * 4096];
    unsigned char* const sc_mem = smem + STAGE_BYTES * STAGES;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31, hl = lane >> 5;
    unsigned char* const stg = sc_mem + SC_BYTES * SCB + wave * 4096;
    const int M = p.m, k16 = p.k16;
    const int tiles_n = p.tiles_n, tiles_m = (M + BM - 1) / BM, ntiles = tiles_m * tiles_n;
    const int wm0 = (wave / WAVES_N) * WM, wn0 = (wave % WAVES_N) * WN;
    const int nk = (k16 + BK - 1) / BK;

    // XCD-major workgroup number: dispatch id b runs on XCD b % 8
    const int G = gridDim.x;
    const int vid = (G % 8 == 0) ? (blockIdx.x % 8) * (G / 8) + blockIdx.x / 8 : blockIdx.x;
    const int my_tiles = vid < ntiles ? (ntiles - 1 - vid) / G + 1 : 0;
    const int total = my_tiles * nk;  // this workgroup's ring of K slices
    if (total == 0) return;
    auto tile_origin = [&](int t, int& bm, int& bn) __attribute__((always_inline)) {  // M-tiles walked in groups of GM
        const int group = t / (GM * tiles_n), first_m = group * GM;
        const int gsize = min(tiles_m - first_m, GM);
        const int in_group = t - group * GM * tiles_n;
        bm = (first_m + in_group % gsize) * BM;
        bn = (in_group / gsize) * BN;
    };

    // DMA of A: instruction i of this wave fills the KiB at (wave A_IT + i) KiB of the stage: row r, slot s of it hold
    // chunk s ^ swz(r). Rows past M re-read the last row (never stored).
    auto a_row = [&](int i) __attribute__((always_inline)) { return ((wave * A_IT + i) * 1024 + lane * 16) / BK; };
    auto a_chunk = [&](int i) __attribute__((always_inline)) {
        return (((wave * A_IT + i) * 1024 + lane * 16) % BK / 16) ^ swz<CPR>(a_row(i));
    };
    const int8_t* a_src[A_IT];
    int i_kt = 0, i_tile = vid, i_seq = 0, i_bn = 0;  // the slice being issued: its k-slice, tile and the tile's column
    auto issue = [&](int gs) __attribute__((always_inline)) {
        unsigned char* st = smem + (gs % STAGES) * STAGE_BYTES;
        if (i_kt == 0) {
            int bm;
            tile_origin(i_tile, bm, i_bn);
#pragma unroll
            for (int i = 0; i < A_IT; i++) a_src[i] = p.a + (int64_t)min(bm + a_row(i), M - 1) * p.lda + a_chunk(i) * 16;
            unsigned char* sc = sc_mem + (i_seq % SCB) * SC_BYTES;
            // (ws and bias are padded to whole tiles of at most 256 columns)
            if (wave == 0 && lane < BN / 4) __builtin_amdgcn_global_load_lds(p.ws + i_bn + lane * 4, LDS_PTR(sc), 16, 0, 0);
            if (wave == 1 && lane < BN / 4)
                __builtin_amdgcn_global_load_lds(p.bias + i_bn + lane * 4, LDS_PTR(sc + BN * 4), 16, 0, 0);
#pragma unroll
            for (int i = 0; i < BM / 64; i++)
                if (wave == i % NW)
                    __builtin_amdgcn_global_load_lds(p.xs + min(bm + i * 64 + lane, M - 1), LDS_PTR(sc + BN * 8 + i * 256), 4, 0, 0);
        }
        const int k0 = i_kt * BK;
        const bool tail = k0 + BK > k16;  // uniform
#pragma unroll
        for (int i = 0; i < A_IT; i++) {
            const int8_t* src = a_src[i] + k0;
            if (tail) src = k0 + a_chunk(i) * 16 < k16 ? src : (const int8_t*)p.zeros;
            __builtin_amdgcn_global_load_lds(src, LDS_PTR(st + (wave * A_IT + i) * 1024), 16, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < B_IT; i++) {
            const int b = wave * B_IT + i, cb = min(i_bn / 32 + b / KS, p.nb - 1);
            const int8_t* src = p.w + ((int64_t)cb * p.kb + i_kt * KS + b % KS) * 1024 + lane * 16;
            __builtin_amdgcn_global_load_lds(src, LDS_PTR(st + A_BYTES + b * 1024), 16, 0, 0);
        }
        if (++i_kt == nk) {
            i_kt = 0;
            i_tile += G;
            i_seq++;
        }
    };

    // fragments: k-step s of a lane covers chunk 2 s + l / 32 of row l % 32 of each block
    const int a_off = (wm0 + l32) * BK + ((hl ^ swz<CPR>(l32)) << 4);  // step s: bits 5.. flipped by s (swz repeats per 32 rows)
    const int b_off = A_BYTES + (wn0 / 32) * KS * 1024 + lane * 16;
    int16v acc[TJ][TI];
    int4v fa0[TI], fb0[TJ], fa1[TI], fb1[TJ];
    auto read_step = [&](int gs, int s, int4v (&fa)[TI], int4v (&fb)[TJ]) __attribute__((always_inline)) {
        const unsigned char* st = smem + (gs % STAGES) * STAGE_BYTES;
#pragma unroll
        for (int j = 0; j < TJ; j++) fb[j] = *(const int4v*)(st + b_off + (j * KS + s) * 1024);
#pragma unroll
        for (int i = 0; i < TI; i++) fa[i] = *(const int4v*)(st + (a_off ^ (s << 5)) + i * 32 * BK);
    };
    auto clear = [&]() __attribute__((always_inline)) {
        static_for<0, TJ * TI>([&](auto ji) { acc[decltype(ji)::value / TI][decltype(ji)::value % TI] = (int16v)0; });
    };
    int m_kt = 0, m_tile = vid, m_seq = 0;  // the tile being multiplied
    auto epilogue = [&]() __attribute__((always_inline)) {
        int bm, bn;
        tile_origin(m_tile, bm, bn);
        const unsigned char* sc = sc_mem + (m_seq % SCB) * SC_BYTES;
        static_for<0, TJ * TI>([&](auto ji) {
            constexpr int j = decltype(ji)::value / TI, i = decltype(ji)::value % TI;
            const float xs = *(const float*)(sc + BN * 8 + (wm0 + i * 32 + l32) * 4);
            static_for<0, 4>([&](auto qq) {
                constexpr int q = decltype(qq)::value;
                const int n = wn0 + j * 32 + 8 * q + 4 * hl;
                const float4v ws = *(const float4v*)(sc + n * 4), bs = *(const float4v*)(sc + BN * 4 + n * 4);
                float4v v;
                static_for<0, 4>([&](auto ee) {
                    constexpr int e = decltype(ee)::value;
                    v[e] = __builtin_fmaf((float)acc[j][i][4 * q + e] * ws[e], xs, bs[e]);
                });
                *(float4v*)(stg + stage_at(l32, 2 * q + hl)) = v;
            });
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // other lanes' rows are read back
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            store_block<T>(p, stg, bm + wm0 + i * 32, bn + wn0 + j * 32);
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // the next block overwrites the stage
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            __builtin_amdgcn_sched_barrier(0);
        });
        m_tile += G;
        m_seq++;
    };

#pragma unroll
    for (int s = 0; s < STAGES; s++)
        if (s < total) issue(s);
    // waits until this wave's loads of the slice after gs have landed. A slice carries LOADS loads or, where it starts a
    // tile, more, so that many newer ones at least may stay in flight for each newer slice; the last slices wait for all
    if (total >= STAGES)
        wait_vmcnt<(STAGES - 1) * LOADS>();
    else
        wait_vmcnt<0>();
    __builtin_amdgcn_s_barrier();
    clear();
    read_step(0, 0, fa0, fb0);
    for (int gs = 0; gs < total; gs++) {
        static_for<0, KS>([&](auto step) {
            constexpr int s = decltype(step)::value;
            int4v(&ca)[TI] = (s & 1) ? fa1 : fa0;
            int4v(&cb)[TJ] = (s & 1) ? fb1 : fb0;
            int4v(&na)[TI] = (s & 1) ? fa0 : fa1;
            int4v(&nb)[TJ] = (s & 1) ? fb0 : fb1;
            if constexpr (s == KS - 1) {
                // slice gs + 1 landed and every read of slice gs done; after the barrier both hold for all waves
                if (gs + STAGES < total)
                    wait_vmcnt<(STAGES - 2) * LOADS>();
                else
                    wait_vmcnt<0>();
                wait_lgkmcnt0();
                __builtin_amdgcn_s_barrier();
                if (gs + STAGES < total) issue(gs + STAGES);
                read_step(gs + 1, 0, na, nb);  // (past the last slice: a stage whose content is not used)
            } else {
                read_step(gs, s + 1, na, nb);
            }
            static_for<0, TJ * TI>([&](auto ji) {
                constexpr int j = decltype(ji)::value / TI, i = decltype(ji)::value % TI;
                acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(cb[j], ca[i], acc[j][i], 0, 0, 0);
            });
            constexpr int RD = TI + TJ, MF = TI * TJ;
            static_for<0, (RD < MF ? RD : MF)>([&](auto) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            });
            if constexpr (MF > RD) __builtin_amdgcn_sched_group_barrier(0x008, MF - RD, 0);
            if constexpr (RD > MF) __builtin_amdgcn_sched_group_barrier(0x100, RD - MF, 0);
            __builtin_amdgcn_sched_barrier(0);
        });
        wait_lgkmcnt0();  // the next slice's first fragments
        if (++m_kt == nk) {
            m_kt = 0;
            epilogue();
            clear();
        }
    }
}

#define SOX_QGEMM(TILE, BM, BN, BK, WM, WN, ST, NW, OCC, GM)                                                     \
    extern "C" __global__ void __launch_bounds__(64 * NW, OCC) sox_qgemm_f16_##TILE(sox_qgemm_args p) {        \
        qgemm_body<half_t, BM, BN, BK, WM, WN, ST, NW, GM>(p);                                                 \
    }                                                                                                          \
    extern "C" __global__ void __launch_bounds__(64 * NW, OCC) sox_qgemm_bf16_##TILE(sox_qgemm_args p) {       \
        qgemm_body<bf16_t, BM, BN, BK, WM, WN, ST, NW, GM>(p);                                                 \
    }                                                                                                          \
    extern "C" __global__ void __launch_bounds__(64 * NW, OCC) sox_qgemm_f32_##TILE(sox_qgemm_args p) {        \
        qgemm_body<float, BM, BN, BK, WM, WN, ST, NW, GM>(p);                                                  \
    }
