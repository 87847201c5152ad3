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
//  * Epilogue per 32 x 32 block: scaled and activated in registers, turned into rows through 2 KiB of LDS per wave, so
//    residual loads and output stores are whole row segments.
//
// Tiles by size (the host's estimates choose): 256 x 256 with its 8 waves holds a wave's 128 x 64 outputs in registers and
// multiplies 43 times for each byte of LDS that it reads, 128 times for each that comes from memory; 256 x 192 for shapes
// whose tiles it deals to the CUs in fuller rounds (8192 x 1024 -> 1536: one round, 19.4 us; 256 x 256 21.5, 256 x 128 24.3,
// 128 x 128 24.6); down to 64 x 64, four slices deep, where there are few tiles and a slice's latency counts.
// Bound: with long K by DMA, LDS reads and MFMAs that overlap in part, 4096 x 4096 -> 8192 in 117 to 122 us by box (2.25 to
// 2.35e15 operations a second; a large library product of 8-bit integers reaches 2.0 to 2.1e15). Of a 256 x 256 tile's 52 us at
// K = 4096, 43 are left without its DMA and 35 without its MFMAs; its epilogue is 4. With short K by the prologue (2 us), the
// epilogue (nothing multiplies meanwhile) and the outputs' stores.
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

// A wave's stage for outputs on their way to memory, 2 KiB: a 32 x 32 block of 16-bit values (rows of 4 16-byte chunks, chunk
// c of row r at slot c ^ r / 4 % 4), or 16 rows of a block of fp32 ones (8 chunks, slot c ^ r / 2). The writers (a row per
// lane) and the readers (a row per 4 or 8 lanes) both spread over all banks, and the stores are whole row segments.
constexpr int STG_BYTES = 2048;
template <typename T> SOX_DEV int stage_at(int r, int c) {
    return sizeof(T) == 2 ? r * 64 + ((c ^ ((r >> 2) & 3)) << 4) : r * 128 + ((c ^ (r >> 1)) << 4);
}

// What a kernel knows of its outputs' rows:
//   Q_LINES  they stand on 128-byte lines and hold whole 16-byte chunks. Their stores pass L2 by, which leaves it to the A and W
//            lines that are read again: 4096 x 4096 -> 8192 with its rounding 125 us, 133 with stores through L2, 128 with the
//            choice made in the kernel
//   Q_CHUNKS they hold whole chunks. Their stores go through L2: a line that different stores write in parts would reach memory
//            in parts, 2954 x 320 -> 3112 19.8 us so and 13.3 through L2
//   Q_PART   any
enum { Q_LINES, Q_CHUNKS, Q_PART };

// A block's rows between memory at (m0, n0) and the stage, 16 bytes at a time, single elements in the chunk that a row ends in.
// LOAD: the residual's into the stage (zeros outside), else the stage's to the output.
template <typename T, bool LOAD, int FORM>
SOX_DEV void move_rows(T* __restrict__ base, int64_t ld, int M, int N, unsigned char* stg, int m0, int n0, int lane) {
    constexpr int E = 16 / sizeof(T), PER = 32 / E, ROWS = STG_BYTES / (32 * sizeof(T));  // elements of a chunk, chunks of a row
    typedef typename Chunk16<T>::V TE;
    typedef typename Chunk16<T>::At At;
#pragma unroll
    for (int t = 0; t < ROWS * PER / 64; t++) {
        const int idx = t * 64 + lane, r = idx / PER, u = idx % PER, m = m0 + r, n = n0 + u * E;
        TE* s = (TE*)(stg + stage_at<T>(r, u));
        T* g = base + (int64_t)m * ld + n;
        if constexpr (LOAD) {
            TE v = {};
            if (m < M && n + E <= N) {
                v = *(const At*)g;
            }
            *s = v;
            if (FORM == Q_PART && m < M && n < N && n + E > N)
#pragma unroll 1
                for (int e = 0; e < N - n; e++) ((T*)s)[e] = g[e];
        } else {
            const TE v = *s;
            if (m < M && n + E <= N) {
                if constexpr (FORM == Q_LINES)
                    __builtin_nontemporal_store(v, (TE*)g);
                else
                    *(At*)g = v;
            } else if (FORM == Q_PART && m < M && n < N) {
#pragma unroll 1
                for (int e = 0; e < N - n; e++) g[e] = ((const T*)s)[e];
            }
        }
    }
}
// Lanes read what others wrote to the wave's stage, or overwrite what others have read
SOX_DEV void stage_turn() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A 32 x 32 block's outputs from its sums (lane l: row l % 32, columns 8 q + 4 (l / 32) + e in element 4 q + e): scaled, joined
// with the residual and activated in registers, staged and stored. One copy of this with its choices inside, none of
// them per element: a choice per element, or a copy per form, multiplied the ring's code until its instruction fetches
// took most of a short product's time and registers ran out. ws, bias: the block's 32 columns.
template <typename T, int FORM = Q_PART>
SOX_DEV void finish_block(const sox_qgemm_args& p, const int16v& sums, float xs, const float* ws, const float* bias,
                          unsigned char* stg, int m0, int n0, int lane) {
    constexpr int PARTS = sizeof(T) == 2 ? 1 : 2, ROWS = 32 / PARTS;
    typedef vec_t<T, 4> T4;
    const int l32 = lane & 31, hl = lane >> 5;
    float val[16];
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const float4v w4 = *(const float4v*)(ws + 8 * q + 4 * hl), b4 = *(const float4v*)(bias + 8 * q + 4 * hl);
#pragma unroll
        for (int e = 0; e < 4; e++) val[4 * q + e] = __builtin_fmaf((float)sums[4 * q + e] * w4[e], xs, b4[e]);
    }
    // the lane's four of the stage: 16-bit rows 64 bytes, fp32 ones 128 (and half of them at a time)
    auto at = [&](int q) __attribute__((always_inline)) {
        return sizeof(T) == 2 ? (T4*)(stg + stage_at<T>(l32, q) + hl * 8) : (T4*)(stg + stage_at<T>(l32 % ROWS, 2 * q + hl));
    };
    if (p.add) {
#pragma unroll
        for (int half = 0; half < PARTS; half++) {
            move_rows<T, true, FORM>((T*)p.add, p.ldr, p.m, p.n, stg, m0 + half * ROWS, n0, lane);
            stage_turn();
            if (PARTS == 1 || l32 / ROWS == half) {
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const T4 r = *at(q);
#pragma unroll
                    for (int e = 0; e < 4; e++) val[4 * q + e] += (float)r[e];
                }
            }
            stage_turn();
        }
    }
    if (p.act == SOX_ACT_GELU) {
#pragma unroll
        for (int e = 0; e < 16; e++) val[e] = q_out<T, SOX_ACT_GELU>(val[e]);
    } else if (p.act == SOX_ACT_RELU) {
#pragma unroll
        for (int e = 0; e < 16; e++) val[e] = q_out<T, SOX_ACT_RELU>(val[e]);
    } else if (p.act != SOX_ACT_NONE) {
#pragma unroll
        for (int e = 0; e < 16; e++) val[e] = q_out<T, Q_ACT_GATES>(val[e], p.act);
    }
#pragma unroll
    for (int half = 0; half < PARTS; half++) {
        if (PARTS == 1 || l32 / ROWS == half) {
#pragma unroll
            for (int q = 0; q < 4; q++) {
                T4 h;
#pragma unroll
                for (int e = 0; e < 4; e++) h[e] = (T)val[4 * q + e];
                *at(q) = h;
            }
        }
        stage_turn();
        move_rows<T, false, FORM>((T*)p.y, p.ldy, p.m, p.n, stg, m0 + half * ROWS, n0, lane);
        stage_turn();
    }
}

template <typename T, int BM, int BN, int BK, int WM, int WN, int STAGES, int NW, int GM, int FORM>
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
    __shared__ __attribute__((aligned(1024))) unsigned char smem[STAGE_BYTES * STAGES + SC_BYTES * SCB + NW * STG_BYTES];
    unsigned char* const sc_mem = smem + STAGE_BYTES * STAGES;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31, hl = lane >> 5;
    unsigned char* const stg = sc_mem + SC_BYTES * SCB + wave * STG_BYTES;
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
    // Ring slice gs = (place in this workgroup's tile list) * nk + k-slice; slices are started in order. Past the last tile
    // they re-read its rows into a stage that nobody reads again, so that every slice has its loads, one count covers
    // them all and the k-steps stay one basic block.
    const int8_t* a_src[A_IT];
    int i_kt = nk - 1, i_tile = vid - G, i_seq = -1, i_bn = 0;  // the slice being issued: its k-slice, tile and the tile's column
    auto start_slice = [&](int gs) __attribute__((always_inline)) {
        if (++i_kt < nk) return;
        i_kt = 0;
        i_tile += G;
        if (gs >= total) return;
        i_seq++;
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
    };
    // load x of the slice started last
    auto fire = [&](int gs, auto xx) __attribute__((always_inline)) {
        constexpr int x = decltype(xx)::value;
        unsigned char* st = smem + (gs % STAGES) * STAGE_BYTES;
        if constexpr (x < A_IT) {
            const int k = i_kt * BK;
            const int8_t* src = k + a_chunk(x) * 16 < k16 ? a_src[x] + k : (const int8_t*)p.zeros;
            __builtin_amdgcn_global_load_lds(src, LDS_PTR(st + (wave * A_IT + x) * 1024), 16, 0, 0);
        } else {
            const int b = wave * B_IT + x - A_IT, cb = min(i_bn / 32 + b / KS, p.nb - 1);
            const int8_t* src = p.w + ((int64_t)cb * p.kb + i_kt * KS + b % KS) * 1024 + lane * 16;
            __builtin_amdgcn_global_load_lds(src, LDS_PTR(st + A_BYTES + b * 1024), 16, 0, 0);
        }
    };
    // A slice's loads go out in two parts, behind the slice barrier and a k-step later, one after each MFMA: a wave that
    // issues them stalls while the CU's 64 bytes a cycle drain, and MFMAs queued between keep the matrix cores busy.
    constexpr int PART0 = (LOADS + 1) / 2;

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
        static_for<0, TJ * TI>([&](auto ji) __attribute__((always_inline)) {
            constexpr int j = decltype(ji)::value / TI, i = decltype(ji)::value % TI;
            const float* ws = (const float*)sc + wn0 + j * 32;
            const float xs = *(const float*)(sc + BN * 8 + (wm0 + i * 32 + l32) * 4);
            finish_block<T, FORM>(p, acc[j][i], xs, ws, ws + BN, stg, bm + wm0 + i * 32, bn + wn0 + j * 32, lane);
            __builtin_amdgcn_sched_barrier(0);  // one block at a time: bounded register pressure
        });
        m_tile += G;
        m_seq++;
    };

#pragma unroll
    for (int s = 0; s < STAGES; s++) {
        start_slice(s);
        static_for<0, LOADS>([&](auto xx) { fire(s, xx); });
    }
    // slice 0. (Loads complete in order; a slice carries LOADS loads or, where it starts a tile, more, so at least that many
    // may stay in flight for each newer slice.)
    wait_vmcnt<(STAGES - 1) * LOADS>();
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
            constexpr int DM = s == KS - 1 ? PART0 : s == 0 ? LOADS - PART0 : 0;  // loads issued in this k-step
            if constexpr (s == KS - 1) {
                // slice gs + 1 landed and every read of slice gs done; after the barrier both hold for all waves, and the
                // stage of slice gs takes slice gs + STAGES
                wait_vmcnt<(STAGES - 2) * LOADS>();
                wait_lgkmcnt0();
                __builtin_amdgcn_s_barrier();
                start_slice(gs + STAGES);
                static_for<0, PART0>([&](auto xx) { fire(gs + STAGES, xx); });
                read_step(gs + 1, 0, na, nb);  // (past the last slice: a stage whose content is not used)
            } else {
                if constexpr (s == 0)
                    if (gs > 0) static_for<PART0, LOADS>([&](auto xx) { fire(gs - 1 + STAGES, xx); });
                read_step(gs, s + 1, na, nb);
            }
            static_for<0, TJ * TI>([&](auto ji) {
                constexpr int j = decltype(ji)::value / TI, i = decltype(ji)::value % TI;
                acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(cb[j], ca[i], acc[j][i], 0, 0, 0);
            });
            constexpr int RD = TI + TJ, MF = TI * TJ;
            static_for<0, MF>([&](auto ii) {
                constexpr int i = decltype(ii)::value;
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                if constexpr (i < DM) __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
                if constexpr (i < RD) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            });
            if constexpr (DM > MF) __builtin_amdgcn_sched_group_barrier(0x010, DM - MF, 0);
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
    wait_vmcnt<0>();  // the slices past the end land before the workgroup's LDS is given back
}

// Two kernels per storage type and tiling, for outputs on lines (_l) and others, named BMxBN tile, wNW waves, kBK bytes of K per
// slice, sSTAGES; WM x WN of a tile to a wave, OCC waves per SIMD, GM M-tiles to a group.
#define SOX_QGEMM_FORM(NAME, T, TILE, BM, BN, BK, WM, WN, ST, NW, OCC, GM, FORM)                                  \
    extern "C" __global__ void __launch_bounds__(64 * NW, OCC) sox_qgemm_##NAME##_##TILE(sox_qgemm_args p) { \
        qgemm_body<T, BM, BN, BK, WM, WN, ST, NW, GM, FORM>(p);                                                   \
    }
#define SOX_QGEMM(NAME, T, TILE, BM, BN, BK, WM, WN, ST, NW, OCC, GM, FORM)                           \
    SOX_QGEMM_FORM(NAME, T, TILE, BM, BN, BK, WM, WN, ST, NW, OCC, GM, FORM)                          \
    SOX_QGEMM_FORM(NAME, T, TILE##_l, BM, BN, BK, WM, WN, ST, NW, OCC, GM, Q_LINES)
#define SOX_QGEMM_TILES(NAME, T)                                                     \
    SOX_QGEMM(NAME, T, 256x192_w8k128s2, 256, 192, 128, 64, 96, 2, 8, 2, 4, Q_PART) \
    SOX_QGEMM(NAME, T, 256x128_w8k128s2, 256, 128, 128, 64, 64, 2, 8, 2, 4, Q_PART) \
    SOX_QGEMM(NAME, T, 128x128_w4k128s2, 128, 128, 128, 64, 64, 2, 4, 2, 4, Q_PART) \
    SOX_QGEMM(NAME, T, 64x64_w4k128s4, 64, 64, 128, 32, 32, 4, 4, 2, 4, Q_PART)
