// Attention of new tokens over a paged cache: for each new row at position t of its sequence and each query head,
//   y = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - reference),  j <= t and, with a window w, j > t - w
// in one pass over the sequence's tokens with the running reference of a softmax. Two kernels:
//   many  a workgroup takes 128 pairs (new row, query head of one kv head's group), 32 a wave, and walks the tokens tile by
//         tile through LDS, which all of its waves read; bound by the softmax's instructions beside the matrix cores. Two prompts of
//         8192, 32 query heads over 8: heads of 128 1.25 ms in bf16 (880 TFLOP/s), 1.39 in 8 bits; of 64 0.69; of 256 (one
//         wave a SIMD, for its registers) 1.91 with 16 over 4
//   few   16 pairs (a single new token's group): its waves walk different tokens, K straight to registers; bound by reading the
//         cache. One token over 131072: 93 us in bf16 (5.8 TB/s), 64 over 4096 to 8192 in 8 bits 161 (5.2 TB/s)
// (both: the two in one launch)
// Both compute S^T = K Q^T, so a lane holds one pair's scores, 16 (or 8) tokens in its registers: the softmax needs no other
// lane but for the maximum, and the scores, rounded, are as they stand the operand of O^T += V^T P^T. The token order within a
// step is that of the score registers; V's rows are read to match it (transposing LDS reads for 16 bits).
// The reference moves only when a score passes it by 2^8: what it leaves in p is divided out by the sum, and the outputs are
// rescaled a few times, not once a tile. Sums and outputs in fp32; p is rounded to the storage type for its product (half a
// step each, unbiased, on terms that the sum averages). In fp16 the reference stands 2^7 below the score that moved it, which with
// the 2^8 is what its numbers have room for: small weights, of which a long context has many, are then normal numbers down
// to 2^-21 of the largest.
// An 8-bit cache: k and v go into the products as whole numbers (exact in every storage type); k's scale multiplies the score,
// v's p, before its rounding. In fp16, whose exponents end soon, p times scale would lose its bits beside a token of far larger
// scale, in the channels where that one holds zeros too. There V takes the scale's power of two and p the rest of it, in its
// exponent (scale_power, scale_rest; the reference bounds p times the rest, the sum divides it out again). With its scale even a p
// of one is rounded, so in `few`, which the memory bounds, what the rounding leaves is the operand of a second product: 1.5 times the
// output's own rounding without it where a few tokens have the weight, and as fast (64 tokens over 4096 to 8192 in bf16
// 160 to 168 us either way). V is finite there, so that nothing not finite meets a part of the other sign.
// Tokens that a row does not see add nothing, whatever their K and V hold: tokens that no row of the tile sees are not read,
// masked scores are replaced, and a V that is not finite within a tile that is masked in part goes through without its values
// that are not finite (special4).
#pragma once
#include "kv_cache.h"

constexpr int AT_THREADS = 256;
constexpr float AT_SLACK = 8.0f;  // powers of two that p may rise before the reference moves

// ---- storage types' steps ----
template <typename T> struct Frag {  // 16 bytes of a row
    static constexpr int E = 16 / sizeof(T);
    typedef vec_t<T, E> V;
};
template <typename T> SOX_DEV float16v mma32(typename Frag<T>::V a, typename Frag<T>::V b, float16v c) {
    if constexpr (sizeof(T) == 2) {
        c = mfma32x32x16(a, b, c);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
    }
    return c;
}
template <typename T> SOX_DEV float4v mma16(typename Frag<T>::V a, typename Frag<T>::V b, float4v c) {
    if constexpr (sizeof(T) == 2) {
        c = mfma16x16x32(a, b, c);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    }
    return c;
}

// A byte of a word as a number, in the one instruction that the compiler makes two of. Its result goes into a conversion: a
// matrix instruction may not read it at once, and the compiler, which keeps that distance elsewhere, does not see into an asm.
template <int I> SOX_DEV float signed_byte(int w) {
    float f;
    if constexpr (I == 0) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0" : "=v"(f) : "v"(w));
    if constexpr (I == 1) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(f) : "v"(w));
    if constexpr (I == 2) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(f) : "v"(w));
    if constexpr (I == 3) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(f) : "v"(w));
    return f;
}
// 16 bytes of the cache as they go to LDS: values of T
template <typename T, typename C> struct Wide {
    static constexpr int N = sizeof(T) / sizeof(C);  // 16-byte chunks of them
    typename Frag<T>::V v[N];
    // (POWER: times a power of two, scale_power's, in fp16)
    template <bool POWER = false> SOX_DEV Wide of(int4v raw, half2v power = {}) {
        Wide w;
        if constexpr (N == 1) {
            w.v[0] = __builtin_bit_cast(typename Frag<T>::V, raw);
        } else {
            constexpr int E = Frag<T>::E;
            asm("" : "+v"(raw));  // (here, not where it was loaded: the compiler takes its first steps there, and waits)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                auto& to = w.v[4 * i / E];
                const int e = 4 * i % E;
                if constexpr (std::is_same<T, half_t>::value) {  // 0x6400 + u is the number 1024 + u, u = q + 128
                    const uint32_t u = (uint32_t)raw[i] ^ 0x80808080u;
                    const half2v by = {(half_t)1152.0f, (half_t)1152.0f};
                    half2v a = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u));
                    half2v b = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u));
                    if constexpr (POWER) {
                        a = __builtin_elementwise_fma(a, power, -by * power), b = __builtin_elementwise_fma(b, power, -by * power);
                    } else {
                        a -= by, b -= by;
                    }
                    to[e] = a[0], to[e + 1] = a[1], to[e + 2] = b[0], to[e + 3] = b[1];
                } else if constexpr (sizeof(T) == 4) {
#pragma unroll
                    for (int n = 0; n < 4; n++) to[e + n] = (float)(int8_t)(raw[i] >> 8 * n);
                } else {
                    to[e] = (T)signed_byte<0>(raw[i]), to[e + 1] = (T)signed_byte<1>(raw[i]);
                    to[e + 2] = (T)signed_byte<2>(raw[i]), to[e + 3] = (T)signed_byte<3>(raw[i]);
                }
            }
        }
        return w;
    }
};

template <typename T> SOX_DEV bool any_not_finite(int4v raw) {
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t w = (uint32_t)raw[i];
        if constexpr (sizeof(T) == 4) {
            bad |= (w & 0x7f800000u) == 0x7f800000u;
        } else {
            constexpr uint32_t EXP = std::is_same<T, half_t>::value ? 0x7c00u : 0x7f80u;
            bad |= (w & EXP) == EXP || ((w >> 16) & EXP) == EXP;
        }
    }
    return bad;
}

// Places of 16-byte chunks within LDS rows of CH chunks, so that what one read touches spreads over all banks: K's chunk by 16
// rows (a chunk of 16 or 32 rows at once); V's, in 16 bits by 4 rows x 4 chunks (many) or 8 rows x 2 (few) of the transposing
// reads, in 32 by rows 4 apart (8 chunks of two, or 4 of four)
template <int CH> SOX_DEV int at_k(int row) { return CH >= 16 ? row & 15 : (row >> 1) & 7; }
template <int CH, int BYTES, bool FEW> SOX_DEV int at_v(int row) {
    if (BYTES == 4) return FEW ? row & 12 : (row & 4) << 1;
    return CH >= 16 ? ((row & 3) << 2) | ((row >> 1) & 2) : (((row >> 1) & 1) << 2) | ((row >> 1) & 2);
}

typedef short short4v __attribute__((ext_vector_type(4)));
// Four values of a column from four rows for each lane: in each 16 lanes, lane l gives the address of columns 4 (l & 3) .. + 3
// of row l / 4 and gets column l of the four
SOX_DEV short4v read_columns(const unsigned char* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)p);
}
template <typename T> SOX_DEV typename Frag<T>::V join(short4v lo, short4v hi) {
    typedef short short8v __attribute__((ext_vector_type(8)));
    return __builtin_bit_cast(typename Frag<T>::V, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// ---- a value of V that is not finite, in a tile that some rows see in part ----
// The matrix cores would carry 0 * inf into rows that do not see it, so such a tile goes through the product with those
// values replaced by 0, and rows that see them get them from memory (special4).
template <typename T> SOX_DEV int4v finite_only(int4v raw) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t w = (uint32_t)raw[i];
        if constexpr (sizeof(T) == 4) {
            raw[i] = (w & 0x7f800000u) == 0x7f800000u ? 0 : (int)w;
        } else {
            constexpr uint32_t EXP = std::is_same<T, half_t>::value ? 0x7c00u : 0x7f80u;
            raw[i] = (int)(((w & EXP) == EXP ? 0u : w & 0xffffu) | ((w >> 16 & EXP) == EXP ? 0u : w & 0xffff0000u));
        }
    }
    return raw;
}
// What four channels of a token's V add to a row that sees it: their values that are not finite
template <typename T> SOX_DEV float4v special4(const T* v) {
    typedef vec_t<T, 4> V4;
    typedef V4 At __attribute__((aligned(sizeof(T))));
    const V4 x = *(const At*)v;
    float4v o;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float f = (float)x[e];
        o[e] = abs_bits(f) < 0x7f800000u ? 0.0f : f;
    }
    return o;
}

template <int I, int N, class F> SOX_DEV void static_for(F&& f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        static_for<I + 1, N>(f);
    }
}

// How v's scale in 8 bits takes part: not at all, as a factor of p, or in V's and p's exponents
enum { SCALE_NONE, SCALE_FACTOR, SCALE_EXPONENT };
template <typename T, typename C> constexpr int scale_form() {
    return sizeof(C) == 1 ? std::is_same<T, half_t>::value ? SCALE_EXPONENT : SCALE_FACTOR : SCALE_NONE;
}
// A scale's power of two, as V takes it: from 2^-24 (V's whole numbers times that are fp16's smallest steps) to 2^5 (times 1152, as
// the bytes become numbers, it is in fp16's range)
SOX_DEV float scale_power(float scale) {
    return __uint_as_float(min(max(__float_as_uint(scale) & 0x7f800000u, 103u << 23), 132u << 23));
}
SOX_DEV half2v scale_power2(float scale) { return half2v{(half_t)scale_power(scale), (half_t)scale_power(scale)}; }
// and the rest, 1 to 2 for scales of 2^-24 to 2^6: it moves p by that much, a scale of 2^9, the last of fp16 rows, by 16. Below,
// where V is less than half of fp16's smallest step, it ends at 2^-20; a row of zeros has 1; a NaN stays one. (Scales past 2^26, of
// values that fp16 rows cannot have, take p of other tokens below its normal numbers.)
SOX_DEV float scale_rest(float scale) {
    const float rest = scale * __uint_as_float(0x7f000000u - __float_as_uint(scale_power(scale)));
    return scale == 0.0f ? 1.0f : __builtin_elementwise_maximum(rest, 0x1p-20f);
}

// c + the sum of eight values
SOX_DEV float sum8(half8 v, float c) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) c = __builtin_amdgcn_fdot2(half2v{v[i], v[i + 1]}, half2v{(half_t)1.0f, (half_t)1.0f}, c, false);
    return c;
}
SOX_DEV float sum8(bf16x8 v, float c) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) c = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{v[i], v[i + 1]}, bf16x2{(bf16_t)1.0f, (bf16_t)1.0f}, c, false);
    return c;
}

// f of this lane's value and that of the lane 32 (or 16) away, in both
template <class F> SOX_DEV float over_32(float v, F&& f) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <class F> SOX_DEV float over_16(float v, F&& f) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
SOX_DEV float larger(float a, float b) { return fmaxf(a, b); }
SOX_DEV float added(float a, float b) { return a + b; }

// ---- which rows a workgroup has ----
struct RowTile {
    int sequence, first;      // first: its first new row
    int rows, pairs, m0;      // new rows and pairs of the sequence, first pair of the tile
    int64_t length;           // tokens
    bool some;
};
// The t-th tile of PAIRS pairs, counted over the sequences; every lane finds the same. `only` leaves out sequences of at most 16
// pairs (LARGE) or of more.
template <int PAIRS, bool LARGE> SOX_DEV RowTile row_tile(const sox_kv_attend_args& p, int t, int lane) {
    RowTile r{};
    int base = 0;
    for (int c = 0; c < p.b.sequences; c += 64) {
        int tiles = 0, first = 0, rows = 0;
        if (c + lane < p.b.sequences) {
            first = min(max(p.b.starts[c + lane], 0), p.b.rows);
            rows = max(min(p.b.starts[c + lane + 1], p.b.rows) - first, 0);
            const int64_t pairs = (int64_t)rows * p.group;
            if (!p.only || (pairs > 16) == LARGE) tiles = (int)((pairs + PAIRS - 1) / PAIRS);
        }
        int sum = tiles;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(sum, o);
            if (lane >= o) sum += v;
        }
        const uint64_t past = __ballot(base + sum > t);
        if (past) {
            const int l = __builtin_ctzll(past);
            r.sequence = c + l;
            r.first = __builtin_amdgcn_readlane(first, l);
            r.rows = __builtin_amdgcn_readlane(rows, l);
            r.pairs = r.rows * p.group;
            // (a sequence's later tiles, which see more, start first)
            const int before = base + __builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(tiles, l);
            r.m0 = (__builtin_amdgcn_readlane(tiles, l) - 1 - (t - before)) * PAIRS;
            r.length = max(p.b.lengths[r.sequence], 0);
            r.some = true;
            return r;
        }
        base += __builtin_amdgcn_readlane(sum, 63);
    }
    return r;
}

// The tokens of a tile of rows, and a split's share of them in steps of TT
struct Span {
    int lo, hi;              // tokens that any row sees, within the table: at most 2^30, so that no sum of them leaves 32 bits
    int begin, end;          // of this split, begin a multiple of TT
    int pos_first, pos_last; // positions of the tile's first and last row
    int low_last;            // the last token that the last row's window leaves out, or -1
};
// The last token that a window leaves out for a row at `pos`, or -1
SOX_DEV int window_low(const sox_kv_attend_args& p, int pos) {
    return p.window > 0 ? (int)max((int64_t)pos - p.window, (int64_t)-1) : -1;
}
template <int PAIRS, int TT> SOX_DEV Span span_of(const sox_kv_attend_args& p, const RowTile& r, int split, int splits, int min_tokens) {
    Span s;
    const int64_t base = r.length - r.rows;
    const int last = min(r.m0 + PAIRS, r.pairs) - 1;
    s.pos_first = (int)(base + r.m0 / p.group);
    s.pos_last = (int)(base + last / p.group);
    s.low_last = window_low(p, s.pos_last);
    s.hi = (int)min((int64_t)s.pos_last + 1, (int64_t)p.b.table_pages << p.b.shift);
    s.lo = min(window_low(p, s.pos_first) + 1, max(s.hi, 0));
    const int from = s.lo / TT * TT, tiles = max((s.hi - from + TT - 1) / TT, 0);
    const int per = max((tiles + splits - 1) / splits, (min_tokens + TT - 1) / TT);
    s.begin = min(from + (int)min((int64_t)split * per * TT, (int64_t)1 << 30), max(s.hi, from));
    s.end = min(s.begin + per * TT, s.hi);
    return s;
}

// A lane's token of a tile: its table entry, from the table's nearest one where it has none, so that the load needs no branch
// and nothing waits for it until tile_page looks at it, a tile later
SOX_DEV int tile_entry(const sox_kv_view& b, const int32_t* table, int token) {
    return table[min(max(token, 0) >> b.shift, b.table_pages - 1)];
}
// and its page, or -1: no page of the pool, or a token outside of [lo, hi) (which lies within the table)
SOX_DEV int tile_page(const sox_kv_view& b, int entry, int token, int lo, int hi) {
    return token >= lo && token < hi && (uint32_t)entry < (uint32_t)b.pages ? entry : -1;
}
// The head's rows of a page, `bytes` into their region: a page is below 4 GiB
SOX_DEV const uint8_t* head_rows(const sox_kv_view& b, const uint8_t* head, int page, uint32_t bytes) {
    return head + (uint64_t)(uint32_t)page * (uint32_t)b.page_bytes + bytes;
}

// Where a row's results go
template <typename T> struct RowOut {
    T* y;
    float* part;
    float* ml;
};
template <typename T> SOX_DEV RowOut<T> row_out(const sox_kv_attend_args& p, const RowTile& r, int kvh, int m, int split) {
    const int64_t row = r.first + m / p.group;
    const int head = kvh * p.group + m % p.group;
    const int64_t at = (row * p.q_heads + head) * p.stride + split;
    return {(T*)p.y + row * p.ldy + (int64_t)head * p.b.dim, p.part + at * p.b.dim, p.ml + at * 2};
}
template <typename T> SOX_DEV const T* row_q(const sox_kv_attend_args& p, const RowTile& r, int kvh, int m) {
    return (const T*)p.q + (int64_t)(r.first + m / p.group) * p.ldq + (int64_t)(kvh * p.group + m % p.group) * p.b.dim;
}
template <typename T> SOX_DEV void store4(T* to, float4v v) {
    typedef vec_t<T, 4> V4;
    typedef V4 At __attribute__((aligned(sizeof(T))));
    fp32_rounded(v);
    *(At*)to = __builtin_convertvector(v, V4);
}
// A chunk of q, zeros past the head's channels
template <typename T> SOX_DEV typename Frag<T>::V load_q(const T* q, int ch, int dim, bool valid) {
    typename Frag<T>::V v = {};
    if (valid && ch < dim) v = *(const typename Chunk16<T>::At*)(q + ch);
    return v;
}

// The running reference and sum of a lane's pair. Scores in powers of two.
template <typename T> struct Soft {
    static constexpr float LIFT = std::is_same<T, half_t>::value ? 7.0f : 0.0f;  // of the score that moves the reference above it
    float ref = -__builtin_inff(), limit = -__builtin_inff(), sum = 0.0f;
    SOX_DEV float of(float ref) { return ref == -__builtin_inff() ? 0.0f : ref; }  // (nothing seen yet: any reference will do)
    // whether `top` passes the reference by AT_SLACK more (a limit held from the last move on: the sum with a reference whose steps are
    // 2 to 16 may be off by half of that, and p of 2^16 is too much for fp16)
    __device__ __forceinline__ bool passed(float top) const { return top > limit; }
    // moves the reference up to `top`; what the sum and the outputs are to be multiplied by
    __device__ __forceinline__ float move(float top) {
        const float now = fmaxf(ref, top - LIFT);
        const float by = ref == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(ref - now);
        ref = now;
        limit = ref + (LIFT + AT_SLACK);
        if (limit - ref > LIFT + AT_SLACK) limit = ref;
        sum *= by;
        return by;
    }
};

// =====================================================================================================================
// many: 128 pairs, 4 waves of 32, tiles of TT tokens through LDS
// =====================================================================================================================
template <typename T, typename C, int DP> struct Many {
    static constexpr int FORM = scale_form<T, C>();
    static constexpr bool QUANT = FORM != SCALE_NONE;
    static constexpr int E = Frag<T>::E, CH = DP / E, KS = CH / 2, PITCH = DP * (int)sizeof(T);
    static constexpr int TT = PITCH >= 512 ? 32 : 64, TB = TT / 32, DB = DP / 32;
    static constexpr int EC = 16 / (int)sizeof(C), UR = DP / EC, NCH = Wide<T, C>::N;  // values of a unit of 16 bytes of the cache, units of a row
    static constexpr int SU = TT * UR / AT_THREADS;                                     // units a thread stages
    static constexpr int BUF = 2 * TT * PITCH;                                          // K and V of a tile
    static constexpr int LDS = 2 * BUF + 2 * 3 * TT * 4 + 64;
    static constexpr int WAVES = PITCH > 256 ? 1 : 2;  // on a SIMD
    static constexpr int GROUP = sizeof(T) == 2 ? 4 : 2, VGROUP = 4;  // fragments read at once
    static constexpr bool AHEAD = PITCH <= 512;        // the next tile's loads in flight behind a tile (beyond, registers are short)
    static_assert(SU >= 1 && TT * UR % AT_THREADS == 0, "staging");
};

template <typename T, typename C, int DP> __device__ __forceinline__ void attend_many(const sox_kv_attend_args& p, uint32_t block) {
    typedef Many<T, C, DP> M;
    typedef typename Frag<T>::V FV;
    constexpr bool QUANT = M::QUANT;
    constexpr int FORM = M::FORM;
    constexpr int TT = M::TT, TB = M::TB, DB = M::DB, E = M::E;
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    float(*const scales)[3][TT] = (float(*)[3][TT])(lds + 2 * M::BUF);
    int* const flags = (int*)(lds + 2 * M::BUF + 2 * 3 * TT * 4);  // a wave found what is not finite in a cut tile's V
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, col = lane & 31;
    const sox_kv_view& b = p.b;
    const int kvh = block % b.heads, rest = block / b.heads, splits = p.splits_many, split = rest % splits;
    const RowTile r = row_tile<128, true>(p, rest / splits, lane);
    if (!r.some) return;
    const Span s = span_of<128, TT>(p, r, split, splits, p.min_many);
    const int32_t* const table = b.tables + r.sequence * b.ldt;
    const int mask = (1 << b.shift) - 1;
    const int64_t scale_at = tid < TT ? b.ks_at : b.vs_at;  // of what this thread stages of the scales

    // this lane's pair
    const int m = r.m0 + 32 * wave + col;
    const bool mine = m < r.pairs;
    // (a lane without a pair sees all: nothing, and its wave would look for a reference in every tile)
    const int pos = mine ? (int)(r.length - r.rows + m / p.group) : 0x7fffffff, low = mine ? window_low(p, pos) : -1;
    const int wave_last = r.m0 + 32 * wave < r.pairs ? (int)(r.length - r.rows + (min(r.m0 + 32 * wave + 32, r.pairs) - 1) / p.group) : -1;
    FV qf[M::KS];
    {
        const T* const q = row_q<T>(p, r, kvh, mine ? m : r.m0);
#pragma unroll
        for (int ks = 0; ks < M::KS; ks++) qf[ks] = load_q<T>(q, (2 * ks + half) * E, b.dim, mine);
    }
    float16v out[DB];
#pragma unroll
    for (int d = 0; d < DB; d++) out[d] = float16v{};
    Soft<T> soft;
    // Scores without scales of their own meet the score's in the subtraction, one instruction for both. The reference is a product
    // rounded, the fma's is not: up to half a step of the reference apart, which past 2^24 are powers of two in p. So behind a
    // reference past 2^20, of any of the wave's pairs, products are rounded first.
    bool large = false;

    // ---- staging ----
    int4v raw_k[M::SU], raw_v[M::SU];
    float raw_s = 0.0f;  // threads 0 .. TT - 1: K's scale of their token, TT .. 2 TT - 1: V's
    float raw_e[FORM == SCALE_EXPONENT ? M::SU : 1];  // V's scales of raw_v's tokens
    const uint32_t row_bytes = (uint32_t)b.dim * sizeof(C);
    const uint8_t* const head = b.pool + ((int64_t)kvh << b.shift) * row_bytes;
    const uint8_t* const head_s = b.pool + ((int64_t)kvh << b.shift) * 4;
    auto entry = [&](int t0) { return tile_entry(b, table, t0 + min(lane, TT - 1)); };
    auto page_of = [&](int t0, int entry) { return lane < TT ? tile_page(b, entry, t0 + lane, s.lo, s.end) : -1; };
    auto thread = [&] {  // (in the widest instances not to be worked with ahead of the loop: registers are short)
        int t = tid;
        if constexpr (!M::AHEAD) asm volatile("" : "+v"(t));
        return t;
    };
    const bool wide_pages = (1 << b.shift) >= 64 / M::UR && b.dim == DP;  // what a wave loads at once of a tile seen whole stands in one page
    auto load = [&](int t0, int pages, bool part, int from = 0, int to = M::SU) {
        typedef int4v At __attribute__((aligned(4)));
        if (wide_pages && !part) {
#pragma unroll
            for (int j = from; j < to; j++) {
                const int row = (j * AT_THREADS + wave * 64) / M::UR, page = __builtin_amdgcn_readlane(pages, row);
                const uint8_t* const at = head_rows(b, head, page, ((t0 + row) & mask) * (DP * (int)sizeof(C)));
                raw_k[j] = *(const At*)(at + lane * 16);
                raw_v[j] = *(const At*)(at + b.v_at + lane * 16);
                if constexpr (FORM == SCALE_EXPONENT) raw_e[j] = *(const float*)(head_rows(b, head_s, page, ((t0 + row) & mask) * 4) + b.vs_at + lane / M::UR * 4);
            }
        } else {
            const int tid = thread();
            int of[M::SU];
#pragma unroll
            for (int j = from; j < to; j++) of[j] = M::UR == 64 ? __builtin_amdgcn_readlane(pages, 4 * j + wave) : __shfl(pages, (j * AT_THREADS + tid) / M::UR);
#pragma unroll
            for (int j = from; j < to; j++) {
                const int u = j * AT_THREADS + tid, row = u / M::UR, c = u % M::UR, page = of[j];
                raw_k[j] = raw_v[j] = int4v{};
                if constexpr (FORM == SCALE_EXPONENT) raw_e[j] = page >= 0 ? *(const float*)(head_rows(b, head_s, page, ((t0 + row) & mask) * 4) + b.vs_at) : 0.0f;
                if (page >= 0 && c * M::EC < b.dim) {
                    const uint8_t* const at = head_rows(b, head, page, ((t0 + row) & mask) * row_bytes + c * 16);
                    raw_k[j] = *(const At*)at;
                    raw_v[j] = *(const At*)(at + b.v_at);
                }
            }
        }
        if constexpr (QUANT) {
            const int page = __shfl(pages, tid & (TT - 1));
            raw_s = 0.0f;
            if (tid < 2 * TT && page >= 0)
                raw_s = *(const float*)(head_rows(b, head_s, page, ((t0 + (tid & (TT - 1))) & mask) * 4) + scale_at);
        }
    };
    bool found = false;  // a value of V that is not finite (of an 8-bit cache its scale), in a tile that is cut
    // cut: a tile that some rows see less of than others, whose V goes without such values
    auto store = [&](int buf, bool cut, int from = 0, int to = M::SU) {
        const int tid = thread();
        unsigned char* const lk = lds + buf * M::BUF;
        unsigned char* const lv = lk + TT * M::PITCH;
        if constexpr (!QUANT) {
            if (cut) {
                uint32_t bad = 0;
#pragma unroll
                for (int j = from; j < to; j++) {
                    bad |= any_not_finite<T>(raw_v[j]);
                    raw_v[j] = finite_only<T>(raw_v[j]);
                }
                found |= __any(bad);
            }
        }
#pragma unroll
        for (int j = from; j < to; j++) {
            const int u = j * AT_THREADS + tid, row = u / M::UR, c = (u % M::UR) * M::NCH;
            const Wide<T, C> k = Wide<T, C>::of(raw_k[j]);
            Wide<T, C> v;
            if constexpr (FORM == SCALE_EXPONENT)
                v = Wide<T, C>::template of<true>(raw_v[j], scale_power2(raw_e[j]));
            else
                v = Wide<T, C>::of(raw_v[j]);
#pragma unroll
            for (int n = 0; n < M::NCH; n++) {
                *(FV*)(lk + row * M::PITCH + (((c + n) ^ at_k<M::CH>(row)) << 4)) = k.v[n];
                *(FV*)(lv + row * M::PITCH + (((c + n) ^ at_v<M::CH, sizeof(T), false>(row)) << 4)) = v.v[n];
            }
            if constexpr (QUANT) __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (QUANT) {
            if (cut) {
                const bool bad = tid >= TT && abs_bits(raw_s) >= 0x7f800000u;
                raw_s = bad ? 0.0f : raw_s;
                found |= __any(bad);
            }
            if (tid < TT) {
                scales[buf][0][tid] = raw_s * p.scale_log2;
            } else if (tid < 2 * TT) {
                if constexpr (FORM == SCALE_EXPONENT) {
                    const float v = scale_rest(raw_s);
                    scales[buf][1][tid - TT] = __builtin_amdgcn_logf(v);
                    scales[buf][2][tid - TT] = 1.0f / v;
                } else {
                    scales[buf][1][tid - TT] = raw_s;
                }
            }
        }
    };
    auto is_cut = [&](int t0) { return t0 + TT - 1 > s.pos_first || t0 <= s.low_last; };
    auto in_part = [&](int t0, uint64_t valid) { return is_cut(t0) || ~valid << (64 - TT) != 0; };  // (or without some of its tokens)

    // ---- a tile ----
    auto tile = [&](int t0, int buf, uint64_t valid, bool part) {
        const unsigned char* const lk = lds + buf * M::BUF;
        const unsigned char* const lv = lk + TT * M::PITCH;
        float16v acc[TB];
#pragma unroll
        for (int tb = 0; tb < TB; tb++) acc[tb] = float16v{};
        // K's fragments a group ahead of their MFMAs (left alone, the compiler waits for each where it is used)
        {
            constexpr int G = M::GROUP, GROUPS = M::KS * TB / G;
            FV kf[2][G];
            auto read_k = [&](int g, FV(&f)[G]) {
#pragma unroll
                for (int i = 0; i < G; i++) {
                    const int ks = (g * G + i) / TB, row = 32 * ((g * G + i) % TB) + col;
                    f[i] = *(const FV*)(lk + row * M::PITCH + (((2 * ks + half) ^ at_k<M::CH>(row)) << 4));
                }
            };
            read_k(0, kf[0]);
#pragma unroll
            for (int g = 0; g < GROUPS; g++) {
                __builtin_amdgcn_sched_barrier(0);
                if (g + 1 < GROUPS) read_k(g + 1, kf[(g + 1) & 1]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < G; i++) {
                    const int ks = (g * G + i) / TB, tb = (g * G + i) % TB;
                    acc[tb] = mma32<T>(kf[g & 1][i], qf[ks], acc[tb]);
                }
            }
        }
        // V's likewise, the first group behind the softmax
        auto v_at = [&](int row, int ch) { return lv + row * M::PITCH + (((ch / E) ^ at_v<M::CH, sizeof(T), false>(row)) << 4) + ch % E * (int)sizeof(T); };
        constexpr int VG = M::VGROUP, VGROUPS = TB * 2 * DB / VG;
        FV vf[2][sizeof(T) == 2 ? VG : 1];
        auto read_v = [&](int g, FV(&f)[sizeof(T) == 2 ? VG : 1]) {
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int i = 0; i < VG; i++) {
                    const int at = g * VG + i, step = at / DB, d = at % DB;  // steps of 16 tokens
                    const int row = 16 * step + 4 * half + ((lane & 15) >> 2), ch = 32 * d + (lane & 16) + 4 * (lane & 3);
                    f[i] = join<T>(read_columns(v_at(row, ch)), read_columns(v_at(row + 8, ch)));
                }
            }
        };
        __builtin_amdgcn_sched_barrier(0);
        read_v(0, vf[0]);
        __builtin_amdgcn_sched_barrier(0);
        // register i of block tb: token t0 + 32 tb + 8 (i / 4) + 4 half + i % 4
        auto token = [&](int tb, int i) { return 32 * tb + 8 * (i >> 2) + 4 * half + (i & 3); };
        // tokens as this lane counts them, from its first one on: constants below
        const uint64_t there = valid >> (4 * half);
        const int until = pos - t0 - 4 * half, after = low - t0 - 4 * half;
        auto seen = [&](int tb, int i) {
            const int t = 32 * tb + 8 * (i >> 2) + (i & 3);
            return (t <= until) & (t > after) & (int)((t < 32 ? (uint32_t)there : (uint32_t)(there >> 32)) >> t % 32 & 1);
        };
        // (scales a group of four tokens ahead of their use)
        auto scales4 = [&](int which, int g) { return *(const float4v*)&scales[buf][which][token(g / 4, 4 * (g % 4))]; };
        constexpr int VS = FORM == SCALE_EXPONENT ? 2 : 1;
        float x[TB][16];
        {
            float4v ks[2], lv[2];
            if constexpr (QUANT) ks[0] = scales4(0, 0);
            if constexpr (FORM == SCALE_EXPONENT) lv[0] = scales4(1, 0);
#pragma unroll
            for (int g = 0; g < 4 * TB; g++) {
                if constexpr (QUANT) {
                    __builtin_amdgcn_sched_barrier(0);
                    if (g + 1 < 4 * TB) {
                        ks[(g + 1) & 1] = scales4(0, g + 1);
                        if constexpr (FORM == SCALE_EXPONENT) lv[(g + 1) & 1] = scales4(1, g + 1);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float a = acc[g / 4][4 * (g % 4) + e];
                    x[g / 4][4 * (g % 4) + e] = FORM == SCALE_EXPONENT ? __builtin_fmaf(a, ks[g & 1][e], lv[g & 1][e]) : QUANT ? a * ks[g & 1][e] : a;
                }
            }
        }
        auto scaled = [&] {
#pragma unroll
            for (int tb = 0; tb < TB; tb++)
#pragma unroll
                for (int i = 0; i < 16; i++) x[tb][i] *= p.scale_log2;
        };
        if (part | large) {
            if (!QUANT && large) scaled();
            if (part) {
#pragma unroll
                for (int tb = 0; tb < TB; tb++)
#pragma unroll
                    for (int i = 0; i < 16; i++) x[tb][i] = seen(tb, i) ? x[tb][i] : -__builtin_inff();
            }
        }
        float top = x[0][0];
#pragma unroll
        for (int tb = 0; tb < TB; tb++)
#pragma unroll
            for (int i = 0; i < 16; i++) top = fmaxf(top, x[tb][i]);
        if constexpr (!QUANT) top *= large ? 1.0f : p.scale_log2;
        if (__any(soft.passed(top))) {
            const float by = soft.move(over_32(top, larger));
            if (!QUANT && !large && __any(__builtin_fabsf(Soft<T>::of(soft.ref)) > 0x1p20f)) {
                large = true;
                scaled();
            }
#pragma unroll
            for (int d = 0; d < DB; d++) {
                out[d] *= by;
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        const float ref = Soft<T>::of(soft.ref), scale = large ? 1.0f : p.scale_log2;
#pragma unroll
        for (int tb = 0; tb < TB; tb++)
#pragma unroll
            for (int i = 0; i < 16; i++) x[tb][i] = __builtin_amdgcn_exp2f(QUANT ? x[tb][i] - ref : __builtin_fmaf(x[tb][i], scale, -ref));
        // the sum, and p as it meets v
        if constexpr (!(sizeof(T) == 2 && !QUANT)) {
            float4v vs[2];
            if constexpr (QUANT) vs[0] = scales4(VS, 0);
#pragma unroll
            for (int g = 0; g < 4 * TB; g++) {
                if constexpr (QUANT) {
                    __builtin_amdgcn_sched_barrier(0);
                    if (g + 1 < 4 * TB) vs[(g + 1) & 1] = scales4(VS, g + 1);
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float& a = x[g / 4][4 * (g % 4) + e];
                    soft.sum = FORM == SCALE_EXPONENT ? __builtin_fmaf(a, vs[g & 1][e], soft.sum) : soft.sum + a;
                    if constexpr (FORM == SCALE_FACTOR) a *= vs[g & 1][e];
                }
            }
        }
        FV pf[2 * TB];
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int st = 0; st < 2 * TB; st++) {
#pragma unroll
                for (int e = 0; e < 8; e++) pf[st][e] = (T)x[st / 2][8 * (st % 2) + e];
                if constexpr (!QUANT) soft.sum = sum8(pf[st], soft.sum);  // (of p as it meets v, two at a time)
            }
        }
        // O^T += V^T P^T
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int g = 0; g < VGROUPS; g++) {
                __builtin_amdgcn_sched_barrier(0);
                if (g + 1 < VGROUPS) read_v(g + 1, vf[(g + 1) & 1]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < VG; i++) {
                    const int at = g * VG + i;
                    out[at % DB] = mfma32x32x16(vf[g & 1][i], pf[at / DB], out[at % DB]);
                }
            }
        } else {
#pragma unroll
            for (int tb = 0; tb < TB; tb++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
#pragma unroll
                    for (int d = 0; d < DB; d++) {
                        out[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(*(const T*)v_at(token(tb, i), 32 * d + col), x[tb][i], out[d], 0, 0, 0);
                        if (d % 4 == 3 || d == DB - 1) __builtin_amdgcn_sched_barrier(0);
                    }
                }
        }
    };

    // ---- the tokens ----
    if (s.begin < s.end) {
        int pages = page_of(s.begin, entry(s.begin));
        int next = entry(s.begin + TT);
        uint64_t valid = __ballot(pages >= 0);
        bool part = in_part(s.begin, valid);
        // a tile's units one after the other
        auto load_and_store = [&](int t0, int buf, bool part) {
            static_for<0, M::SU>([&](auto j) {
                constexpr int at = decltype(j)::value;
                __builtin_amdgcn_sched_barrier(0);
                load(t0, pages, part, at, at + 1);
                store(buf, is_cut(t0), at, at + 1);
            });
        };
        if constexpr (M::AHEAD) {
            load(s.begin, pages, part);
            store(0, is_cut(s.begin));
        } else {
            load_and_store(s.begin, 0, part);
        }
        __syncthreads();
        int buf = 0;
        for (int t0 = s.begin; t0 < s.end; t0 += TT, buf ^= 1) {
            const bool more = t0 + TT < s.end;
            pages = page_of(t0 + TT, next);
            const uint64_t next_valid = __ballot(pages >= 0);
            const bool next_part = in_part(t0 + TT, next_valid);
            next = entry(t0 + 2 * TT);
            if (M::AHEAD && more) load(t0 + TT, pages, next_part);
            if (t0 <= wave_last) tile(t0, buf, valid, part);
            if (!M::AHEAD && more) load_and_store(t0 + TT, buf ^ 1, next_part);
            if (M::AHEAD && more) store(buf ^ 1, is_cut(t0 + TT));
            __syncthreads();
            valid = next_valid;
            part = next_part;
        }
    }

    // ---- out ----  (the pair from the lane number anew: held through the loop, it would cost the widest instances a spill)
    soft.sum = over_32(soft.sum, added);
    if (lane == 0) flags[wave] = found;
    __syncthreads();
    const bool special = flags[0] | flags[1] | flags[2] | flags[3];
    const int me = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0)), to = r.m0 + 32 * wave + (me & 31), upper = me >> 5;
    const int64_t at = r.length - r.rows + to / p.group;
    if (to >= r.pairs || at < 0) return;
    const RowOut<T> o = row_out<T>(p, r, kvh, to, split);
    if (splits > 1) {
        if (upper == 0) o.ml[0] = soft.ref, o.ml[1] = s.begin < s.end ? soft.sum : -1.0f;
        if (s.begin >= s.end) return;
    }
    const float inv = splits > 1 ? 1.0f : soft.sum == 0.0f ? 0.0f : 1.0f / soft.sum;
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int i4 = 0; i4 < 4; i4++) {
            const int ch = 32 * d + 8 * i4 + 4 * upper;
            float4v v;
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = out[d][4 * i4 + e] * inv;
            if (ch >= b.dim) continue;
            if (special) {  // what the row sees of the values left out
#pragma unroll 1
                for (int t = s.begin; t < s.end; t++) {
                    if (!is_cut((t - s.begin) / TT * TT + s.begin)) {
                        t += TT - 1;
                        continue;
                    }
                    const int page = t >= s.lo ? kv_page(b, table, t) : -1;
                    if (page < 0 || t > at || (p.window > 0 && t <= at - p.window)) continue;
                    if constexpr (QUANT) {
                        const float f = *(const float*)(head_rows(b, head_s, page, (t & mask) * 4) + b.vs_at);
                        v += abs_bits(f) < 0x7f800000u ? 0.0f : f;
                    } else {
                        v += special4((const T*)(head_rows(b, head, page, (t & mask) * row_bytes) + b.v_at) + ch);
                    }
                }
            }
            if (splits > 1)
                *(float4v*)(o.part + ch) = v;
            else
                store4(o.y + ch, v);
        }
}

// =====================================================================================================================
// few: 16 pairs, 4 waves that walk every fourth tile of TT tokens each
// =====================================================================================================================
template <typename T, typename C, int DP> struct Few {
    static constexpr int FORM = scale_form<T, C>();
    static constexpr bool QUANT = FORM != SCALE_NONE;
    static constexpr int E = Frag<T>::E, CH = DP / E, PITCH = DP * (int)sizeof(T);
    static constexpr int TT = sizeof(T) == 4 ? 16 : 32 /* at most 32: the bits of a word */, NB = TT / 16, DB = DP / 16;
    static constexpr int EC = 16 / (int)sizeof(C), UR = DP / EC, NCH = Wide<T, C>::N;
    static constexpr int SU = TT * UR / 64;  // units of V a lane stages
    static constexpr int KU = UR / 4;        // units of K a lane loads of each of its rows
    static constexpr int OP = DP + 4;        // floats from pair to pair of a wave's results
    static constexpr int BUF = TT * PITCH > 16 * OP * 4 ? TT * PITCH : 16 * OP * 4;
    static constexpr int LDS = 4 * BUF + 4 * 16 * 2 * 4 + 4 * 3 * TT * 4;
    static constexpr int WAVES = PITCH > 256 ? 1 : 2;
    static_assert(SU >= 1 && TT * UR % 64 == 0 && KU >= 1, "staging");
};

template <typename T, typename C, int DP> __device__ __forceinline__ void attend_few(const sox_kv_attend_args& p, uint32_t block) {
    typedef Few<T, C, DP> F;
    typedef typename Frag<T>::V FV;
    constexpr bool QUANT = F::QUANT;
    constexpr int FORM = F::FORM;
    constexpr int TT = F::TT, NB = F::NB, DB = F::DB, E = F::E;
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quad = lane >> 4, col = lane & 15;
    const sox_kv_view& b = p.b;
    const int kvh = block % b.heads, rest = block / b.heads, splits = p.splits_few, split = rest % splits;
    const RowTile r = row_tile<16, false>(p, rest / splits, lane);
    if (!r.some) return;
    const Span s = span_of<16, TT>(p, r, split, splits, p.min_few);
    const int32_t* const table = b.tables + r.sequence * b.ldt;
    const int mask = (1 << b.shift) - 1;
    unsigned char* const lv = lds + wave * F::BUF;
    float* const ends = (float*)(lds + 4 * F::BUF);  // [wave][pair][reference, sum]
    float* const scales = ends + 4 * 16 * 2 + wave * 3 * TT;  // k's times the score's, log2 of v's rest, what v's are to p or the sum

    const int m = r.m0 + col;
    const bool mine = m < r.pairs;
    const int pos = mine ? (int)(r.length - r.rows + m / p.group) : -1, low = window_low(p, pos);
    FV qf[F::KU][F::NCH];
    {
        const T* const q = row_q<T>(p, r, kvh, mine ? m : r.m0);
#pragma unroll
        for (int u = 0; u < F::KU; u++)
#pragma unroll
            for (int n = 0; n < F::NCH; n++) qf[u][n] = load_q<T>(q, (4 * u + quad) * F::EC + n * E, b.dim, mine);
    }
    float4v out[DB];
#pragma unroll
    for (int d = 0; d < DB; d++) out[d] = float4v{};
    Soft<T> soft;

    int4v raw_k[NB][F::KU], raw_v[F::SU];
    float raw_s = 0.0f;  // lanes 0 .. TT - 1: K's scale of their token, TT .. 2 TT - 1: V's
    typedef int4v At __attribute__((aligned(4)));
    const uint32_t row_bytes = (uint32_t)b.dim * sizeof(C);
    const uint8_t* const head = b.pool + ((int64_t)kvh << b.shift) * row_bytes;
    const uint8_t* const head_s = b.pool + ((int64_t)kvh << b.shift) * 4;
    auto entry = [&](int t0) { return tile_entry(b, table, t0 + min(lane, TT - 1)); };
    auto page_of = [&](int t0, int entry) { return lane < TT ? tile_page(b, entry, t0 + lane, s.lo, s.end) : -1; };
    auto row_at = [&](int t0, int page, int row) { return head_rows(b, head, page, ((t0 + row) & mask) * row_bytes); };
    const int64_t scale_at = lane < TT ? b.ks_at : b.vs_at;
    const uint32_t lane_k = (uint32_t)(col * DP * (int)sizeof(C) + quad * 16);
    const bool wide_pages = b.shift >= 4 && b.dim == DP;  // 16 tokens of a tile seen whole stand in one page
    auto load = [&](int t0, int pages, bool part) {
        if (wide_pages && !part) {
#pragma unroll
            for (int n = 0; n < NB; n++) {
                const uint8_t* const at = head_rows(b, head, __builtin_amdgcn_readlane(pages, 16 * n), ((t0 + 16 * n) & mask) * (DP * (int)sizeof(C)));
#pragma unroll
                for (int u = 0; u < F::KU; u++) raw_k[n][u] = *(const At*)(at + u * 64 + lane_k);
            }
#pragma unroll
            for (int j = 0; j < F::SU; j++) {
                const int row = j * 64 / F::UR;
                const uint8_t* const at = head_rows(b, head, __builtin_amdgcn_readlane(pages, row), ((t0 + row) & mask) * (DP * (int)sizeof(C))) + b.v_at;
                raw_v[j] = *(const At*)(at + lane * 16);
            }
        } else {
#pragma unroll
            for (int n = 0; n < NB; n++) {
                const int row = 16 * n + col, page = __shfl(pages, row);
                const uint8_t* const at = row_at(t0, page, row);
#pragma unroll
                for (int u = 0; u < F::KU; u++) {
                    raw_k[n][u] = int4v{};
                    if (page >= 0 && (4 * u + quad) * F::EC < b.dim) raw_k[n][u] = *(const At*)(at + (4 * u + quad) * 16);
                }
            }
#pragma unroll
            for (int j = 0; j < F::SU; j++) {
                const int u = j * 64 + lane, row = u / F::UR, c = u % F::UR, page = __shfl(pages, row);
                raw_v[j] = int4v{};
                if (page >= 0 && c * F::EC < b.dim) raw_v[j] = *(const At*)(row_at(t0, page, row) + b.v_at + c * 16);
            }
        }
        if constexpr (QUANT) {
            const int page = __shfl(pages, lane & (TT - 1));
            raw_s = 0.0f;
            if (page >= 0 && lane < 2 * TT) raw_s = *(const float*)(head_rows(b, head_s, page, ((t0 + (lane & (TT - 1))) & mask) * 4) + scale_at);
        }
    };
    auto v_at = [&](int row, int ch) { return lv + row * F::PITCH + (((ch / E) ^ at_v<F::CH, sizeof(T), true>(row)) << 4) + ch % E * (int)sizeof(T); };

    const int stride = 4 * TT;
    int t0 = s.begin + wave * TT;
    int pages = page_of(t0, entry(t0)), next = entry(t0 + stride);
    auto in_part = [&](int t0, uint64_t valid) {  // a tile that not every row sees whole
        return t0 + TT - 1 > s.pos_first || t0 <= s.low_last || ~valid << (64 - TT) != 0;
    };
    uint64_t next_valid = __ballot(pages >= 0);
    bool next_part = in_part(t0, next_valid);
    if (t0 < s.end) load(t0, pages, next_part);
    for (; t0 < s.end; t0 += stride) {
        const uint64_t valid = next_valid;
        const bool part = next_part;
        const bool more = t0 + stride < s.end;
        // V's scales' powers of two, for what this lane stages: from the lanes that have the scales (TT .. 2 TT - 1), long before they are
        // used (64 single tokens with heads of 128: 165 us, 172 where they are)
        int power[F::SU];
        if constexpr (FORM == SCALE_EXPONENT) {
            const int mine = __builtin_bit_cast(int, scale_power2(raw_s));
#pragma unroll
            for (int j = 0; j < F::SU; j++) power[j] = __shfl(mine, TT + (j * 64 + lane) / F::UR);
        }
        if constexpr (QUANT) {
            if (lane < TT) {
                scales[lane] = raw_s * p.scale_log2;
            } else if (lane < 2 * TT) {
                if constexpr (FORM == SCALE_EXPONENT) {
                    const float v = scale_rest(raw_s);
                    scales[lane] = __builtin_amdgcn_logf(v);
                    scales[TT + lane] = __builtin_amdgcn_rcpf(v);
                } else {
                    scales[TT + lane] = raw_s;
                }
            }
        }
        // S^T = K Q^T: register e of block n is token t0 + 16 n + 4 quad + e
        float4v acc[NB];
        float4v vsc[NB];
#pragma unroll
        for (int n = 0; n < NB; n++) {
            acc[n] = float4v{};
#pragma unroll
            for (int u = 0; u < F::KU; u++) {
                const Wide<T, C> k = Wide<T, C>::of(raw_k[n][u]);
#pragma unroll
                for (int x = 0; x < F::NCH; x++) acc[n] = mma16<T>(k.v[x], qf[u][x], acc[n]);
                if constexpr (QUANT) __builtin_amdgcn_sched_barrier(0);
            }
        }
        bool special = false;
        if constexpr (!QUANT) {
            if (part) {
                bool bad = false;
#pragma unroll
                for (int j = 0; j < F::SU; j++) {
                    bad |= any_not_finite<T>(raw_v[j]);
                    raw_v[j] = finite_only<T>(raw_v[j]);
                }
                special = __any(bad);
            }
        }
        // tokens as this lane counts them, from its first one on: constants below
        const uint32_t there = (uint32_t)(valid >> (4 * quad));
        const int until = pos - t0 - 4 * quad, after = low - t0 - 4 * quad;
        auto seen = [&](int t) { return (t <= until) & (t > after) & (int)(there >> t & 1); };
        float x[NB][4];
#pragma unroll
        for (int n = 0; n < NB; n++) {
            float4v ks, lv;
            if constexpr (QUANT) ks = *(const float4v*)(scales + 16 * n + 4 * quad), vsc[n] = *(const float4v*)(scales + 2 * TT + 16 * n + 4 * quad);
            if constexpr (FORM == SCALE_EXPONENT) lv = *(const float4v*)(scales + TT + 16 * n + 4 * quad);
#pragma unroll
            for (int e = 0; e < 4; e++)
                x[n][e] = FORM == SCALE_EXPONENT ? __builtin_fmaf(acc[n][e], ks[e], lv[e]) : acc[n][e] * (QUANT ? ks[e] : p.scale_log2);
        }
        if (part) {
#pragma unroll
            for (int n = 0; n < NB; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const bool hidden = !seen(16 * n + e);
                    x[n][e] = hidden ? -__builtin_inff() : x[n][e];
                    if constexpr (QUANT) vsc[n][e] = hidden ? 0.0f : vsc[n][e];  // (it may be a NaN)
                }
        }
        float top = x[0][0];
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) top = fmaxf(top, x[n][e]);
        // V into LDS, the next tile's loads behind it
#pragma unroll
        for (int j = 0; j < F::SU; j++) {
            const int u = j * 64 + lane, row = u / F::UR, c = (u % F::UR) * F::NCH;
            Wide<T, C> v;
            if constexpr (FORM == SCALE_EXPONENT)
                v = Wide<T, C>::template of<true>(raw_v[j], __builtin_bit_cast(half2v, power[j]));
            else
                v = Wide<T, C>::of(raw_v[j]);
#pragma unroll
            for (int n = 0; n < F::NCH; n++) *(FV*)(lv + row * F::PITCH + (((c + n) ^ at_v<F::CH, sizeof(T), true>(row)) << 4)) = v.v[n];
            if constexpr (QUANT) __builtin_amdgcn_sched_barrier(0);
        }
        pages = page_of(t0 + stride, next);
        next = entry(t0 + 2 * stride);
        next_valid = __ballot(pages >= 0);
        next_part = in_part(t0 + stride, next_valid);
        if (more) load(t0 + stride, pages, next_part);
        if (__any(soft.passed(top))) {
            const float by = soft.move(over_32(over_16(top, larger), larger));
#pragma unroll
            for (int d = 0; d < DB; d++) {
                out[d] *= by;
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        const float ref = Soft<T>::of(soft.ref);
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[n][e] = __builtin_amdgcn_exp2f(x[n][e] - ref);
                soft.sum = FORM == SCALE_EXPONENT ? __builtin_fmaf(x[n][e], vsc[n][e], soft.sum) : soft.sum + x[n][e];
                if constexpr (FORM == SCALE_FACTOR) x[n][e] *= vsc[n][e];
            }
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int n = 0; n < NB; n += 2) {
                FV pf, left;  // p as it meets V, and over 8 bits what that leaves of it
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    pf[e] = (T)x[n + e / 4][e % 4];
                    if constexpr (QUANT) left[e] = (T)(x[n + e / 4][e % 4] - (float)pf[e]);
                }
                auto v_frag = [&](int d) {
                    const int row = 16 * n + 4 * quad + (col >> 2), ch = 16 * d + 4 * (lane & 3);
                    return join<T>(read_columns(v_at(row, ch)), read_columns(v_at(row + 16, ch)));
                };
#pragma unroll
                for (int d = 0; d < DB; d++) {
                    const FV v = v_frag(d);
                    out[d] = mfma16x16x32(v, pf, out[d]);
                    if constexpr (QUANT) out[d] = mfma16x16x32(v, left, out[d]);
                    if (d % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                }
            }
        } else {
#pragma unroll
            for (int n = 0; n < NB; n++)
#pragma unroll
                for (int e = 0; e < 4; e++)
#pragma unroll
                    for (int d = 0; d < DB; d++) {
                        out[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(*(const T*)v_at(16 * n + 4 * quad + e, 16 * d + col), x[n][e], out[d], 0, 0, 0);
                        if (d % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                    }
        }
        if constexpr (!QUANT) {
            if (special) {
#pragma unroll 1
                for (int t = 0; t < TT; t++) {
                    if (!((valid >> t) & 1)) continue;
                    const T* const v = (const T*)(row_at(t0, kv_page(b, table, t0 + t), t) + b.v_at);
                    if (t0 + t > pos || t0 + t <= low) continue;
#pragma unroll
                    for (int d = 0; d < DB; d++)
                        if (16 * d + 4 * quad < b.dim) out[d] += special4(v + 16 * d + 4 * quad);
                }
            }
        }
    }

    // ---- the waves' results joined ----
    soft.sum = over_32(over_16(soft.sum, added), added);
    float* const mine_o = (float*)lv + col * F::OP;
#pragma unroll
    for (int d = 0; d < DB; d++) *(float4v*)(mine_o + 16 * d + 4 * quad) = out[d];
    if (quad == 0) ends[(wave * 16 + col) * 2] = soft.ref, ends[(wave * 16 + col) * 2 + 1] = soft.sum;
    __syncthreads();
    for (int u = tid; u < 16 * (DP / 4); u += AT_THREADS) {
        const int pair = u / (DP / 4), ch = u % (DP / 4) * 4;
        if (r.m0 + pair >= r.pairs || ch >= b.dim || r.length - r.rows + (r.m0 + pair) / p.group < 0) continue;
        float ref = -__builtin_inff(), sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) ref = fmaxf(ref, ends[(w * 16 + pair) * 2]);
        float4v v = {};
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float l = ends[(w * 16 + pair) * 2 + 1], from = ends[(w * 16 + pair) * 2];
            const float by = l == 0.0f ? 0.0f : from == ref ? 1.0f : __builtin_amdgcn_exp2f(from - ref);
            sum += by * l;
            if (l != 0.0f) v += by * *(const float4v*)((const float*)(lds + w * F::BUF) + pair * F::OP + ch);
        }
        const RowOut<T> o = row_out<T>(p, r, kvh, r.m0 + pair, split);
        if (splits > 1) {
            if (ch == 0) o.ml[0] = ref, o.ml[1] = s.begin < s.end ? sum : -1.0f;
            if (s.begin < s.end) *(float4v*)(o.part + ch) = v;
        } else {
            store4(o.y + ch, v * (sum == 0.0f ? 0.0f : 1.0f / sum));
        }
    }
}

// =====================================================================================================================
// the splits' results joined
// =====================================================================================================================
// A row's splits: none where it is no sequence's, or has one and its result already, or a negative position (left alone)
SOX_DEV int merge_splits(const sox_kv_attend_args& p, int row, int lane) {
    const sox_kv_view& b = p.b;
    const int s = kv_sequence(b, row, lane);
    if (s < 0) return 0;
    const int first = min(max(b.starts[s], 0), b.rows), rows = max(min(b.starts[s + 1], b.rows) - first, 0);
    const int splits = (int64_t)rows * p.group > 16 ? p.splits_many : p.splits_few;
    return splits < 2 || (int64_t)max(b.lengths[s], 0) - rows + (row - first) < 0 ? 0 : splits;
}
// What a partial result counts, from its reference and sum (the sum of one without a token is 0)
SOX_DEV float merge_weight(float from, float l, float ref) { return l == 0.0f ? 0.0f : from == ref ? 1.0f : __builtin_amdgcn_exp2f(from - ref); }
constexpr int MERGE_WAVE = 8;  // results that a lane has on their way; splits that one lane joins alone

// A partial result takes dim / 4 lanes. Up to MERGE_WAVE of them: a wave for a row's 1, 2 or 4 heads, each lane its channels of all
// splits, and everything, whether the row turns out to need it or not, on its way at once (512 rows and 31 tokens of 32 heads, three
// splits: 9 us against 12 with a wave for each head that looked for its row first).
template <typename T> __device__ __forceinline__ void merge_wave(const sox_kv_attend_args& p) {
    const sox_kv_view& b = p.b;
    const int lane = threadIdx.x & 63, lanes = b.dim <= 64 ? 16 : b.dim <= 128 ? 32 : 64, heads = 64 / lanes, units = (p.q_heads + heads - 1) / heads;
    const uint32_t w = __builtin_amdgcn_readfirstlane(blockIdx.x * (AT_THREADS / 64) + threadIdx.x / 64);
    const int row = (int)(w / (uint32_t)units), head = (int)(w % (uint32_t)units) * heads + lane / lanes, ch = lane % lanes * 4;
    if (row >= b.rows) return;
    const bool mine = head < p.q_heads && ch < b.dim;
    const int64_t at = ((int64_t)row * p.q_heads + min(head, p.q_heads - 1)) * p.stride;
    const float* const part = p.part + at * b.dim + min(ch, b.dim - 4);
    float4v o[MERGE_WAVE];
    float from[MERGE_WAVE], l[MERGE_WAVE];
#pragma unroll
    for (int i = 0; i < MERGE_WAVE; i++)
        if (i < p.stride) {
            from[i] = p.ml[(at + i) * 2], l[i] = p.ml[(at + i) * 2 + 1];
            o[i] = *(const float4v*)(part + (int64_t)i * b.dim);
        }
    const int splits = merge_splits(p, row, lane);
    if (splits == 0) return;
    float ref = -__builtin_inff(), sum = 0.0f;
    float4v v = {};
#pragma unroll
    for (int i = 0; i < MERGE_WAVE; i++)
        if (i < splits && l[i] != -1.0f) ref = fmaxf(ref, from[i]);
#pragma unroll
    for (int i = 0; i < MERGE_WAVE; i++)
        if (i < splits && l[i] != -1.0f) {
            const float by = merge_weight(from[i], l[i], ref);
            sum += by * l[i];
            v += by * o[i];
        }
    if (mine) store4((T*)p.y + (int64_t)row * p.ldy + (int64_t)head * b.dim + ch, v * (sum == 0.0f ? 0.0f : 1.0f / sum));
}

// More: 256 threads for a (row, head), 256 / (dim / 4) results in flight for each load, eight loads at a time. A split that had no
// tokens left a sum of -1 and nothing else; such splits are the last.
template <typename T> __device__ __forceinline__ void attend_merge(const sox_kv_attend_args& p) {
    if (p.stride <= MERGE_WAVE) {
        merge_wave<T>(p);
        return;
    }
    const sox_kv_view& b = p.b;
    const int tid = threadIdx.x, lane = tid & 63, row = (int)(blockIdx.x / (uint32_t)p.q_heads), head = (int)(blockIdx.x % (uint32_t)p.q_heads);
    const int splits = merge_splits(p, row, lane);
    const int64_t at = ((int64_t)row * p.q_heads + head) * p.stride;
    const float* const ml = p.ml + at * 2;
    float ref = -__builtin_inff();
    int n = 0;
    for (int i0 = 0; i0 < splits; i0 += 64) {
        const bool some = i0 + lane < splits && ml[2 * (i0 + lane) + 1] != -1.0f;
        if (some) ref = fmaxf(ref, ml[2 * (i0 + lane)]);
        n += __popcll(__ballot(some));
    }
    for (int o = 1; o < 64; o <<= 1) ref = fmaxf(ref, __shfl_xor(ref, o));
    const int lanes = b.dim <= 64 ? 16 : b.dim <= 128 ? 32 : 64, groups = AT_THREADS / lanes;
    const int group = tid / lanes, ch = tid % lanes * 4;
    const float* const part = p.part + at * b.dim + ch;
    float sum = 0.0f;
    float4v v = {};
    for (int i0 = group; i0 < n; i0 += MERGE_WAVE * groups) {
        float4v o[MERGE_WAVE];
        float from[MERGE_WAVE], l[MERGE_WAVE];
#pragma unroll
        for (int k = 0; k < MERGE_WAVE; k++) {
            const int i = i0 + k * groups;
            o[k] = float4v{};
            from[k] = ref, l[k] = 0.0f;
            if (i < n) {
                from[k] = ml[2 * i], l[k] = ml[2 * i + 1];
                if (ch < b.dim) o[k] = *(const float4v*)(part + (int64_t)i * b.dim);
            }
        }
#pragma unroll
        for (int k = 0; k < MERGE_WAVE; k++) {
            const float by = merge_weight(from[k], l[k], ref);
            sum += by * l[k];
            v += by * o[k];
        }
    }
    __shared__ float4v all[AT_THREADS];
    __shared__ float sums[AT_THREADS];
    all[tid] = v;
    sums[tid] = sum;
    __syncthreads();
    if (splits == 0 || group || ch >= b.dim) return;
    for (int g = 1; g < groups; g++) {
        v += all[tid + g * lanes];
        sum += sums[tid + g * lanes];
    }
    store4((T*)p.y + (int64_t)row * p.ldy + (int64_t)head * b.dim + ch, v * (sum == 0.0f ? 0.0f : 1.0f / sum));
}

// A batch of both kinds in one launch: the many rows' workgroups, bound by the matrix cores, first (p.many, as many as a batch most
// often has), the single tokens' (p.few), bound by memory, beside and behind them, and last those that a batch may have at most and
// that mostly find nothing: ahead of the single tokens they cost 15 us of 110.
#define KV_ATTEND(NAME, T, C, DP)                                                                                              \
    extern "C" __global__ void __launch_bounds__(256, (Many<T, C, DP>::WAVES)) sox_kv_many_##NAME##_d##DP(sox_kv_attend_args p) { attend_many<T, C, DP>(p, blockIdx.x); } \
    extern "C" __global__ void __launch_bounds__(256, (Few<T, C, DP>::WAVES)) sox_kv_few_##NAME##_d##DP(sox_kv_attend_args p) { attend_few<T, C, DP>(p, blockIdx.x); } \
    extern "C" __global__ void __launch_bounds__(256, (Many<T, C, DP>::WAVES)) sox_kv_both_##NAME##_d##DP(sox_kv_attend_args p) {                                        \
        const uint32_t at = blockIdx.x, many = p.many, few = p.few;                                                            \
        if (at >= many && at < many + few)                                                                                     \
            attend_few<T, C, DP>(p, at - many);                                                                                \
        else                                                                                                                   \
            attend_many<T, C, DP>(p, at < many ? at : at - few);                                                               \
    }
#define KV_ATTEND_DIMS(NAME, T, C) KV_ATTEND(NAME, T, C, 64) KV_ATTEND(NAME, T, C, 128) KV_ATTEND(NAME, T, C, 256)
