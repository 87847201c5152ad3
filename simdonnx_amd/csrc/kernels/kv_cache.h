// What the kernels of the paged cache share: where a row's token is, and the rotation by position.
#pragma once
#include "qrows.h"

// ---- where a token is ----

// The sequence whose rows hold `row`, or -1; the same in all lanes. All of a wave's loads of `starts` are in flight at once,
// where a binary search would wait for each.
SOX_DEV int kv_sequence(const sox_kv_view& b, int row, int lane) {
    int s = 0;
    for (int c = 0; c < b.sequences; c += 64) {
        const bool past = c + lane < b.sequences && b.starts[c + lane + 1] <= row;
        s += __popcll(__ballot(past));
    }
    s = __builtin_amdgcn_readfirstlane(s);
    return s < b.sequences && b.starts[s] <= row ? s : -1;
}

// The page of a sequence's token, or -1 where no page of the pool holds it
SOX_DEV int kv_page(const sox_kv_view& b, const int32_t* table, int64_t token) {
    if (token < 0 || (token >> b.shift) >= b.table_pages) return -1;
    const int page = table[token >> b.shift];
    return (uint32_t)page < (uint32_t)b.pages ? page : -1;
}

// ---- the rotation ----

// cos and sin of t / 2^64 of a turn: t less its nearest quarter turn, as an angle of [-pi / 4, pi / 4], in their Taylor series
// (the first terms left out are below 2e-14), and the quarter's signs. The product position * turns[j] in whole numbers keeps
// the fraction of a turn exactly, however far the position (its error is the position times turns[j]'s, half of 2^-64 of a turn
// and the frequency times 2^-107), and 64 bits leave nothing next to the borders of a value's 8-bit form.
SOX_DEV void turn_cos_sin(uint64_t t, double& c, double& s) {
    const uint64_t quarter = (t + (1ull << 61)) >> 62;
    const int64_t r = (int64_t)(t - (quarter << 62));
    const double x = ((double)(int32_t)(r >> 32) * 4294967296.0 + (double)(uint32_t)r) * 3.4061215800865545e-19;  // 2 pi / 2^64
    const double z = x * x;
    double a = 1.0 / 6227020800.0, b = -1.0 / 87178291200.0;
    a = __builtin_fma(a, z, -1.0 / 39916800.0);
    a = __builtin_fma(a, z, 1.0 / 362880.0);
    a = __builtin_fma(a, z, -1.0 / 5040.0);
    a = __builtin_fma(a, z, 1.0 / 120.0);
    a = __builtin_fma(a, z, -1.0 / 6.0);
    a = __builtin_fma(a * z, x, x);
    b = __builtin_fma(b, z, 1.0 / 479001600.0);
    b = __builtin_fma(b, z, -1.0 / 3628800.0);
    b = __builtin_fma(b, z, 1.0 / 40320.0);
    b = __builtin_fma(b, z, -1.0 / 720.0);
    b = __builtin_fma(b, z, 1.0 / 24.0);
    b = __builtin_fma(b, z, -0.5);
    b = __builtin_fma(b, z, 1.0);
    const bool swap = quarter & 1;
    c = swap ? a : b;
    s = swap ? b : a;
    if ((quarter + 1) & 2) c = -c;
    if (quarter & 2) s = -s;
}

template <typename F> struct CosSin {
    F c, s;
};
constexpr int TURN_HALF = 128;  // pairs of a head at most

// Rows' tables of cosines and sines. Pair j stands at turn_at<V>(j), V channels a lane: side by side what lanes of a head read
// at once (in order, they would read a bank's words 8 deep, and that took longer than the memory).
template <int V> SOX_DEV int turn_at(int j) { return j % V * (TURN_HALF / V) + j / V; }
template <int V, typename F, class P>
SOX_DEV void turn_tables(const sox_turn_args& t, P position, CosSin<F> (*table)[TURN_HALF], int rows, int thread, int threads) {
    int r = 0, j = thread;
    for (;; j += threads) {
        while (j >= t.half && r < rows) j -= t.half, r++;
        if (r >= rows) break;
        double c, s;
        turn_cos_sin((uint64_t)position(r) * t.turns[j], c, s);
        table[r][turn_at<V>(j)] = {(F)(c * t.amplitude), (F)(s * t.amplitude)};
    }
}

// 16 bytes of a head, channels ch .. ch + V - 1 of it, turned: y[c] = x[c] cos - x[c'] sin for the first channel of a pair,
// x[c] cos + x[c'] sin for the second, c' the other one. Each lane takes its channels' others from memory again (they are in
// L1) rather than pairs of chunks, so that any even number of channels turns by the same code. `head` may be written by the
// wave that reads it: all of its lanes' loads come before their stores.
template <typename T, typename F> struct TurnedChunk {
    static constexpr int V = 16 / sizeof(T);
    typedef typename Chunk16<T>::V TV;
    typedef typename Chunk16<T>::At At;
    TV own, other;
    float v[V];
    __device__ __forceinline__ void load(const T* head, int ch, const sox_turn_args& t, int half) {
        own = *(const At*)(head + ch);
        const int end = 2 * half;
        if (half == 0 || ch >= end || t.interleaved) return;
        if (half % V == 0) {
            other = *(const At*)(head + (ch < half ? ch + half : ch - half));
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) {
                const int c = ch + e, at = c >= end ? c : c < half ? c + half : c - half;
                other[e] = head[at];
            }
        }
    }
    __device__ __forceinline__ void turn(int ch, const sox_turn_args& t, int half, const CosSin<F>* table) {
        const int end = 2 * half;
        if (ch >= end) {
#pragma unroll
            for (int e = 0; e < V; e++) v[e] = (float)own[e];
            return;
        }
        constexpr int NEXT = TURN_HALF / V;
        if (!t.interleaved && half % V == 0) {  // (the usual heads: one place in the table, and what follows it at constant steps)
            const bool first = ch < half;
            const CosSin<F>* const at = table + (first ? ch : ch - half) / V;
#pragma unroll
            for (int e = 0; e < V; e++) v[e] = turned(own[e], first ? -other[e] : other[e], at[e * NEXT]);
        } else if (t.interleaved && end % V == 0) {
            const int j = ch >> 1;
            const CosSin<F>* const at = table + turn_at<V>(j);
#pragma unroll
            for (int e = 0; e < V; e++) v[e] = turned(own[e], e & 1 ? own[e ^ 1] : -own[e ^ 1], at[(e >> 1) * NEXT]);
        } else {
            if (t.interleaved) {
#pragma unroll
                for (int e = 0; e < V; e++) other[e] = own[e ^ 1];
            }
#pragma unroll
            for (int e = 0; e < V; e++) {
                const int c = ch + e, j = t.interleaved ? c >> 1 : c < half ? c : c - half;
                const bool first = t.interleaved ? !(e & 1) : c < half;
                const float y = turned(own[e], first ? -other[e] : other[e], table[turn_at<V>(min(j, half - 1))]);
                v[e] = c < end ? y : (float)own[e];
            }
        }
    }
    // Two chunks of a head that are each other's pairs, a the first ones
    SOX_DEV void turn_pairs(TurnedChunk& a, TurnedChunk& b, int ch, const CosSin<F>* table) {
        const CosSin<F>* const at = table + ch / V;
#pragma unroll
        for (int e = 0; e < V; e++) {
            const CosSin<F> by = at[e * (TURN_HALF / V)];
            a.v[e] = turned(a.own[e], -b.own[e], by);
            b.v[e] = turned(b.own[e], a.own[e], by);
        }
    }
    SOX_DEV float turned(T x, T other, CosSin<F> by) {
        if constexpr (sizeof(F) == 8)
            return (float)__builtin_fma((double)(float)other, by.s, (double)(float)x * by.c);
        else
            return __builtin_fmaf((float)other, by.s, (float)x * by.c);
    }
    __device__ __forceinline__ void store(T* head, int ch) const {
        TV o;
#pragma unroll
        for (int e = 0; e < V; e++) o[e] = (T)v[e];
        *(typename Chunk16<T>::At*)(head + ch) = o;
    }
};
