// Rotary positions (sox_rotary_*), and the rows of a paged cache written (sox_kv_write_*) and read back (sox_kv_read_*).
// Bound by memory for many rows (8 bits written: by instructions) and by latency for few: a workgroup of 256 takes 1 or 4 rows,
// finds their tokens' pages (starts, then length and table entry: three loads that wait for each other, with the first rows'
// values on their way beside them), makes each row's table of cosines and sines once, and then walks its heads, a power of two
// of lanes for one head. That lanes' maximum of a head is its row's in 8 bits, so a row goes from memory to its page in one pass.
// 8192 rows of 40 heads of 128 in bf16 turn in 37 us from memory (4.6 TB/s); 16384 rows of 8 heads of 128 in 8 bits are read back in 20.
#include "kv_cache.h"

// A thread's (row, head)s, one after the other
struct Walk {
    int r, h, step, heads, rows;
    SOX_DEV Walk of(int first, int step, int heads, int rows) {
        Walk w{0, first - step, step, heads, rows};
        w.next();
        return w;
    }
    __device__ __forceinline__ void next() {
        h += step;
        while (h >= heads && r < rows) h -= heads, r++;
    }
    __device__ __forceinline__ bool some() const { return r < rows; }
};

// A lane takes two chunks of a head, `wide` channels apart, about half of the head. In a head that turns whole they are each
// other's pairs: nothing is loaded or converted twice, and what a chunk costs beside its values is paid once for two.
template <typename T, typename F> struct Halves {
    static constexpr int V = 16 / sizeof(T);
    int wide, ch0, ch1;
    bool some0, some1, pairs;
    SOX_DEV Halves of(int dim, const sox_turn_args& t, int sub) {
        Halves l;
        l.wide = (dim / 2 + V - 1) / V * V;
        l.ch0 = sub * V;
        l.ch1 = l.ch0 + l.wide;
        l.some0 = l.ch0 < l.wide;
        l.some1 = l.some0 && l.ch1 < dim;
        l.pairs = t.half == l.wide && dim == 2 * l.wide && !t.interleaved;
        return l;
    }
};
template <typename T, typename F> struct Two {
    TurnedChunk<T, F> a, b;
    __device__ __forceinline__ void load(const Halves<T, F>& l, const T* head, const sox_turn_args& t, bool turned) {
        if (!l.some0) return;
        const int half = turned && !l.pairs ? t.half : 0;
        a.load(head, l.ch0, t, half);
        if (l.some1) b.load(head, l.ch1, t, half);
    }
    __device__ __forceinline__ void turn(const Halves<T, F>& l, const sox_turn_args& t, bool turned, const CosSin<F>* table) {
        if (!l.some0) return;
        if (turned && l.pairs) {
            TurnedChunk<T, F>::turn_pairs(a, b, l.ch0, table);
        } else {
            a.turn(l.ch0, t, turned ? t.half : 0, table);
            if (l.some1) b.turn(l.ch1, t, turned ? t.half : 0, table);
        }
    }
    __device__ __forceinline__ void store(const Halves<T, F>& l, T* head) const {
        if (l.some0) a.store(head, l.ch0);
        if (l.some1) b.store(head, l.ch1);
    }
};

template <typename T> __device__ __forceinline__ void rotary_body(const sox_rotary_args& p) {
    typedef typename std::conditional<sizeof(T) == 4, double, float>::type F;
    __shared__ CosSin<F> table[4][TURN_HALF];
    const int tid = threadIdx.x, rpb = p.rows_per_block, row0 = blockIdx.x * rpb, rows = min(rpb, p.rows - row0);
    const Halves<T, F> l = Halves<T, F>::of(p.dim, p.turn, tid & ((1 << p.lanes) - 1));
    Walk w = Walk::of(tid >> p.lanes, 256 >> p.lanes, p.heads, rows);
    Two<T, F> next;
    auto load = [&] {
        if (w.some()) next.load(l, (const T*)p.x + (row0 + w.r) * p.ldx + (int64_t)w.h * p.dim, p.turn, true);
    };
    load();
    turn_tables<16 / sizeof(T)>(p.turn, [&](int r) { return p.positions[row0 + r]; }, table, rows, tid, 256);
    __syncthreads();
    while (w.some()) {
        Two<T, F> c = next;
        const int r = w.r, h = w.h;
        w.next();
        load();
        c.turn(l, p.turn, true, table[r]);
        c.store(l, (T*)p.y + (row0 + r) * p.ldy + (int64_t)h * p.dim);
    }
}

// A row's token: -2 where the row is no sequence's (left alone), else its position, and its place in its page
struct RowAt {
    int64_t page;  // -1: no page holds it
    int64_t position;
};
SOX_DEV RowAt row_at(const sox_kv_view& b, int row, int lane) {
    const int s = kv_sequence(b, row, lane);
    if (s < 0) return {-1, -2};
    const int64_t position = (int64_t)b.lengths[s] - b.starts[s + 1] + row;
    if (position < 0) return {-1, -2};
    return {kv_page(b, b.tables + s * b.ldt, position), position};
}

constexpr int KV_ROWS = 4;  // of a workgroup at most

// Bound by its instructions in 8 bits: 16384 rows of 8 heads of 128 from bf16 take 37 us (42 with one chunk a lane), and the memory's
// share of that is 20.
template <typename T, typename C> __device__ __forceinline__ void kv_write_body(const sox_kv_rows_args& p) {
    constexpr bool QUANT = sizeof(C) == 1;
    typedef typename std::conditional<QUANT || sizeof(T) == 4, double, float>::type F;
    constexpr int V = 16 / sizeof(T);
    __shared__ CosSin<F> table[KV_ROWS][TURN_HALF];
    __shared__ RowAt where[KV_ROWS];
    const sox_kv_view& b = p.b;
    const int tid = threadIdx.x, lane = tid & 63, rpb = p.rows_per_block, row0 = blockIdx.x * rpb, rows = min(rpb, b.rows - row0);
    const int sub = tid & ((1 << p.lanes) - 1), half = p.turn.half;
    const Halves<T, F> l = Halves<T, F>::of(b.dim, p.turn, sub);
    Walk w = Walk::of(tid >> p.lanes, 256 >> p.lanes, p.q_heads + 2 * b.heads, rows);
    Two<T, F> next;  // on its way while the one before is worked on, the first while the rows' pages are looked for
    auto load = [&] {
        if (!w.some()) return;
        const bool q = w.h < p.q_heads, k = w.h < p.q_heads + b.heads;
        const int64_t ld = q ? p.ldq : k ? p.ldk : p.ldv;
        const T* const from = (const T*)(q ? p.q : k ? p.k : p.v) + (row0 + w.r) * ld + (q ? w.h : w.h - p.q_heads - (k ? 0 : b.heads)) * b.dim;
        next.load(l, from, p.turn, k);
    };
    load();
    for (int r = tid >> 6; r < rows; r += 4) {
        const RowAt at = row_at(b, row0 + r, lane);
        if (lane == 0) where[r] = at;
    }
    __syncthreads();
    if (half) turn_tables<V>(p.turn, [&](int r) { return where[r].position; }, table, rows, tid, 256);
    __syncthreads();
    while (w.some()) {
        Two<T, F> c = next;
        const int r = w.r, h = w.h;
        w.next();
        load();
        const bool is_q = h < p.q_heads, is_k = h < p.q_heads + b.heads;
        const int head = is_q ? h : h - p.q_heads - (is_k ? 0 : b.heads);
        const RowAt at = where[r];
        if (at.position < 0 || (at.page < 0 && !is_q)) continue;
        const bool turned = is_k && half;
        c.turn(l, p.turn, turned, table[r]);
        if (is_q) {
            c.store(l, (T*)p.y + (row0 + r) * p.ldy + head * b.dim);
            continue;
        }
        const int64_t token = ((int64_t)head << b.shift) + (at.position & ((1 << b.shift) - 1));
        uint8_t* const page = b.pool + at.page * b.page_bytes;
        C* const to = (C*)(page + (is_k ? 0 : b.v_at)) + token * b.dim;
        if constexpr (!QUANT) {
            c.store(l, (T*)to);
        } else {
            float v[2 * V];
#pragma unroll
            for (int e = 0; e < V; e++) v[e] = l.some0 ? c.a.v[e] : 0.0f, v[V + e] = l.some1 ? c.b.v[e] : 0.0f;
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 2 * V; e++) top = max(top, abs_bits(v[e]));
            for (int o = 1; o < 1 << p.lanes; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
            float scale;
            uint32_t q[V / 2];
            bool sure = false;
            if (turned) {  // (of full precision, whatever T is)
                // In fp32 first: 127 / amax and its product with x are off by less than 2^-15 for a result up to 127, so one
                // that is at least 2^-14 from the middle between two integers rounds as the exact one does. About one wave's
                // chunks in 15 have a value that is nearer and take the steps in 64 bits, as rows at fp32's ends do.
                const float a = __uint_as_float(top), by = 127.0f / a;
                float far = 0.0f;
                uint32_t low[2 * V];
#pragma unroll
                for (int e = 0; e < 2 * V; e++) {
                    const float x = v[e] * by, up = x + 12582912.0f;
                    low[e] = __float_as_uint(up);
                    far = fmaxf(far, fabsf(x - (up - 12582912.0f)));
                }
                sure = !__any(!(far < 0.5f - 0x1p-14f) || !(a > 0x1p-60f && a < 0x1p60f));
                if (sure) {
                    scale = a / 127.0f;
#pragma unroll
                    for (int e = 0; e < 2 * V; e += 4)
                        q[e / 4] = __builtin_amdgcn_perm(low[e + 1], low[e], 0x0c0c0400) | __builtin_amdgcn_perm(low[e + 3], low[e + 2], 0x04000c0c);
                }
            }
            auto exact = [&](const auto& by) {
                typedef typename std::decay<decltype(by)>::type Q;
#pragma unroll
                for (int e = 0; e < 2 * V; e += 4) q[e / 4] = Q::q4(v[e], v[e + 1], v[e + 2], v[e + 3], by);
                scale = by.scale;
            };
            if (!turned)
                exact(RowQuant<T>::make(top));
            else if (!sure)
                exact(RowQuant<float>::make(top));
            typedef uint32_t Q4 __attribute__((ext_vector_type(V / 4)));
            typedef Q4 At __attribute__((aligned(4)));
            Q4 q0, q1;
#pragma unroll
            for (int e = 0; e < V / 4; e++) q0[e] = q[e], q1[e] = q[V / 4 + e];
            if (l.some0) *(At*)(to + l.ch0) = q0;
            if (l.some1) *(At*)(to + l.ch1) = q1;
            if (sub == 0) ((float*)(page + (is_k ? b.ks_at : b.vs_at)))[token] = scale;
        }
    }
}

template <typename T, typename C> __device__ __forceinline__ void kv_read_body(const sox_kv_rows_args& p) {
    constexpr int V = 16 / sizeof(T);
    __shared__ RowAt where[KV_ROWS];
    const sox_kv_view& b = p.b;
    const int tid = threadIdx.x, lane = tid & 63, rpb = p.rows_per_block, row0 = blockIdx.x * rpb, rows = min(rpb, b.rows - row0);
    for (int r = tid >> 6; r < rows; r += 4) {
        const RowAt at = row_at(b, row0 + r, lane);
        if (lane == 0) where[r] = at;
    }
    __syncthreads();
    const int ch = (tid & ((1 << p.lanes) - 1)) * V;
    if (ch >= b.dim) return;
    typedef typename Chunk16<T>::V TV;
    typedef int8_t Bytes __attribute__((ext_vector_type(V)));
    typedef Bytes BytesAt __attribute__((aligned(4)));
    Walk w = Walk::of(tid >> p.lanes, 256 >> p.lanes, 2 * b.heads, rows);
    struct Chunk {
        TV v;
        Bytes q;
        float scale;
    };
    auto load = [&](Chunk& c) {
        c.v = TV{};
        c.q = Bytes{};
        c.scale = 0.0f;
        if (!w.some()) return;
        const RowAt at = where[w.r];
        if (at.page < 0) return;
        const bool is_k = w.h < b.heads;
        const int64_t token = ((int64_t)(is_k ? w.h : w.h - b.heads) << b.shift) + (at.position & ((1 << b.shift) - 1));
        const uint8_t* const page = b.pool + at.page * b.page_bytes;
        const C* const from = (const C*)(page + (is_k ? 0 : b.v_at)) + token * b.dim + ch;
        if constexpr (sizeof(C) == 1) {
            c.scale = ((const float*)(page + (is_k ? b.ks_at : b.vs_at)))[token];
            c.q = *(const BytesAt*)from;
        } else {
            c.v = *(const typename Chunk16<T>::At*)from;
        }
    };
    Chunk next;
    load(next);
    while (w.some()) {  // (a chunk's loads on their way while the one before is stored)
        Chunk c = next;
        const int r = w.r, h = w.h;
        w.next();
        load(next);
        if (where[r].position < 0) continue;
        if constexpr (sizeof(C) == 1) {
#pragma unroll
            for (int e = 0; e < V; e++) c.v[e] = (T)((float)c.q[e] * c.scale);
        }
        T* const to = (h < b.heads ? (T*)p.k + (int64_t)(row0 + r) * p.ldk + (int64_t)h * b.dim : (T*)p.v + (int64_t)(row0 + r) * p.ldv + (int64_t)(h - b.heads) * b.dim) + ch;
        *(typename Chunk16<T>::At*)to = c.v;
    }
}

#define KV_ROWS_KERNELS(NAME, T)                                                                                              \
    extern "C" __global__ void __launch_bounds__(256) sox_rotary_##NAME(sox_rotary_args p) { rotary_body<T>(p); }             \
    extern "C" __global__ void __launch_bounds__(256) sox_kv_write_##NAME(sox_kv_rows_args p) { kv_write_body<T, T>(p); }     \
    extern "C" __global__ void __launch_bounds__(256) sox_kv_write_##NAME##_i8(sox_kv_rows_args p) { kv_write_body<T, int8_t>(p); } \
    extern "C" __global__ void __launch_bounds__(256) sox_kv_read_##NAME(sox_kv_rows_args p) { kv_read_body<T, T>(p); }       \
    extern "C" __global__ void __launch_bounds__(256) sox_kv_read_##NAME##_i8(sox_kv_rows_args p) { kv_read_body<T, int8_t>(p); }
KV_ROWS_KERNELS(f16, half_t)
KV_ROWS_KERNELS(bf16, bf16_t)
KV_ROWS_KERNELS(f32, float)
