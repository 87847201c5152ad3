// Rotary positions (sox_rotary_*), and the rows of a paged cache written (sox_kv_write_*) and read back (sox_kv_read_*).
// Bound by memory for many rows and by latency for few: a workgroup of 256 takes 1 or 4 rows, finds their tokens' pages
// (starts, then length and table entry: three loads that wait for each other), makes each row's table of cosines and sines
// once, and then walks its heads, a power of two of lanes with 16 bytes each for one head. That lanes' maximum of a head is
// its row's in 8 bits, so a row goes from memory to its page in one pass.
#include "kv_cache.h"

template <typename T> __device__ __forceinline__ void rotary_body(const sox_rotary_args& p) {
    typedef typename std::conditional<sizeof(T) == 4, double, float>::type F;
    constexpr int V = 16 / sizeof(T);
    __shared__ CosSin<F> table[4][TURN_HALF];
    const int tid = threadIdx.x, rpb = p.rows_per_block, row0 = blockIdx.x * rpb, rows = min(rpb, p.rows - row0);
    for (int r = 0; r < rows; r++) turn_table(p.turn, p.positions[row0 + r], table[r], tid, 256);
    __syncthreads();
    const int ch = (tid & ((1 << p.lanes) - 1)) * V, step = 256 >> p.lanes;
    int r = 0, h = tid >> p.lanes;
    for (;; h += step) {
        while (h >= p.heads && r < rows) h -= p.heads, r++;
        if (r >= rows) break;
        if (ch >= p.dim) continue;
        const int64_t at = (int64_t)h * p.dim, row = row0 + r;
        TurnedChunk<T, F> c;
        c.load((const T*)p.x + row * p.ldx + at, ch, p.turn, table[r]);
        c.store((T*)p.y + row * p.ldy + at, ch);
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

template <typename T, typename C> __device__ __forceinline__ void kv_write_body(const sox_kv_rows_args& p) {
    constexpr bool QUANT = sizeof(C) == 1;
    typedef typename std::conditional<QUANT || sizeof(T) == 4, double, float>::type F;
    constexpr int V = 16 / sizeof(T);
    __shared__ CosSin<F> table[KV_ROWS][TURN_HALF];
    __shared__ RowAt where[KV_ROWS];
    const sox_kv_view& b = p.b;
    const int tid = threadIdx.x, lane = tid & 63, rpb = p.rows_per_block, row0 = blockIdx.x * rpb, rows = min(rpb, b.rows - row0);
    for (int r = tid >> 6; r < rows; r += 4) {
        const RowAt at = row_at(b, row0 + r, lane);
        if (lane == 0) where[r] = at;
    }
    __syncthreads();
    if (p.turn.half)
        for (int r = 0; r < rows; r++) turn_table(p.turn, where[r].position, table[r], tid, 256);
    __syncthreads();
    const int sub = tid & ((1 << p.lanes) - 1), ch = sub * V, step = 256 >> p.lanes, heads = p.q_heads + 2 * b.heads;
    const sox_turn_args straight{nullptr, 1.0, 0, 0};
    int r = 0, h = tid >> p.lanes;
    for (;; h += step) {
        while (h >= heads && r < rows) h -= heads, r++;
        if (r >= rows) break;
        const int64_t row = row0 + r;
        const RowAt at = where[r];
        if (at.position < 0) continue;
        TurnedChunk<T, F> c;
        if (h < p.q_heads) {
            if (ch >= b.dim) continue;
            c.load((const T*)p.q + row * p.ldq + (int64_t)h * b.dim, ch, p.turn, table[r]);
            c.store((T*)p.y + row * p.ldy + (int64_t)h * b.dim, ch);
            continue;
        }
        if (at.page < 0) continue;
        const bool is_k = h < p.q_heads + b.heads;
        const int kh = h - p.q_heads - (is_k ? 0 : b.heads);
        const T* from = is_k ? (const T*)p.k + row * p.ldk : (const T*)p.v + row * p.ldv;
        from += (int64_t)kh * b.dim;
        const int64_t token = ((int64_t)kh << b.shift) + (at.position & ((1 << b.shift) - 1));
        uint8_t* const page = b.pool + at.page * b.page_bytes;
        C* const to = (C*)(page + (is_k ? 0 : b.v_at)) + token * b.dim;
        if (ch < b.dim) c.load(from, ch, is_k ? p.turn : straight, table[r]);
        if constexpr (!QUANT) {
            if (ch < b.dim) c.store((T*)to, ch);
        } else {
            uint32_t top = 0;
            if (ch < b.dim)
#pragma unroll
                for (int e = 0; e < V; e++) top = max(top, abs_bits(c.v[e]));
            for (int o = 1; o < 1 << p.lanes; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
            const RowQuant<float> q = RowQuant<float>::make(top);
            if (ch < b.dim) {
#pragma unroll
                for (int e = 0; e < V; e += 4)
                    *(uint32_t*)(to + ch + e) = RowQuant<float>::q4(c.v[e], c.v[e + 1], c.v[e + 2], c.v[e + 3], q);
            }
            if (sub == 0) ((float*)(page + (is_k ? b.ks_at : b.vs_at)))[token] = q.scale;
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
    const int ch = (tid & ((1 << p.lanes) - 1)) * V, step = 256 >> p.lanes, heads = 2 * b.heads;
    int r = 0, h = tid >> p.lanes;
    for (;; h += step) {
        while (h >= heads && r < rows) h -= heads, r++;
        if (r >= rows) break;
        if (ch >= b.dim) continue;
        const int64_t row = row0 + r;
        const RowAt at = where[r];
        if (at.position < 0) continue;
        const bool is_k = h < b.heads;
        const int kh = is_k ? h : h - b.heads;
        T* const to = (is_k ? (T*)p.k + row * p.ldk : (T*)p.v + row * p.ldv) + (int64_t)kh * b.dim + ch;
        typedef typename Chunk16<T>::V TV;
        TV o = {};
        if (at.page >= 0) {
            const int64_t token = ((int64_t)kh << b.shift) + (at.position & ((1 << b.shift) - 1));
            const uint8_t* const page = b.pool + at.page * b.page_bytes;
            const C* const from = (const C*)(page + (is_k ? 0 : b.v_at)) + token * b.dim + ch;
            if constexpr (sizeof(C) == 1) {
                const float scale = ((const float*)(page + (is_k ? b.ks_at : b.vs_at)))[token];
                typedef int8_t Bytes __attribute__((ext_vector_type(V)));
                typedef Bytes BytesAt __attribute__((aligned(4)));
                const Bytes q = *(const BytesAt*)from;
#pragma unroll
                for (int e = 0; e < V; e++) o[e] = (T)((float)q[e] * scale);
            } else {
                o = *(const typename Chunk16<T>::At*)from;
            }
        }
        *(typename Chunk16<T>::At*)to = o;
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
