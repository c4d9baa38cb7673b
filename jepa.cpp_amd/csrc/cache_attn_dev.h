// cache_attn_dev.h - what the kernels that read the 4-bit paged cache share: codes to f16, queries to f16, the running softmax of 64 keys x 16
// columns, the product with V, and results of several workgroups joined by the last of them.
#pragma once
#include "cache_dev.h"
#include "kernels.h"
#include "lds_dma.h"

namespace {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef float float8_t __attribute__((ext_vector_type(8)));
typedef int int2_t __attribute__((ext_vector_type(2)));
typedef uint32_t word2_t __attribute__((ext_vector_type(2)));
typedef uint32_t word3_t __attribute__((ext_vector_type(3)));
typedef uint32_t word4_t __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.4426950408889634f;
constexpr int NT = 256;              // threads of a workgroup
constexpr int TILE = 64;             // keys of a wave's step
// the 8 codes of a word less 8, in the order of its elements (nibbles 0 4 1 5 2 6 3 7), exact in f16: a nibble or'ed into the low
// mantissa bits of 1024 is 1024 + c, into the next four 1024 + 16 c. `k1024` is the pair of f16 1024 in a vector register (an
// instruction reads one scalar register: with the mask in it, and + or are one v_and_or_b32).
__device__ __forceinline__ half8_t codes8(uint32_t w, uint32_t k1024) {
    const half2_t off = {(_Float16) -1032.0f, (_Float16) -1032.0f}, off16 = {(_Float16) -72.0f, (_Float16) -72.0f};
    const half2_t sixteenth = {(_Float16) 0.0625f, (_Float16) 0.0625f};
    const uint32_t u = w >> 8;
    const half2_t a = __builtin_bit_cast(half2_t, (w & 0x000f000fu) | k1024) + off;
    const half2_t b = __builtin_elementwise_fma(__builtin_bit_cast(half2_t, (w & 0x00f000f0u) | k1024), sixteenth, off16);
    const half2_t c = __builtin_bit_cast(half2_t, (u & 0x000f000fu) | k1024) + off;
    const half2_t d = __builtin_elementwise_fma(__builtin_bit_cast(half2_t, (u & 0x00f000f0u) | k1024), sixteenth, off16);
    return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The codes of a word in the order of its elements as f16 subnormals, without less 8: c 2^-24, elements 2, 3, 6 and 7 sixteen times that. The matrix
// instruction takes subnormals as they are, and half the work of codes8 goes where the other operand can hold the factors and the sum the offset.
__device__ __forceinline__ half8_t raw8(uint32_t w) {
    const uint32_t u = w >> 8;
    const word4_t x = {w & 0x000f000fu, w & 0x00f000f0u, u & 0x000f000fu, u & 0x00f000f0u};
    return __builtin_bit_cast(half8_t, x);
}

// the largest over the four lanes l, l ^ 16, l ^ 32, l ^ 48 (the lanes of one column)
__device__ __forceinline__ float col_max(float x) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// the largest over the 16 lanes of a row: mirrored, mirrored in halves, in quads, in pairs
__device__ __forceinline__ float row_max16(float x) {
#define DPP(ctrl) __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), ctrl, 0xf, 0xf, true))
    x = fmaxf(x, DPP(0x140));
    x = fmaxf(x, DPP(0x141));
    x = fmaxf(x, DPP(0x1b));
    return fmaxf(x, DPP(0xb1));
#undef DPP
}

// N words per lane of a buffer
template <int N>
__device__ __forceinline__ void load_words(uint32_t * x, brsrc r, int at, int off) {
    if constexpr (N == 1) x[0] = __builtin_amdgcn_raw_buffer_load_b32(r, at, off, 0);
    if constexpr (N == 2) { const word2_t v = __builtin_amdgcn_raw_buffer_load_b64(r, at, off, 0); x[0] = v[0]; x[1] = v[1]; }
    if constexpr (N == 3) { const word3_t v = __builtin_amdgcn_raw_buffer_load_b96(r, at, off, 0); x[0] = v[0]; x[1] = v[1]; x[2] = v[2]; }
    if constexpr (N == 4) { const word4_t v = __builtin_amdgcn_raw_buffer_load_b128(r, at, off, 0); x[0] = v[0]; x[1] = v[1]; x[2] = v[2]; x[3] = v[3]; }
}
__device__ __forceinline__ float col_sum(float x) {      // (the same of sums)
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ void wave_order() {      // LDS accesses of the wave's lanes before and after stay in this order
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// one sequence of the call, within the call's buffers whatever the arrays hold
struct seq_view { int32_t row0, rows, len; };
__device__ __forceinline__ seq_view view_of(const int32_t * row_start, const int32_t * kv_len, int64_t n_rows, int width, int page_size, int i) {
    seq_view v;
    const int32_t n = (int32_t) n_rows;
    v.row0 = min(max(row_start[i], 0), n);
    v.rows = max(min(max(row_start[i + 1], 0), n) - v.row0, 0);
    const int64_t cap = (int64_t) width * page_size;
    v.len = (int32_t) min<int64_t>(max(kv_len[i], 0), cap);
    return v;
}
template <typename A> __device__ __forceinline__ seq_view view_of(const A & a, int i) { return view_of(a.row_start, a.kv_len, a.n_rows, a.width, a.page_size, i); }

__device__ __forceinline__ int32_t uniform(int32_t x) { return __builtin_amdgcn_readfirstlane(x); }
// sums over the lanes up to this one, and over all of them, in the VALU: within rows of 16 lanes, then across rows
template <typename X>
__device__ __forceinline__ X wave_scan(X x) {
    static_assert(sizeof(X) == 4, "one register");
#define DPP(ctrl, rows) __builtin_bit_cast(X, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), ctrl, rows, 0xf, true))
    x += DPP(0x111, 0xf);      // row_shr 1, 2, 4, 8
    x += DPP(0x112, 0xf);
    x += DPP(0x114, 0xf);
    x += DPP(0x118, 0xf);
    x += DPP(0x142, 0xa);      // row_bcast 15, 31
    x += DPP(0x143, 0xc);
#undef DPP
    return x;
}
template <typename X>
__device__ __forceinline__ X wave_add(X x) { return __builtin_bit_cast(X, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wave_scan(x)), 63)); }

// The sequence of packed row r and its view, for the whole wave; false: none. A call of up to 64 sequences takes one round of loads, a sequence a lane, more take
// two to find it and one for its view. In bounds whatever the arrays hold.
template <typename A>
__device__ __forceinline__ bool place_of(const A & a, int32_t r, int & seq, seq_view & v) {
    static_assert(CACHE_MAX_SEQ <= 64 * 64, "a sequence a lane, or 64");
    const int lane = (int) threadIdx.x & 63;
    if (a.n_seq <= 64) {
        const int i = min(lane, a.n_seq - 1);
        const seq_view mine = view_of(a, i);
        const uint64_t has = __ballot(lane < a.n_seq && r >= mine.row0 && r < mine.row0 + mine.rows);
        if (!has) return false;
        seq = __builtin_ctzll(has);
        v = {__builtin_amdgcn_readlane(mine.row0, seq), __builtin_amdgcn_readlane(mine.rows, seq), __builtin_amdgcn_readlane(mine.len, seq)};
        return true;
    }
    const int step = (a.n_seq + 63) >> 6;
    const int32_t * ends = a.row_start + 1;
    int at = (int) __popcll(__ballot(ends[min((lane + 1) * step, a.n_seq) - 1] <= r)) * step;
    if (at >= a.n_seq) return false;
    const int i = at + lane;
    at += (int) __popcll(__ballot(lane < step && i < a.n_seq && ends[min(i, a.n_seq - 1)] <= r));
    if (at >= a.n_seq) return false;
    seq = uniform(at);
    v = view_of(a, seq);
    return r >= v.row0 && r < v.row0 + v.rows;
}

template <typename T>
__device__ __forceinline__ void store4(T * p, float4_t x) {
    typedef T vec __attribute__((ext_vector_type(4)));
    *(vec *) p = __builtin_convertvector(x, vec);
}

// `work`: a counter for each column tile of several pieces and K/V head (at the place of its first part), then the parts, [part][kv head]:
// sums [C][hd], (maximum, sum) [C][2]. The parts bypass the L2s of the XCDs (cache policy sc1, what agent-scope atomics use): once a
// wave's stores have completed they are visible to every XCD, and no L2 is written back or invalidated.
constexpr int64_t COUNTERS = 8192;
template <int HD, int C>
struct parts_view {
    static constexpr int SC1 = 16, PART = C * (HD + 2) * 4;      // bytes
    const brsrc r;
    const uint32_t at, step;      // this tile's first part, from one to the next
    __device__ parts_view(float * work, int64_t parts, int n_kv_head, int64_t part, int kvh)
        : r(make_brsrc(work + 2 * COUNTERS, parts * n_kv_head * PART)), at((uint32_t) (part * n_kv_head + kvh) * PART), step((uint32_t) n_kv_head * PART) {}
    __device__ void put(int piece, int col, int n, float4_t x) const {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(word4_t, x), r, at + piece * step + (uint32_t) (col * HD + n) * 4, 0, SC1);
    }
    __device__ void put_stat(int piece, int col, float mu, float l) const {
        __builtin_amdgcn_raw_buffer_store_b64(word2_t{__float_as_uint(mu), __float_as_uint(l)}, r, at + piece * step + (uint32_t) (C * HD * 4 + col * 8), 0, SC1);
    }
    __device__ float4_t get(int piece, int col, int n) const {
        return __builtin_bit_cast(float4_t, __builtin_amdgcn_raw_buffer_load_b128(r, at + piece * step + (uint32_t) (col * HD + n) * 4, 0, SC1));
    }
    __device__ void get_stat(int piece, int col, float & mu, float & l) const {
        const word2_t x = __builtin_amdgcn_raw_buffer_load_b64(r, at + piece * step + (uint32_t) (C * HD * 4 + col * 8), 0, SC1);
        mu = __uint_as_float(x[0]);
        l = __uint_as_float(x[1]);
    }
};

// Whether this workgroup's piece, whose part it has stored, is the last of its tile's. The counter is 0 between calls; what is no
// counter (a work space not used before holds anything) is told by its upper 40 bits, and made one by whoever comes first. Every
// wait ends: each workgroup adds to a word that is no counter once, so one of the exchanges succeeds.
__device__ __forceinline__ bool last_to_arrive(float * work, int64_t at, int pieces) {
    typedef unsigned long long u64;
    constexpr u64 TAG = 0x6a65706163ull;
    __shared__ int last;
    __builtin_amdgcn_s_waitcnt(0x0f70);      // vmcnt(0): this wave's part has been written
    __syncthreads();
    if (threadIdx.x == 0) {
        u64 * counter = (u64 *) work + at, was;
        while ((was = atomicAdd(counter, 1ull)) >> 24 != TAG) {
            u64 now;
            while ((now = __hip_atomic_load(counter, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) >> 24 != TAG) atomicCAS(counter, now, TAG << 24);
        }
        last = (int) (was & 0xffffff) + 1 == pieces;
        if (last) __hip_atomic_store(counter, TAG << 24, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return last;
}

// The pieces of a tile's columns added in their order, HD / 4 threads a column, 8 pieces in flight; out_at: where a column goes
template <typename T, int HD, int C, typename OUT>
__device__ __forceinline__ void join_pieces(const parts_view<HD, C> & part, int pieces, int n_cols, OUT out_at) {
    constexpr int W = HD / 4, PG = NT / W, AT_ONCE = 8;
    const int tid = (int) threadIdx.x, n = tid % W * 4;
    for (int at = tid / W; at < C && at < n_cols && tid < PG * W; at += PG) {
        float top = -INFINITY, all = 0.0f;
        float4_t x = {0, 0, 0, 0};
        for (int k0 = 0; k0 < pieces; k0 += AT_ONCE) {
            float mu[AT_ONCE], l[AT_ONCE], to = top;
            float4_t y[AT_ONCE];
#pragma unroll
            for (int k = 0; k < AT_ONCE; k++) {
                const int piece = min(k0 + k, pieces - 1);
                part.get_stat(piece, at, mu[k], l[k]);
                y[k] = part.get(piece, at, n);
            }
#pragma unroll
            for (int k = 0; k < AT_ONCE; k++) to = fmaxf(to, mu[k]);
            const float m = to == -INFINITY ? 0.0f : to, back = __builtin_amdgcn_exp2f(top - m);
            all *= back;
            x *= back;
#pragma unroll
            for (int k = 0; k < AT_ONCE; k++) {
                const float f = k0 + k < pieces ? __builtin_amdgcn_exp2f(mu[k] - m) : 0.0f;
                all += l[k] * f;
                x += y[k] * f;
            }
            top = to;
        }
        store4((T *) out_at(at) + n, x * (all == 0.0f ? 0.0f : 1.0f / all));
    }
}

// The column's query row to f16: scaled by a power of two to a largest value in [2^14, 2^15), one term or two; c: what a product of it with
// a key is multiplied by to be an exponent of 2 (never negative: the row carries the scale's sign)
template <typename T> struct vec8 {
    typedef T t __attribute__((ext_vector_type(8)));
    typedef t at16 __attribute__((aligned(16)));      // rows lie at whole 16 bytes, f32's 8 values too
};
template <typename T, int HD>
__device__ __forceinline__ void fetch_query(const T * p, int g, typename vec8<T>::t * y) {      // (of the head at p)
    p += g * 8;
#pragma unroll
    for (int b = 0; b < HD / 32; b++) y[b] = *(const typename vec8<T>::at16 *) (p + b * 32);
}
template <typename T, int HD, int TERMS>
__device__ __forceinline__ void turn_query(float scale, const typename vec8<T>::t * y, half8_t (*q)[TERMS], float & c) {
    constexpr int NB = HD / 32;
    float8_t x[NB];
    float top = 0.0f;
#pragma unroll
    for (int b = 0; b < NB; b++) {
        x[b] = __builtin_convertvector(y[b], float8_t);
        for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(x[b][j]));
    }
    const uint32_t of_top = __float_as_uint(col_max(top)) >> 23, ex = max(of_top, 15u);      // (a row below 2^-112 is scaled by 2^126)
    float f = of_top == 255 ? __builtin_nanf("") : __uint_as_float((268 - ex) << 23);      // an infinity in the row: all of it NaN
    c = fabsf(scale) * LOG2E * __uint_as_float((ex - 14) << 23);
    if (scale < 0.0f) f = -f;
#pragma unroll
    for (int b = 0; b < NB; b++) {
        x[b] *= f;
        q[b][0] = __builtin_convertvector(x[b], half8_t);
        if constexpr (TERMS == 2) q[b][1] = __builtin_convertvector(x[b] - __builtin_convertvector(q[b][0], float8_t), half8_t);
    }
}

// One column's scores of a tile to weights; its maximum and accumulators (of ND tiles of dimensions, and the weights' sum behind them)
// follow. MASKED: some of the scores may be -infinity, and weigh nothing
template <bool MASKED, int ND>
__device__ __forceinline__ void softmax_weights(float4_t * s, float c, float & mu, float4_t * o) {
    float top = s[0][0];
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) top = fmaxf(top, s[t][r]);
    const float want = col_max(top) * c;
    const bool move = want - mu > 15.0f;
    if (__any(move)) {
        const float to = move ? want - 10.0f : mu;
        const float f = move ? __builtin_amdgcn_exp2f(mu - to) : 1.0f;
        mu = to;
#pragma unroll
        for (int d = 0; d <= ND; d++) o[d] *= f;
    }
    const float m = mu == -INFINITY ? 0.0f : mu;
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float x = s[t][r];
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x, c, -m));
            s[t][r] = MASKED && x == -INFINITY ? 0.0f : p;
        }
}

// The same of keys key + 16 t + r, of which those from lim on and the strips t of `hidden` are not read
template <bool MASKED, int ND>
__device__ __forceinline__ void softmax_step(float4_t * s, int32_t key, int32_t lim, uint32_t hidden, float c, float & mu, float4_t * o) {
    if constexpr (MASKED) {
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (key + t * 16 + r >= lim || (hidden >> t & 1)) s[t][r] = -INFINITY;
    }
    softmax_weights<MASKED, ND>(s, c, mu, o);
}

// The B operand of the product with V, 32 keys of strips 2 h and 2 h + 1: weights as one f16 or two. Their sum goes to every element of l.
template <int TERMS>
__device__ __forceinline__ void turn_weights(const float4_t * s, int h, half8_t * p, float4_t & l) {
    const half8_t ones = {1, 1, 1, 1, 1, 1, 1, 1};
#pragma unroll
    for (int r = 0; r < 8; r++) {
        const float w = s[2 * h + (r >> 2)][r & 3];
        p[0][r] = (_Float16) w;
        if constexpr (TERMS == 2) p[1][r] = (_Float16) (w - (float) p[0][r]);
    }
#pragma unroll
    for (int k = 0; k < TERMS; k++) l = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, p[k], l, 0, 0, 0);
}

// O^T += V^T P^T of 16 dimensions and 32 keys, from V's codes and the scales of the same keys (4 at d, 4 at d + stride); EXACT: values as two f16, else
// rounded to one
template <int TERMS, bool EXACT = true>
__device__ __forceinline__ float4_t add_values(half8_t codes, const unsigned char * d, int stride, const half8_t * p, float4_t o) {
    const half8_t scales = __builtin_shufflevector(*(const half4_t *) d, *(const half4_t *) (d + stride), 0, 1, 2, 3, 4, 5, 6, 7);
    const half8_t v = codes * scales;
    o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[0], o, 0, 0, 0);
    if constexpr (EXACT) o = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_elementwise_fma(codes, scales, -v), p[0], o, 0, 0, 0);
    if constexpr (TERMS == 2) o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[1], o, 0, 0, 0);
    return o;
}

template <int HD> constexpr int wave_lds() { return HD / 16 * 528 + 8 * HD; }      // V codes of a tile, then its scales

}  // namespace
