// cache_attention.hip - attention of packed query rows over the 4-bit paged cache on gfx950.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp2(c (q . k_j) - mu),  k_j[n] = dk_jb (ck_jn - 8), v_j[n] = dv_jb (cv_jn - 8)
//
// Columns are the query rows times the heads of one K/V head ("group"): column = row * group + head. S^T = K Q^T puts one
// column in a lane (16x16x32 f16 MFMA, 16 keys x 16 columns), so the softmax is lane work and P^T feeds the second product,
// O^T += V^T P^T, from its registers.
//
// Numerics. 4-bit codes are exact in f16, so both products run on codes and every scale is applied in 32 bits:
//   - the MFMA's depth (32) is one q4_0 block: its sum times dk, in f32, added over the blocks of a head;
//   - q is scaled by a power of two to a largest value in [1, 2) (exact) and taken as one f16 (f16 and bf16 rows: below
//     2^-14 of the row's largest value they lose bits, 2^-25 of it at most) or as the sum of two (f32 rows: 22 bits);
//   - dv goes into the weights: P'_jb = p_j dv_jb in f32, rounded to one f16 (16-bit rows: 2^-12 relative, half a step of
//     f16, under the output's own rounding) or the sum of two (f32 rows). V itself then holds no NaN whatever a
//     masked token contains. mu is the running maximum of the scores plus the exponent of the tile's largest dv, less 6, and moves
//     when a tile passes it by more than 2^8: so P' is below 2^14, f16's range, however small or large the values are.
// Scores, maxima, sums and accumulators are f32.
//
// Layout. A wave owns 16 CT columns and sweeps its keys in tiles of 64 (4 strips), by itself: no barrier in the loop. K
// codes go from memory to the registers of the MFMA's A operand (the strip's layout is the operand's); V codes and scales go
// through the wave's own LDS, because V^T needs 16 keys of one dimension in a lane: ds_read_b64_tr_b4 turns 16 x 16
// nibbles around. The next tile's loads (and the page numbers of the one after) are in flight while a tile is computed.
// The four waves of a workgroup share one tile of columns and split its keys (KW 4, few columns: joined in LDS at the end), or
// have a tile of columns each (KW 1, prompts: the K/V they share comes from the CU's cache).
//
// Work. A unit is (sequence, tile of columns, piece of its keys, K/V head). The piece length is the same for all sequences
// of a call and chosen on the device from the sum of their lengths, so that long sequences are split and short ones are not and
// the chip is filled evenly by ragged batches; the host knows only a bound on the units, and workgroups past the last one
// leave. Pieces of a column tile write their sums to `work` and k_cache_join adds them in order.
#include "cache_dev.h"
#include "common.h"
#include "kernels.h"
#include "lds_dma.h"

#include <algorithm>
#include <type_traits>

namespace {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef float float8_t __attribute__((ext_vector_type(8)));
typedef int int2_t __attribute__((ext_vector_type(2)));

constexpr float LOG2E = 1.4426950408889634f;
constexpr int NT = 256;              // threads of a workgroup
constexpr int TILE = 64;             // keys of a wave's step
constexpr int PIECE = 4 * TILE;      // pieces are multiples of this: one step of each of four waves
constexpr int UNITS = 1024;          // units that a call is split into where its columns alone are fewer

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

// f over the four lanes l, l ^ 16, l ^ 32, l ^ 48 (the lanes of one column), the same bits in each
__device__ __forceinline__ float col_max(float x) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float col_sum(float x) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ uint32_t wave_umax(uint32_t x) {
    x = max(x, (uint32_t) __builtin_amdgcn_update_dpp(0, (int) x, 0xb1, 0xf, 0xf, false));       // quad_perm 1 0 3 2
    x = max(x, (uint32_t) __builtin_amdgcn_update_dpp(0, (int) x, 0x4e, 0xf, 0xf, false));       // quad_perm 2 3 0 1
    x = max(x, (uint32_t) __builtin_amdgcn_update_dpp(0, (int) x, 0x141, 0xf, 0xf, false));      // row_half_mirror
    x = max(x, (uint32_t) __builtin_amdgcn_update_dpp(0, (int) x, 0x140, 0xf, 0xf, false));      // row_mirror
    auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max((uint32_t) r[0], (uint32_t) r[1]);
    r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return (uint32_t) __builtin_amdgcn_readfirstlane((int) max((uint32_t) r[0], (uint32_t) r[1]));
}
// N words per lane of a buffer
template <int N>
__device__ __forceinline__ void load_words(uint32_t * x, brsrc r, int at, int off) {
    typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));
    typedef uint32_t uint3_t __attribute__((ext_vector_type(3)));
    typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));
    if constexpr (N == 1) x[0] = __builtin_amdgcn_raw_buffer_load_b32(r, at, off, 0);
    if constexpr (N == 2) { const uint2_t v = __builtin_amdgcn_raw_buffer_load_b64(r, at, off, 0); x[0] = v[0]; x[1] = v[1]; }
    if constexpr (N == 3) { const uint3_t v = __builtin_amdgcn_raw_buffer_load_b96(r, at, off, 0); x[0] = v[0]; x[1] = v[1]; x[2] = v[2]; }
    if constexpr (N == 4) { const uint4_t v = __builtin_amdgcn_raw_buffer_load_b128(r, at, off, 0); x[0] = v[0]; x[1] = v[1]; x[2] = v[2]; x[3] = v[3]; }
}
__device__ __forceinline__ void wave_order() {      // LDS accesses of the wave's lanes before and after stay in this order
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// one sequence of the call, within the call's buffers whatever the arrays hold
struct seq_view { int32_t row0, rows, len; };
__device__ __forceinline__ seq_view view_of(const cache_attn_args & a, int i) {
    seq_view v;
    const int32_t n = (int32_t) a.n_rows;
    v.row0 = min(max(a.row_start[i], 0), n);
    v.rows = max(min(max(a.row_start[i + 1], 0), n) - v.row0, 0);
    const int64_t cap = (int64_t) a.width * a.page_size;
    v.len = (int32_t) min<int64_t>(max(a.kv_len[i], 0), cap);
    return v;
}

struct unit { int seq, tile, piece, pieces; int32_t length; int64_t part; };      // part: the first piece's place in `work`

__device__ __forceinline__ uint64_t wave_sum64(uint64_t x) {
    for (int o = 32; o; o >>= 1) x += __shfl_xor((unsigned long long) x, o, 64);
    return x;
}

// Unit x of the call (x-th column tile if TILES), for column tiles of C. Every thread gets it; false past the last.
template <int C, bool TILES>
__device__ __forceinline__ bool find_unit(const cache_attn_args & a, uint32_t x, unit & u) {
    __shared__ uint64_t sums[3][NT / 64];
    __shared__ unit found;
    const int tid = (int) threadIdx.x, lane = tid & 63, wv = tid >> 6, group = a.n_head / a.n_kv_head;
    const int per = (a.n_seq + NT - 1) / NT, i0 = min(tid * per, a.n_seq), i1 = min(i0 + per, a.n_seq);
    uint64_t keys = 0;
    for (int i = i0; i < i1; i++) {
        const seq_view v = view_of(a, i);
        keys += (uint64_t) (((int64_t) v.rows * group + C - 1) / C) * (uint32_t) v.len;
    }
    keys = wave_sum64(keys);
    if (tid == 0) found.seq = -1;
    if (lane == 0) sums[0][wv] = keys;
    __syncthreads();
    keys = (sums[0][0] + sums[0][1] + sums[0][2] + sums[0][3]) * (uint32_t) a.n_kv_head;
    const int32_t length = (int32_t) min<uint64_t>((keys / UNITS + PIECE) / PIECE * PIECE, 0x7fffff00u);
    uint64_t mine = 0, parts = 0;
    for (int i = i0; i < i1; i++) {
        const seq_view v = view_of(a, i);
        const uint64_t tiles = (uint64_t) (((int64_t) v.rows * group + C - 1) / C), pieces = max((v.len + (int64_t) length - 1) / length, (int64_t) 1);
        mine += TILES ? tiles : tiles * pieces;
        parts += pieces > 1 ? tiles * pieces : 0;
    }
    uint64_t before = mine, parts_before = parts;
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t y = __shfl_up((unsigned long long) before, o, 64), z = __shfl_up((unsigned long long) parts_before, o, 64);
        if (lane >= o) { before += y; parts_before += z; }
    }
    if (lane == 63) { sums[1][wv] = before; sums[2][wv] = parts_before; }
    __syncthreads();
    for (int w = 0; w < wv; w++) { before += sums[1][w]; parts_before += sums[2][w]; }
    before -= mine;
    parts_before -= parts;
    if (x >= before && x < before + mine) {
        uint64_t at = x - before;
        for (int i = i0; i < i1; i++) {
            const seq_view v = view_of(a, i);
            const uint64_t tiles = (uint64_t) (((int64_t) v.rows * group + C - 1) / C), pieces = max((v.len + (int64_t) length - 1) / length, (int64_t) 1);
            const uint64_t n = TILES ? tiles : tiles * pieces;
            if (at < n) {
                // a prompt's last rows read the most keys: they go first
                found.tile = (int) (tiles - 1 - (TILES ? at : at / pieces));
                found.piece = TILES ? 0 : (int) (at % pieces);
                found.pieces = (int) pieces;
                found.length = length;
                found.part = (int64_t) (parts_before + (uint64_t) found.tile * pieces);
                found.seq = i;
                break;
            }
            at -= n;
            parts_before += pieces > 1 ? n : 0;
            if (TILES && pieces > 1) parts_before += tiles * pieces - n;
        }
    }
    __syncthreads();
    u = found;
    return u.seq >= 0;
}

// the parts of `work`: sums [part][kv head][C][hd], then (maximum, sum) [part][kv head][C][2]
template <int HD, int C>
struct parts_view {
    float * o, * s;
    __device__ parts_view(const cache_attn_args & a, int64_t part, int kvh) {
        const int64_t p = (part * a.n_kv_head + kvh) * C;
        o = a.work + p * (HD + 2);
        s = o + (int64_t) C * HD;
    }
};

template <typename T>
__device__ __forceinline__ void store4(T * p, float4_t x) {
    typedef T vec __attribute__((ext_vector_type(4)));
    *(vec *) p = __builtin_convertvector(x, vec);
}

template <int HD> constexpr int wave_lds() { return HD / 16 * 528 + 8 * HD; }      // V codes of a tile, then its scales
template <int HD, int CT, int KW> constexpr int group_lds() {
    const int loop = 4 * wave_lds<HD>(), join = KW == 4 ? 4 * 16 * CT * (HD + 4) * 4 + 4 * 16 * CT * 8 : 0;
    return loop > join ? loop : join;
}

template <typename T, int HD, int CT, int KW>
__global__ __launch_bounds__(NT, CT == 1 ? 3 : 2) void k_cache_attention(cache_attn_args a) {
    constexpr int NB = HD / 32, ND = HD / 16, TERMS = sizeof(T) == 4 ? 2 : 1, WC = 16 * CT, C = KW == 4 ? WC : 4 * WC;
    __shared__ __attribute__((aligned(16))) unsigned char lds[group_lds<HD, CT, KW>()];
    unit u;
    const int kvh = (int) (blockIdx.x % (unsigned) a.n_kv_head);
    if (!find_unit<C, false>(a, blockIdx.x / (unsigned) a.n_kv_head, u)) return;
    if (u.pieces > 1 && u.part + u.piece >= a.parts) return;      // (row_start that overlaps itself: more pieces than rows can have)
    const int tid = (int) threadIdx.x, lane = tid & 63, l15 = lane & 15, g = lane >> 4, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int seq = __builtin_amdgcn_readfirstlane(u.seq), group = a.n_head / a.n_kv_head;
    const seq_view sv = view_of(a, seq);
    const int32_t n_cols = __builtin_amdgcn_readfirstlane((int32_t) min<int64_t>((int64_t) sv.rows * group, 0x7fffffff));
    const int32_t col0 = u.tile * C + (KW == 4 ? 0 : wv * WC);
    auto visible = [&](int32_t col) { return cache_visible((int64_t) sv.len - sv.rows + col / group, sv.len, a.block); };

    // the wave's columns: their queries, and the keys that the first and the last of them read
    int32_t lim[CT];
    float c[CT];
    half8_t q[CT][NB][TERMS];
    const bool has = col0 < n_cols;
    const int32_t lim_lo = has ? visible(col0) : 0, lim_hi = has ? visible(min(col0 + WC, n_cols) - 1) : 0;
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        const int32_t col = min(col0 + ct * 16 + l15, n_cols - 1);
        lim[ct] = visible(col);
        const T * p = (const T *) a.q + (sv.row0 + (int64_t) (col / group)) * a.ldq + ((int64_t) kvh * group + col % group) * HD + g * 8;
        float8_t x[NB];
        typedef T vec __attribute__((ext_vector_type(8)));
        float top = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            x[b] = __builtin_convertvector(*(const vec *) (p + b * 32), float8_t);
            for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(x[b][j]));
        }
        const uint32_t ex = __float_as_uint(col_max(top)) >> 23;
        float f = ex < 254 ? __uint_as_float((254 - ex) << 23) : 0x1p-127f;      // (an f32 below its normal range: 2^127 will do)
        c[ct] = fabsf(a.scale) * LOG2E * (ex ? __uint_as_float(ex << 23) : 0x1p-127f);
        if (ex == 0) f = 0x1p127f;
        if (ex == 255) f = __builtin_nanf("");      // an infinity in the row: all of it NaN
        if (a.scale < 0.0f) f = -f;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            x[b] *= f;
            q[ct][b][0] = __builtin_convertvector(x[b], half8_t);
            if constexpr (TERMS == 2) q[ct][b][1] = __builtin_convertvector(x[b] - __builtin_convertvector(q[ct][b][0], float8_t), half8_t);
        }
    }

    float4_t o[CT][ND];
    float mu[CT], l[CT];      // mu: -inf before the first key
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        mu[ct] = -INFINITY;
        l[ct] = 0.0f;
        for (int d = 0; d < ND; d++) o[ct][d] = float4_t{0, 0, 0, 0};
    }

    // this wave's tiles of the unit's keys
    constexpr int STEP = KW * TILE;
    const int32_t kend = (int32_t) min<int64_t>((int64_t) (u.piece + 1) * u.length, lim_hi);
    int32_t k0 = __builtin_amdgcn_readfirstlane((int32_t) min<int64_t>((int64_t) u.piece * u.length + (KW == 4 ? wv * TILE : 0), 0x7fffff00));
    const int last_strip = (kend - 1) / 16, strips_of_page = a.page_size / 16, page_shift = __builtin_ctz(strips_of_page);
    const int32_t * table = a.table + (int64_t) seq * a.width;
    auto load_pages = [&](int32_t key) { return table[min(key / 16 + (lane & 3), last_strip) >> page_shift]; };
    uint32_t kn[4][NB], vn[4][NB], sn[4], bad_n = 0;      // the tile's codes and scales, in flight
    int pages = 0;                                         // page numbers of the next one, in lanes 0 to 3
    // a strip as a buffer resource (no bytes past the end of this wave's keys: such loads give 0 without a memory access)
    auto strip_of = [&](int32_t key, int pages, int t, uint32_t & bad) {
        const int strip = min(key / 16 + t, last_strip);
        int64_t page = __builtin_amdgcn_readlane(pages, t);
        if (page < 0 || page >= a.n_pages) { page = 0; bad |= 1u << t; }
        return make_brsrc(a.cache + ((page * a.n_kv_head + kvh) * strips_of_page + (strip & (strips_of_page - 1))) * (18 * HD), key < kend ? 18 * HD : 0);
    };
    auto load_v = [&](int32_t key, int pages) {
        bad_n = 0;
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const brsrc s = strip_of(key, pages, t, bad_n);
            load_words<NB>(vn[t], s, lane * (4 * NB), 8 * HD);
            load_words<1>(&sn[t], s, 16 * HD + lane * 4, 0);      // (0 past the strip's scales, from lane HD / 2 on)
        }
    };
    auto load_k = [&](int32_t key, int pages) {
        uint32_t bad = 0;
#pragma unroll
        for (int t = 0; t < 4; t++) load_words<NB>(kn[t], strip_of(key, pages, t, bad), lane * (4 * NB), 0);
    };
    unsigned char * const mine = lds + wv * wave_lds<HD>();
    unsigned char * const scales = mine + ND * 528;
    // where this lane's V words go, [dimension tile][64 keys][8 bytes], and the row that it names for the transposed read
    const int e = (l15 & 3) * 2 + ((l15 & 7) >> 2);
    const int tr_at = (((l15 >> 3) * 2 + (e >> 2)) * 16 + g * 4 + (e & 3)) * 8;
    uint32_t k1024 = 0x64006400u;
    asm volatile("" : "+v"(k1024));
    // one tile: MASKED where it passes some column's last key, the end, or has a page that is none
    auto tile = [&](auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        const uint32_t bad = bad_n;
        uint32_t dmax = 0;
        wave_order();
#pragma unroll
        for (int t = 0; t < 4; t++) {
            uint32_t sc = sn[t];
            if constexpr (MASKED) {      // scales of tokens that nobody reads are 0: what lies there does not matter
                const int d = lane % (HD / 4);
                const int32_t key = k0 + t * 16 + d / (2 * NB) * 4 + (d & 1) * 2;
                if (key >= kend || (bad >> t & 1)) sc = 0;
                else if (key + 1 >= kend) sc &= 0xffffu;
            }
            if (lane < HD / 2) *(uint32_t *) (scales + t * 2 * HD + lane * 4) = sc;
            if (lane >= HD / 4) dmax = max(dmax, max(sc & 0x7fffu, sc >> 16 & 0x7fffu));
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const int w = (lane & 3) * NB + b;
                *(uint32_t *) (mine + (w >> 1) * 528 + (t * 16 + (lane >> 2)) * 8 + (w & 1) * 4) = vn[t][b];
            }
        }
        load_v(k0 + STEP, pages);
        const float dexp = (float) ((int) (wave_umax(dmax) >> 10) - 14);      // every |dv| of the tile is below 2^dexp
        wave_order();

        // scores
        float4_t s[CT][4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const half4_t * dk = (const half4_t *) (scales + t * 2 * HD + g * (8 * NB));
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const half8_t kc = codes8(kn[t][b], k1024);
                const half4_t d = dk[b];
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
                    float4_t x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, q[ct][b][0], float4_t{0, 0, 0, 0}, 0, 0, 0);
                    if constexpr (TERMS == 2) x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, q[ct][b][1], x, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < 4; r++) s[ct][t][r] = __builtin_fmaf((float) d[r], x[r], b == 0 ? 0.0f : s[ct][t][r]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        load_k(k0 + STEP, pages);
        pages = load_pages(k0 + 2 * STEP);
        // weights
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            if constexpr (MASKED) {
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (k0 + t * 16 + g * 4 + r >= lim[ct] || (bad >> t & 1)) s[ct][t][r] = -INFINITY;
            }
            float top = s[ct][0][0];
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) top = fmaxf(top, s[ct][t][r]);
            const float want = col_max(top) * c[ct] + dexp;
            const bool move = want - mu[ct] > 14.0f;
            if (__any(move)) {
                const float to = move ? want - 6.0f : mu[ct];
                const float f = move ? __builtin_amdgcn_exp2f(mu[ct] - to) : 1.0f;
                mu[ct] = to;
                l[ct] *= f;
#pragma unroll
                for (int d = 0; d < ND; d++) o[ct][d] *= f;
            }
            const float m = mu[ct] == -INFINITY ? 0.0f : mu[ct];
            float4_t sum = {0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < 4; t++) {
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float x = s[ct][t][r];
                    float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x, c[ct], -m));
                    if constexpr (MASKED) p = x == -INFINITY ? 0.0f : p;
                    s[ct][t][r] = p;
                }
                sum += s[ct][t];
            }
            l[ct] += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        }
        // O^T += V^T P'^T, block by block of the head (the fma with 0 is one v_fma_mix from and to f16)
#pragma unroll
        for (int b = 0; b < NB; b++) {
            half8_t p[CT][2][TERMS];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const half4_t d0 = *(const half4_t *) (scales + 2 * h * 2 * HD + HD + g * (8 * NB) + b * 8);
                const half4_t d1 = *(const half4_t *) (scales + (2 * h + 1) * 2 * HD + HD + g * (8 * NB) + b * 8);
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
#pragma unroll
                    for (int r = 0; r < 8; r++) {
                        const float w = s[ct][2 * h + (r >> 2)][r & 3], d = (float) (r < 4 ? d0[r & 3] : d1[r & 3]);
                        if constexpr (TERMS == 1) {
                            p[ct][h][0][r] = (_Float16) __builtin_fmaf(w, d, 0.0f);
                        } else {
                            const float x = __builtin_fmaf(w, d, 0.0f);
                            p[ct][h][0][r] = (_Float16) x;
                            p[ct][h][1][r] = (_Float16) (x - (float) p[ct][h][0][r]);
                        }
                    }
                }
            }
#pragma unroll
            for (int dd = 0; dd < 2; dd++) {
                const int d = 2 * b + dd;
                const int2_t w = __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) int2_t *) (mine + d * 528 + tr_at));
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const half8_t vc = codes8((uint32_t) w[h], k1024);
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) {
                        o[ct][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vc, p[ct][h][0], o[ct][d], 0, 0, 0);
                        if constexpr (TERMS == 2) o[ct][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vc, p[ct][h][1], o[ct][d], 0, 0, 0);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    if (k0 < kend) {
        pages = load_pages(k0);
        load_v(k0, pages);
        load_k(k0, pages);
        pages = load_pages(k0 + STEP);
    }
    for (; k0 + TILE <= min(lim_lo, kend) && bad_n == 0; k0 += STEP) tile(std::false_type{});
    for (; k0 < kend; k0 += STEP) tile(std::true_type{});
#pragma unroll
    for (int ct = 0; ct < CT; ct++) l[ct] = col_sum(l[ct]);

    const parts_view<HD, C> part(a, u.part + u.piece, kvh);
    auto out_at = [&](int32_t col) { return (T *) a.out + (sv.row0 + (int64_t) (col / group)) * a.ldo + ((int64_t) kvh * group + col % group) * HD; };
    if constexpr (KW == 1) {
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            const int32_t at = wv * WC + ct * 16 + l15, col = u.tile * C + at;
            if (col >= n_cols) continue;
            if (u.pieces > 1) {
                if (g == 0) { part.s[2 * at] = mu[ct]; part.s[2 * at + 1] = l[ct]; }
                for (int d = 0; d < ND; d++) *(float4_t *) (part.o + (int64_t) at * HD + d * 16 + g * 4) = o[ct][d];
            } else {
                const float inv = l[ct] == 0.0f ? 0.0f : 1.0f / l[ct];
                T * p = out_at(col);
                for (int d = 0; d < ND; d++) store4(p + d * 16 + g * 4, o[ct][d] * inv);
            }
        }
    } else {
        // the four waves' sums at the largest of their maxima
        float * const stat = (float *) (lds + 4 * WC * (HD + 4) * 4), * const sum = (float *) lds;
        __syncthreads();      // the loop's LDS is read out
        if (g == 0)
            for (int ct = 0; ct < CT; ct++) { stat[(wv * WC + ct * 16 + l15) * 2] = mu[ct]; stat[(wv * WC + ct * 16 + l15) * 2 + 1] = l[ct]; }
#pragma unroll
        for (int ct = 0; ct < CT; ct++)
            for (int d = 0; d < ND; d++) *(float4_t *) (sum + (wv * WC + ct * 16 + l15) * (HD + 4) + d * 16 + g * 4) = o[ct][d];
        __syncthreads();
        for (int i = tid; i < WC * (HD / 4); i += NT) {
            const int at = i / (HD / 4), n = i % (HD / 4) * 4;
            const int32_t col = col0 + at;
            if (col >= n_cols) break;
            float top = -INFINITY, all = 0.0f;
            for (int w = 0; w < 4; w++) top = fmaxf(top, stat[(w * WC + at) * 2]);
            const float m = top == -INFINITY ? 0.0f : top;
            float4_t x = {0, 0, 0, 0};
            for (int w = 0; w < 4; w++) {
                const float f = __builtin_amdgcn_exp2f(stat[(w * WC + at) * 2] - m);
                all += stat[(w * WC + at) * 2 + 1] * f;
                x += *(const float4_t *) (sum + (w * WC + at) * (HD + 4) + n) * f;
            }
            if (u.pieces > 1) {
                if (n == 0) { part.s[2 * at] = top; part.s[2 * at + 1] = all; }
                *(float4_t *) (part.o + (int64_t) at * HD + n) = x;
            } else {
                store4(out_at(col) + n, x * (all == 0.0f ? 0.0f : 1.0f / all));
            }
        }
    }
}

// the pieces of a column tile added in their order
template <typename T, int HD, int C>
__global__ __launch_bounds__(NT) void k_cache_join(cache_attn_args a) {
    unit u;
    const int kvh = (int) (blockIdx.x % (unsigned) a.n_kv_head);
    if (!find_unit<C, true>(a, blockIdx.x / (unsigned) a.n_kv_head, u) || u.pieces < 2 || u.part + u.pieces > a.parts) return;
    const seq_view sv = view_of(a, u.seq);
    const int group = a.n_head / a.n_kv_head;
    const int64_t n_cols = (int64_t) sv.rows * group, col0 = (int64_t) u.tile * C;
    for (int i = (int) threadIdx.x; i < C * (HD / 4); i += NT) {
        const int at = i / (HD / 4), n = i % (HD / 4) * 4;
        const int64_t col = col0 + at;
        if (col >= n_cols) break;
        float top = -INFINITY, all = 0.0f;
        for (int k = 0; k < u.pieces; k++) top = fmaxf(top, parts_view<HD, C>(a, u.part + k, kvh).s[2 * at]);
        const float m = top == -INFINITY ? 0.0f : top;
        float4_t x = {0, 0, 0, 0};
        for (int k = 0; k < u.pieces; k++) {
            const parts_view<HD, C> p(a, u.part + k, kvh);
            const float f = __builtin_amdgcn_exp2f(p.s[2 * at] - m);
            all += p.s[2 * at + 1] * f;
            x += *(const float4_t *) (p.o + (int64_t) at * HD + n) * f;
        }
        T * out = (T *) a.out + (sv.row0 + col / group) * a.ldo + ((int64_t) kvh * group + col % group) * HD;
        store4(out + n, x * (all == 0.0f ? 0.0f : 1.0f / all));
    }
}

// Column tiles of 16, 32 or 128: by the columns that a sequence of the call has on average
int columns_of(const cache_shape & c, int64_t n_seq, int64_t n_rows) {
    const int64_t cols = n_rows * (c.n_head / c.n_kv_head);
    return cols <= 16 * n_seq ? 16 : cols <= 64 * n_seq ? 32 : 128;
}

// bounds on the column tiles of all sequences, and on the pieces that the ones split into several have
int64_t tiles_bound(const cache_shape & c, int64_t n_seq, int64_t n_rows) {
    return n_rows * (c.n_head / c.n_kv_head) / columns_of(c, n_seq, n_rows) + n_seq;
}
// Pieces are at least keys * kv heads / UNITS long, keys summed over column tiles: all of them without rounding up are UNITS / kv
// heads at most, and rounding up doubles that at most where there are two or more of a tile, as there must be to have parts.
int64_t parts_bound(const cache_shape & c, int64_t n_seq, int64_t n_rows, int64_t width) {
    const int64_t most = (width * c.page_size + PIECE - 1) / PIECE;
    if (most < 2) return 0;
    return std::min(tiles_bound(c, n_seq, n_rows) * most, 2 * (int64_t) ((UNITS + c.n_kv_head - 1) / c.n_kv_head));
}

template <typename T, int HD, int CT, int KW>
hipError_t attend(const cache_shape & c, const cache_attn_args & a, hipStream_t s) {
    constexpr int C = KW == 4 ? 16 * CT : 64 * CT;
    cache_attn_args args = a;
    void * p[] = {&args};
    const int64_t tiles = tiles_bound(c, a.n_seq, a.n_rows), parts = parts_bound(c, a.n_seq, a.n_rows, a.width);
    args.parts = parts;
    const int64_t blocks = (tiles + parts) * c.n_kv_head;
    if (blocks >= 1 << 24) return hipErrorInvalidConfiguration;      // threads of a launch are below 2^32
    const hipError_t e = hipLaunchKernel((const void *) k_cache_attention<T, HD, CT, KW>, dim3((unsigned) blocks), dim3(NT), p, 0, s);
    if (e != hipSuccess || !parts) return e;
    return hipLaunchKernel((const void *) k_cache_join<T, HD, C>, dim3((unsigned) (tiles * c.n_kv_head)), dim3(NT), p, 0, s);
}

template <typename T, int HD>
hipError_t by_columns(const cache_shape & c, const cache_attn_args & a, hipStream_t s) {
    const int cols = columns_of(c, a.n_seq, a.n_rows);
    return cols == 16 ? attend<T, HD, 1, 4>(c, a, s) : cols == 32 ? attend<T, HD, 2, 4>(c, a, s) : attend<T, HD, 2, 1>(c, a, s);
}

template <typename T>
hipError_t by_head(const cache_shape & c, const cache_attn_args & a, hipStream_t s) {
    return c.hd == 32 ? by_columns<T, 32>(c, a, s) : c.hd == 64 ? by_columns<T, 64>(c, a, s) : c.hd == 96 ? by_columns<T, 96>(c, a, s) : by_columns<T, 128>(c, a, s);
}

}  // namespace

int64_t cache_attention_work_bytes(const cache_shape & c, int64_t n_seq, int64_t n_rows, int64_t width) {
    return std::max<int64_t>(16, parts_bound(c, n_seq, n_rows, width) * c.n_kv_head * columns_of(c, n_seq, n_rows) * (c.hd + 2) * 4);
}

hipError_t launch_cache_attention(const cache_shape & c, int type, const cache_attn_args & a, hipStream_t s) {
    return type == T_F32 ? by_head<float>(c, a, s) : type == T_F16 ? by_head<_Float16>(c, a, s) : by_head<__bf16>(c, a, s);
}
