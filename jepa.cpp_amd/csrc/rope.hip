// rope.hip - rows of heads rotated by positions of several axes (rope_dev.h), their gradient, and rows appended to the 4-bit
// cache with the rotation applied on the way.
//
// Both are bound by memory once there are rows enough: a value is read and written once, and the 64-bit operations of a cosine and sine (some 35) are
// shared by the heads that one thread goes through, four of them in flight. Measured: the gradient of 8192 bf16 rows of 16 heads of 88 11.4 us
// (46 MB, 4.1 TB/s; a large copy reaches 5.05), 4128 f32 frame rows of 16 + 16 + 16 heads of 64 appended 18.4 us (73 MB, 4.0 TB/s, the VALU busy 35 % of it), 32768 bf16 rows of
// 32 + 8 + 8 heads of 128 151 us (709 MB, 4.7 TB/s), 64 f16 rows of 40 heads of 128 5.0 us (a launch and a chain of three loads and the cosines),
// 64 rows of 32 + 8 + 8 heads of 128, one token of 64 requests, appended 4.4 us, one row of 16 + 16 + 16 heads of 64 4.2 (calls of a captured graph; the same chain).
#include "common.h"
#include "rope_dev.h"

#include <algorithm>

namespace {

constexpr int AHEAD = 4;      // heads of a row in flight

// Rows of heads: a thread has one unit (8 neighbours, or 8 elements and their 8 partners) of a row and goes through some of its heads.
template <typename T, bool HALVES>
__device__ __forceinline__ void rope_part(const rope_args & a, const rope_map & m, int64_t row_block, int head_block) {
    typedef typename vec8<T>::t V;
    typedef typename at16<T>::t V16;
    const int tid = (int) threadIdx.x, in = tid / a.units, u = tid % a.units;
    const int64_t row = row_block * a.rows_per + in;
    if (in >= a.rows_per || row >= a.n_rows) return;
    const int h0 = head_block * a.heads_per, h1 = min(h0 + a.heads_per, a.n_head);
    const int e0 = HALVES ? 8 * m.lead[u] : 8 * u, to = HALVES ? m.delta[m.lead[u]] : 0;
    const T * x = (const T *) a.x + row * a.ldx + e0;
    T * out = (T *) a.out + row * a.ldo + e0;
    V p[AHEAD], q[AHEAD];
    auto load = [&](int h) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            if (h + i < h1) {
                p[i] = *(const V16 *) (x + (int64_t) (h + i) * a.hd);
                if constexpr (HALVES) q[i] = *(const V16 *) (x + (int64_t) (h + i) * a.hd + to);      // (itself, where it does not turn)
            }
    };
    load(h0);
    const row_pos r = pos_of(a.pos, row, m.n_axes);
    float8 c, s;
    turns8(m, r, e0, c, s);
    const int left = m.rot - e0;
    if (HALVES && a.back) s = -s;
    for (int h = h0; h < h1; h += AHEAD) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            if (h + i >= h1) break;
            const float8 f = __builtin_convertvector(p[i], float8);
            T * at = out + (int64_t) (h + i) * a.hd;
            if constexpr (HALVES) {
                const float8 g = __builtin_convertvector(q[i], float8);
                if (to) {
                    store8(at, f * c - g * s);
                    store8(at + to, g * c + f * s);
                } else {
                    store8(at, f);
                }
            } else {
                store8(at, turn_neighbours(f, c, s, left, a.back));
            }
        }
        if (h + AHEAD < h1) load(h + AHEAD);
    }
}

template <typename T, bool HALVES>
__global__ __launch_bounds__(256) void k_rope_rows(rope_args a, rope_map m) {
    rope_part<T, HALVES>(a, m, blockIdx.x / (unsigned) a.head_blocks, (int) (blockIdx.x % (unsigned) a.head_blocks));
}

// Keys rotated and stored with their values, queries rotated: workgroups of the first kind have whole strips of some heads, as k_cache_store has.
template <typename T, int HD, bool HALVES>
__global__ __launch_bounds__(256) void k_cache_append(append_args a, rope_args qa, rope_map m) {
    if (blockIdx.x >= a.kv_blocks) {
        const unsigned b = blockIdx.x - a.kv_blocks;
        rope_part<T, HALVES>(qa, m, b / (unsigned) qa.head_blocks, (int) (b % (unsigned) qa.head_blocks));
        return;
    }
    constexpr int GS = group<HD>::size, GW = group<HD>::work, ROWS = group<HD>::rows;
    const int tid = (int) threadIdx.x, lane = tid & 63, t = tid % GS;
    const int64_t row = (int64_t) (blockIdx.x / (unsigned) a.head_blocks) * ROWS + tid / GS;
    const int h0 = (int) (blockIdx.x % (unsigned) a.head_blocks) * a.heads_per, h1 = min(h0 + a.heads_per, a.n_kv_head);
    const bool has = row < a.n_rows && t < GW;
    const int64_t slot = has ? a.slots[row] : -1;
    const int e0 = has ? 8 * t : 0, to = HALVES ? m.delta[e0 / 8] : 0;
    const T * k = (const T *) a.k + (has ? row : 0) * a.ldk + e0, * v = (const T *) a.v + (has ? row : 0) * a.ldv + e0;
    float8 xk = load8(k + (int64_t) h0 * HD), xp = HALVES ? load8(k + (int64_t) h0 * HD + to) : float8{}, xv = load8(v + (int64_t) h0 * HD);
    const row_pos r = pos_of(a.pos, has ? row : 0, m.n_axes);
    float8 c, s;
    turns8(m, r, e0, c, s);
    if (HALVES && to > 0) s = -s;      // of the first half
    for (int h = h0; h < h1; h++) {
        const int hn = min(h + 1, h1 - 1);
        const float8 nk = load8(k + (int64_t) hn * HD), np = HALVES ? load8(k + (int64_t) hn * HD + to) : float8{}, nv = load8(v + (int64_t) hn * HD);
        const float8 y = HALVES ? (to ? xk * c + xp * s : xk) : turn_neighbours(xk, c, s, m.rot - e0, false);
        store_head<HD>(a.cache, y, xv, slot, lane, t, h, a.n_kv_head, a.page_shift, a.n_slots);
        xk = nk; xp = np; xv = nv;
    }
}

// A thread makes its cosines and sines once for some heads, up to 8, as long as that leaves the chip threads enough. Measured, us: 8192 bf16 rows of 16 heads of 88
// with 2^16 threads 11.4, 2^17 12.3, 2^18 12.9, 2^19 17.3; 4128 f32 frame rows of 16 + 16 + 16 heads of 64 appended with 2^17 threads for keys 18.4 to 18.6 (2^16 19.2,
// 2^18 23.8, 2^19 34); 32768 bf16 rows of 32 + 8 + 8 heads of 128 with up to 16 heads a thread 164, 8 151, 4 164, 2 214.
constexpr int64_t THREADS = 1 << 16, KEY_THREADS = 1 << 17;
constexpr int MOST_HEADS = 8;
void share(rope_args & a, const rope_map & m, bool halves) {
    a.units = halves ? m.rot / 16 + (m.hd - m.rot) / 8 : m.hd / 8;
    a.rows_per = 256 / a.units;
    a.heads_per = (int) std::clamp<int64_t>(a.n_rows * a.units * a.n_head / THREADS, 1, std::min(MOST_HEADS, a.n_head));
    a.head_blocks = (a.n_head + a.heads_per - 1) / a.heads_per;
}
int64_t blocks_of(const rope_args & a) { return (a.n_rows + a.rows_per - 1) / a.rows_per * a.head_blocks; }
bool halves_of(const rope_map & m) { return m.form >= 2; }

template <typename T>
hipError_t rope(rope_args a, rope_map m, hipStream_t s) {
    share(a, m, halves_of(m));
    void * p[] = {&a, &m};
    return hipLaunchKernel(halves_of(m) ? (const void *) k_rope_rows<T, true> : (const void *) k_rope_rows<T, false>, dim3((unsigned) blocks_of(a)), dim3(256), p, 0, s);
}

template <typename T, int HD>
hipError_t append(append_args a, rope_args q, rope_map m, hipStream_t s) {
    const int64_t rows = group<HD>::rows, row_blocks = (a.n_rows + rows - 1) / rows;
    a.heads_per = (int) std::clamp<int64_t>(row_blocks * a.n_kv_head * 256 / KEY_THREADS, 1, std::min(MOST_HEADS, a.n_kv_head));
    a.head_blocks = (a.n_kv_head + a.heads_per - 1) / a.heads_per;
    a.kv_blocks = (unsigned) (row_blocks * a.head_blocks);
    int64_t q_blocks = 0;
    if (q.x) {
        share(q, m, halves_of(m));
        q_blocks = blocks_of(q);
    }
    void * p[] = {&a, &q, &m};
    return hipLaunchKernel(halves_of(m) ? (const void *) k_cache_append<T, HD, true> : (const void *) k_cache_append<T, HD, false>,
                           dim3((unsigned) (a.kv_blocks + q_blocks)), dim3(256), p, 0, s);
}

}  // namespace

hipError_t launch_rope_axes(const rope_args & a, const rope_map & m, int type, hipStream_t s) {
    return type == T_F32 ? rope<float>(a, m, s) : type == T_F16 ? rope<_Float16>(a, m, s) : rope<__bf16>(a, m, s);
}

hipError_t launch_cache_append(const append_args & a, const rope_args & q, const rope_map & m, int type, hipStream_t s) {
#define CALL(T, HD) append<T, HD>(a, q, m, s)
#define BY_HEAD(T) (m.hd == 32 ? CALL(T, 32) : m.hd == 64 ? CALL(T, 64) : m.hd == 96 ? CALL(T, 96) : CALL(T, 128))
    return type == T_F32 ? BY_HEAD(float) : type == T_F16 ? BY_HEAD(_Float16) : BY_HEAD(__bf16);
#undef BY_HEAD
#undef CALL
}
