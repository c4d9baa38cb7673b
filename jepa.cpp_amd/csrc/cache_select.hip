// cache_select.hip - the pages of the cache that each row reads, by a cheap score of each page's digest.
//
//   P_n = sum_h max(q_hn, 0), N_n = sum_h min(q_hn, 0) over the heads h that share a K/V head
//   score(page) = scale(page) * sum_n (P_n hi_n + N_n lo_n): the sum over those heads of the largest product that a key in the page's box could have
//
// The sums P and N are made in 64 bits, rounded to f32 and held as 8-bit codes with one factor for all 2 hd of them, which the order of the
// scores does not depend on. The dot product is of whole numbers, at most 2 * 128 * 127^2 < 2^24: it is exact in the matrix instruction
// (16x16x64 i8, 16 pages x 16 rows) and as an f32, so a score has one rounding and the selection does not depend on how the pages
// are dealt out. Ties go to the lower page.
//
// A workgroup has a K/V head and a tile of 16 consecutive packed rows, or one row where rows are few (then, if the table is long, a piece of
// its pages; the last piece to arrive joins the pieces' candidates). It goes through the pages in chunks: its waves score 16 pages each, then
// take rows: what passes a row's threshold is put behind its candidates, in the pages' order, and when they might not take the
// next chunk's the best are kept. The best n of some hundred keys are found bit by bit, the keys in registers, a ballot for each 64.
#include "cache_attn_dev.h"
#include "common.h"

#include <algorithm>

namespace {

typedef int int4_t __attribute__((ext_vector_type(4)));

constexpr int MOST = CACHE_MOST_SELECTED;
constexpr float LEAST = 0x1p-100f;
constexpr int ROWS = 16;                                                   // of a tile
constexpr int chunk_of(int rt) { return rt == 1 ? 1024 : 128; }             // pages scored before rows are taken
constexpr int MOST_PIECES = 64;
constexpr int SPLIT_UNITS = 2048;                                           // pieces of all rows and K/V heads of a call together

// f32 -> a number in the same order; 0 and 1 are none's
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u ^ ((uint32_t) ((int32_t) u >> 31) | 0x80000000u);
}
constexpr uint32_t KEY_LOWEST = 0x007fffffu;      // -infinity's

// The `keep` largest of n candidates (E 64 at most), ties to the first, left at the front in their order; by one wave. Returns how many are left,
// and a threshold that a later candidate has to pass.
template <int E>
__device__ __forceinline__ int keep_best(uint32_t * keys, uint32_t * pages, int n, int keep, uint32_t & pass) {
    const int lane = (int) threadIdx.x & 63;
    if (n <= keep) return n;
    uint32_t k[E], p[E];
    uint32_t most = 0, least = 0xffffffffu;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const bool has = e * 64 + lane < n;
        k[e] = has ? keys[e * 64 + lane] : 0u;
        p[e] = has ? pages[e * 64 + lane] : 0u;
        most = max(most, k[e]);
        if (has) least = min(least, k[e]);
    }
#define DPP(x, ctrl, rows) (uint32_t) __builtin_amdgcn_update_dpp((int) x, (int) x, ctrl, rows, 0xf, false)
#define JOIN(ctrl, rows) most = max(most, DPP(most, ctrl, rows)); least = min(least, DPP(least, ctrl, rows))
    JOIN(0x111, 0xf); JOIN(0x112, 0xf); JOIN(0x114, 0xf); JOIN(0x118, 0xf); JOIN(0x142, 0xa); JOIN(0x143, 0xc);
#undef JOIN
#undef DPP
    most = (uint32_t) __builtin_amdgcn_readlane((int) most, 63);
    least = (uint32_t) __builtin_amdgcn_readlane((int) least, 63);
    auto count = [&](uint32_t c) {
        int s = 0;
#pragma unroll
        for (int e = 0; e < E; e++) s += (int) __popcll(__ballot(k[e] >= c));
        return s;
    };
    // the largest t that `keep` or more pass, from the bits that all have on
    uint32_t t = least;
    if (most != least) {
        int bit = 31 - __builtin_clz(most ^ least);
        t = most & ~(((2u << bit) - 1));
        for (; bit >= 0; bit--) {
            const uint32_t c = t | 1u << bit;
            const int s = count(c);
            if (s >= keep) t = c;
            if (s == keep) break;
        }
    }
    int above = 0;      // more than t: all of them; t itself: the first ones
#pragma unroll
    for (int e = 0; e < E; e++) above += (int) __popcll(__ballot(k[e] > t));
    int ties = keep - above, at = 0;
    if (ties < 0) ties = 0;
    wave_order();
    const uint64_t before = (1ull << lane) - 1;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const uint64_t eq = __ballot(k[e] == t && e * 64 + lane < n);
        const bool mine = k[e] > t || ((eq >> lane & 1) && (int) __popcll(eq & before) < ties);
        const uint64_t in = __ballot(mine);
        if (mine) {
            const int i = at + (int) __popcll(in & before);
            keys[i] = k[e];
            pages[i] = p[e];
        }
        at += (int) __popcll(in);
        ties -= min(ties, (int) __popcll(eq));
    }
    wave_order();
    pass = t;
    return at;
}

// `work`: a counter for each (row, K/V head) of several pieces, SPLIT_UNITS of them, then [row][K/V head][piece] candidates: their number, keys [take], pages [take]
struct pieces_view {
    static constexpr int SC1 = 16;
    const brsrc r;
    const uint32_t bytes;
    __device__ pieces_view(const cache_select_args & a, int64_t unit)
        : r(make_brsrc((unsigned char *) a.work + SPLIT_UNITS * 8 + unit * a.pieces * (8 * a.take + 16), (int64_t) a.pieces * (8 * a.take + 16))), bytes(8 * a.take + 16) {}
    __device__ void put(int piece, int word, uint32_t x) const { __builtin_amdgcn_raw_buffer_store_b32(x, r, piece * bytes + word * 4, 0, SC1); }
    __device__ uint32_t get(int piece, int word) const { return __builtin_amdgcn_raw_buffer_load_b32(r, piece * bytes + word * 4, 0, SC1); }
};

template <typename T, int HD, int RT>
__global__ __launch_bounds__(NT) void k_cache_select(cache_select_args a) {
    constexpr int CH = chunk_of(RT), QS = 2 * HD + 16, SS = CH + 4, E = (CH + MOST) / 64, DIMS = HD / 16;
    __shared__ __attribute__((aligned(16))) unsigned char codes[ROWS * QS];
    __shared__ __attribute__((aligned(16))) int32_t dots[RT * SS];
    __shared__ float scales[CH];
    extern __shared__ __attribute__((aligned(16))) uint32_t lists[];      // keys [RT][cap], pages [RT][cap]
    const int tid = (int) threadIdx.x, lane = tid & 63, l15 = lane & 15, g = lane >> 4, wv = uniform(tid >> 6);
    const int group = a.n_head / a.n_kv_head, kvh = (int) (blockIdx.x % (unsigned) a.n_kv_head);
    const unsigned at_block = blockIdx.x / (unsigned) a.n_kv_head;
    const int piece = RT == 1 ? (int) (at_block % (unsigned) a.pieces) : 0;
    const int64_t t0 = (int64_t) (RT == 1 ? at_block / (unsigned) a.pieces : at_block) * RT, t1 = min(t0 + RT, a.n_rows);
    const int page_shift = __builtin_ctz((unsigned) a.page_size), cap = CH + a.take;
    uint32_t * const keys = lists, * const pages = lists + RT * cap;

    for (int64_t r0 = t0; r0 < t1;) {      // the sequences of the tile's rows
        const int seq = seq_of_row(a.row_start, a.n_seq, (int32_t) r0);
        if (seq < 0) {
            if (r0 >= a.row_start[0]) break;
            r0 = min((int64_t) a.row_start[0], t1);
            continue;
        }
        const seq_view v = view_of(a, seq);
        const int64_t r1 = min(t1, (int64_t) v.row0 + v.rows);
        if (r1 <= r0) { r0++; continue; }
        const int rows = (int) (r1 - r0);
        auto see_of = [&](int row) {      // pages that a row of these sees
            return (cache_visible(v.len - v.rows + (int32_t) (r0 - v.row0) + row, v.len, a.block) + a.page_size - 1) >> page_shift;
        };
        const int see_all = see_of(rows - 1);      // (the last row sees the most)
        // pages that are scored: neither a first nor a last one of the last row
        const int p0 = RT == 1 ? a.first + piece * a.piece : a.first, p1 = RT == 1 ? min(see_all - a.last, p0 + a.piece) : see_all - a.last;
        const bool choose = see_all > a.take && a.take > a.first + a.last;
        if (RT == 1 && !choose && piece != 0) return;
        int n[RT == 1 ? 1 : ROWS / 4] = {};            // candidates of this wave's rows, and what a key has to pass
        uint32_t pass[RT == 1 ? 1 : ROWS / 4] = {};
        if (choose && p0 < p1) {
            // queries: 16 threads a row
            __syncthreads();
            {
                const int row = min(tid >> 4, rows - 1), d0 = (tid & 15) * DIMS;
                constexpr int WORDS = DIMS * sizeof(T) / 4;
                struct values { T x[DIMS]; };
                struct words { uint32_t w[WORDS]; };
                const T * q = (const T *) a.q + (r0 + row) * a.ldq + (int64_t) kvh * group * HD + d0;
                double pos[DIMS] = {}, neg[DIMS] = {};
                bool odd = false;
                for (int h = 0; h < group; h++) {
                    words w;
#pragma unroll
                    for (int i = 0; i < WORDS; i++) w.w[i] = ((const uint32_t *) (q + (int64_t) h * HD))[i];
                    const values y = __builtin_bit_cast(values, w);
#pragma unroll
                    for (int d = 0; d < DIMS; d++) {
                        const float x = (float) y.x[d];
                        odd |= !(fabsf(x) < INFINITY);
                        pos[d] += (double) fmaxf(x, 0.0f);
                        neg[d] += (double) fminf(x, 0.0f);
                    }
                }
                float top = 0.0f;
#pragma unroll
                for (int d = 0; d < DIMS; d++) top = fmaxf(top, fmaxf((float) pos[d], -(float) neg[d]));
                if (odd) top = INFINITY;
                top = row_max16(top);
                const float inv = top >= LEAST && top < INFINITY ? 127.0f / top : 0.0f;
                unsigned char * const c = codes + (tid >> 4) * QS + d0;
#pragma unroll
                for (int d = 0; d < DIMS; d++) {
                    c[d] = (unsigned char) (signed char) (inv == 0.0f ? 0 : (int) rintf((float) pos[d] * inv));
                    c[HD + d] = (unsigned char) (signed char) (inv == 0.0f ? 0 : (int) rintf((float) neg[d] * inv));
                }
            }
            __syncthreads();
            int4_t b[2 * HD / 64];
#pragma unroll
            for (int k = 0; k < 2 * HD / 64; k++) b[k] = *(const int4_t *) (codes + l15 * QS + k * 64 + g * 16);
            const int32_t * table = a.table + (int64_t) seq * a.width;
            for (int c0 = p0; c0 < p1; c0 += CH) {
                const int c1 = min(c0 + CH, p1);
                for (int s0 = c0 + wv * 16; s0 < c1; s0 += 64) {
                    int64_t page = table[min(s0 + l15, c1 - 1)];
                    const bool bad = page < 0 || page >= a.n_pages;
                    if (bad) page = 0;
                    const unsigned char * d = a.digest + (page * a.n_kv_head + kvh) * cache_digest_bytes(HD);
                    int4_t x = {0, 0, 0, 0};
                    int4_t y[2 * HD / 64];
#pragma unroll
                    for (int k = 0; k < 2 * HD / 64; k++) y[k] = *(const int4_t *) (d + k * 64 + g * 16);
                    if (g == 0) scales[s0 - c0 + l15] = bad ? -1.0f : *(const float *) (d + 2 * HD);
#pragma unroll
                    for (int k = 0; k < 2 * HD / 64; k++) x = __builtin_amdgcn_mfma_i32_16x16x64_i8(y[k], b[k], x, 0, 0, 0);
                    if (l15 < RT) *(int4_t *) (dots + l15 * SS + (s0 - c0) + g * 4) = x;
                }
                __syncthreads();
                // rows
#pragma unroll
                for (int i = 0; i < (RT == 1 ? 1 : ROWS / 4); i++) {
                    const int row = RT == 1 ? 0 : i * 4 + wv;
                    if (row >= rows || (RT == 1 && wv != 0)) continue;
                    const int see = see_of(row);
                    if (see <= a.take) continue;
                    const int end = min(c1, see - a.last), keep = a.take - a.first - a.last;
                    for (int s = c0; s < end; s += 64) {
                        const int p = s + lane;
                        const float scale = scales[p - c0];
                        uint32_t key = scale < 0.0f ? KEY_LOWEST : key_of((float) dots[row * SS + p - c0] * scale);
                        const bool in = p < end && key > pass[i];
                        const uint64_t all = __ballot(in);
                        if (in) {
                            const int to = n[i] + (int) __popcll(all & ((1ull << lane) - 1));
                            keys[row * cap + to] = key;
                            pages[row * cap + to] = (uint32_t) p;
                        }
                        n[i] += (int) __popcll(all);
                    }
                    wave_order();
                    if (n[i] > keep) n[i] = keep_best<E>(keys + row * cap, pages + row * cap, n[i], keep, pass[i]);
                }
                if (c0 + CH < p1) __syncthreads();
            }
        }
        // what was found, between the first and the last pages
        auto write = [&](int row, const uint32_t * found, int n) {
            int32_t * out = a.selected + ((r0 + row) * a.n_kv_head + kvh) * a.take;
            const int see = see_of(row);
            const bool all = see <= a.take;
            for (int i = lane; i < a.take; i += 64) {
                int32_t p;
                if (all) p = i < see ? i : -1;
                else p = i < a.first ? i : i < a.first + n ? (int32_t) found[i - a.first] : i < a.first + n + a.last ? see - a.last + (i - a.first - n) : -1;
                out[i] = p;
            }
        };
        if constexpr (RT == 1) {
            if (a.pieces > 1 && choose) {
                const int64_t unit = r0 * a.n_kv_head + kvh;
                const pieces_view w(a, unit);
                if (wv == 0) {
                    if (lane == 0) w.put(piece, 0, (uint32_t) n[0]);
                    for (int i = lane; i < n[0]; i += 64) {
                        w.put(piece, 4 + i, keys[i]);
                        w.put(piece, 4 + a.take + i, pages[i]);
                    }
                }
                if (!last_to_arrive(a.work, unit, a.pieces)) return;
                if (wv != 0) return;
                int m = 0;
                uint32_t over = 0;
                const int keep = a.take - a.first - a.last;
                for (int k = 0; k < a.pieces; k++) {
                    const int has = min((int) w.get(k, 0), a.take);
                    for (int i = lane; i < has; i += 64) {
                        keys[m + i] = w.get(k, 4 + i);
                        pages[m + i] = w.get(k, 4 + a.take + i);
                    }
                    m += uniform(has);
                    wave_order();
                    if (m + a.take > cap || k + 1 == a.pieces) m = keep_best<E>(keys, pages, m, keep, over);
                }
                n[0] = m;
            }
            if (wv == 0) write(0, pages, n[0]);
            return;
        } else {
#pragma unroll
            for (int i = 0; i < ROWS / 4; i++)
                if (i * 4 + wv < rows) write(i * 4 + wv, pages + (i * 4 + wv) * cap, n[i]);
            __syncthreads();
            r0 = r1;
        }
    }
}

// Tiles of 16 rows where they fill the chip and sequences have rows for them; else a row a workgroup, and pieces of its pages where a table is long
int rows_of(const cache_shape & c, int64_t n_seq, int64_t n_rows) { return n_rows >= 4 * n_seq && n_rows * c.n_kv_head >= 256 * ROWS ? ROWS : 1; }
int pieces_of(const cache_shape & c, int64_t n_seq, int64_t n_rows, int64_t width) {
    if (rows_of(c, n_seq, n_rows) != 1) return 1;
    return (int) std::clamp<int64_t>(std::min((width + chunk_of(1) - 1) / chunk_of(1), SPLIT_UNITS / (n_rows * c.n_kv_head)), 1, MOST_PIECES);
}

template <typename T, int HD>
hipError_t select(const cache_shape & c, const cache_select_args & a, hipStream_t s) {
    cache_select_args args = a;
    void * p[] = {&args};
    const int rt = rows_of(c, a.n_seq, a.n_rows);
    args.pieces = pieces_of(c, a.n_seq, a.n_rows, a.width);
    args.piece = (a.width + args.pieces - 1) / args.pieces;
    const unsigned lds = (unsigned) (2 * rt * (chunk_of(rt) + a.take) * 4);
    return hipLaunchKernel(rt == 1 ? (const void *) k_cache_select<T, HD, 1> : (const void *) k_cache_select<T, HD, ROWS>,
                           dim3((unsigned) cache_select_blocks(c, a.n_seq, a.n_rows, a.width)), dim3(NT), p, lds, s);
}

template <typename T>
hipError_t by_head(const cache_shape & c, const cache_select_args & a, hipStream_t s) {
    return c.hd == 32 ? select<T, 32>(c, a, s) : c.hd == 64 ? select<T, 64>(c, a, s) : c.hd == 96 ? select<T, 96>(c, a, s) : select<T, 128>(c, a, s);
}

}  // namespace

int64_t cache_select_blocks(const cache_shape & c, int64_t n_seq, int64_t n_rows, int64_t width) {
    const int rt = rows_of(c, n_seq, n_rows);
    return (n_rows + rt - 1) / rt * pieces_of(c, n_seq, n_rows, width) * c.n_kv_head;
}

// What any call of no more rows, pages and pages taken needs
int64_t cache_select_work_bytes(const cache_shape & c, int64_t n_rows, int64_t width, int take) {
    const int64_t most = (width + chunk_of(1) - 1) / chunk_of(1);
    return most > 1 ? SPLIT_UNITS * 8 + std::min<int64_t>(n_rows * c.n_kv_head * most, SPLIT_UNITS) * (8 * (int64_t) take + 16) : 0;
}

hipError_t launch_cache_select(const cache_shape & c, int type, const cache_select_args & a, hipStream_t s) {
    return type == T_F32 ? by_head<float>(c, a, s) : type == T_F16 ? by_head<_Float16>(c, a, s) : by_head<__bf16>(c, a, s);
}
