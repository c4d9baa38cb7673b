// cache_select.hip - the pages of the cache that each row reads, by a cheap score of each page's digest.
//
//   P_n = sum_h max(q_hn, 0), N_n = sum_h min(q_hn, 0) over the heads h that share a K/V head
//   score(page) = scale(page) * sum_n (P_n hi_n + N_n lo_n): the sum over those heads of the largest product that a key in the page's box could have
//
// The sums P and N are made in 64 bits, rounded to f32 and held as 8-bit codes with one factor for all 2 hd of them, which the order of the
// scores does not depend on (codes of zeros where a query is no number, a sum passes f32's end or all are below 2^-100). The dot product is of whole
// numbers, at most 2 * 128 * 127^2 < 2^24: it is exact in the matrix instruction (16x16x64 i8, 16 pages x 16 rows) and as an f32, so a score has one rounding and
// the selection does not depend on how the pages are dealt out. Ties go to the lower page.
//
//   few rows (k_select_row)    a workgroup has a row and K/V head, or a piece of its pages where the table is long (the last piece to arrive takes the
//                              best of all pieces' best). Its waves score 64 pages at a time, the loads of four matrix tiles in flight.
//   many rows (k_select_rows)  a workgroup has a K/V head and 16 consecutive rows, which share the digests that it reads; scores go from the matrix
//                              instruction's registers into the search, all rows in step.
// The best of some keys are found by histograms of 256 bins between the smallest and the largest: they narrow the range of the last one that is taken, 8
// bits at a time and mostly twice; counts and a scan of them put the taken ones behind each other in their order.
//
// Measured: a token of 64 requests of 200 to 8000 tokens in pages of 16, 32 heads over 8 of 128, 15.6 us (35 MB of digests, 2.2 TB/s; of a workgroup, medians: 0.9 us until
// its row's sequence is known, 4.7 for page numbers and queries' codes, 2 to 10 as the loads of others go before, 1.4 for the digests, 3.5 for scores and search); two contexts of 90000 to 131000 tokens in pages of 32, 14.2; 2000 rows over 250 pages of 64,
// 32 heads over 4, 19.4: 9.4 us of the VALU's time, 1450 instructions of each wave, in phases that wait for each other.
#include "cache_attn_dev.h"
#include "common.h"

#include <algorithm>
#include <type_traits>

namespace {

typedef int int4_t __attribute__((ext_vector_type(4)));

constexpr int MOST = CACHE_MOST_SELECTED;
constexpr float LEAST = 0x1p-100f;
constexpr int WAVES = 8;                      // of a workgroup
constexpr int ROWS = 16;                      // of k_select_rows' tile
constexpr int CHUNK = 256;                    // pages that it scores before rows take the best
constexpr int CAP = 2048;                     // keys that k_select_row takes the best of at once
constexpr int PIECE = 512;                    // pages of a piece, at least
constexpr int MOST_PIECES = 64;
constexpr int SPLIT_UNITS = 2048;             // pieces of all rows and K/V heads of a call together

// f32 -> a number in the same order; smaller ones than KEY_LOWEST, -infinity's, are no score's
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u ^ ((uint32_t) ((int32_t) u >> 31) | 0x80000000u);
}
constexpr uint32_t KEY_LOWEST = 0x007fffffu;

// x of this lane and the one 32 (16) further, added
template <int BY>
__device__ __forceinline__ double add_across(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    auto swap = [](uint32_t w) {
        if constexpr (BY == 32) return __builtin_amdgcn_permlane32_swap(w, w, false, false);
        else return __builtin_amdgcn_permlane16_swap(w, w, false, false);
    };
    const auto lo = swap((uint32_t) u), hi = swap((uint32_t) (u >> 32));
    return __builtin_bit_cast(double, (uint64_t) hi[0] << 32 | lo[0]) + __builtin_bit_cast(double, (uint64_t) hi[1] << 32 | lo[1]);
}

// The codes of P and N of a row's queries at q (group heads) to out [2 HD], by a wave: a lane has two dimensions, of all heads or of every second or fourth.
// Some heads are fetched ahead: loads come back in their order, and the digests' are to be on their way behind them.
template <typename T, int HD>
struct row_queries {
    static constexpr int LANES = HD / 2, EACH = HD == 96 ? 1 : 64 / LANES, WORDS = 2 * sizeof(T) / 4, AHEAD = 8 / EACH / WORDS;
    struct values { T x[2]; };
    struct words { uint32_t w[WORDS]; };
    words w[AHEAD];
    __device__ __forceinline__ static int first() { return EACH == 1 ? 0 : ((int) threadIdx.x & 63) / LANES; }
    __device__ __forceinline__ static int dim() { return min(((int) threadIdx.x & 63) % (EACH == 1 ? 64 : LANES), LANES - 1) * 2; }
    __device__ __forceinline__ static words load(const T * q, int h) {
        words x;
        const uint32_t * at = (const uint32_t *) (q + (int64_t) h * HD + dim());
#pragma unroll
        for (int i = 0; i < WORDS; i++) x.w[i] = at[i];
        return x;
    }
    __device__ __forceinline__ void fetch(const T * q, int group) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++) w[i] = load(q, min(first() + EACH * i, group - 1));
    }
    __device__ __forceinline__ void codes(const T * q, int group, unsigned char * out) const {
        double pos[2] = {}, neg[2] = {};
        bool odd = false;
        auto add = [&](const words & from) {
            const values y = __builtin_bit_cast(values, from);
#pragma unroll
            for (int d = 0; d < 2; d++) {
                const float x = (float) y.x[d];
                odd |= !(fabsf(x) < INFINITY);
                pos[d] += (double) fmaxf(x, 0.0f);
                neg[d] += (double) fminf(x, 0.0f);
            }
        };
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            if (first() + EACH * i < group) add(w[i]);
        for (int h = first() + EACH * AHEAD; h < group; h += EACH) add(load(q, h));
        float p[2], n[2], top = 0.0f;
#pragma unroll
        for (int d = 0; d < 2; d++) {
            if constexpr (EACH >= 2) { pos[d] = add_across<32>(pos[d]); neg[d] = add_across<32>(neg[d]); }
            if constexpr (EACH >= 4) { pos[d] = add_across<16>(pos[d]); neg[d] = add_across<16>(neg[d]); }
            p[d] = (float) pos[d];
            n[d] = (float) neg[d];
            top = fmaxf(top, fmaxf(p[d], -n[d]));
        }
        top = col_max(row_max16(top));
        if (__any(odd)) top = INFINITY;
        const float inv = top >= LEAST && top < INFINITY ? 127.0f / top : 0.0f;
        auto code = [&](float x) { return inv == 0.0f ? 0u : (uint32_t) (int) rintf(x * inv) & 255u; };
        if (((int) threadIdx.x & 63) < LANES) {
            *(uint16_t *) (out + dim()) = (uint16_t) (code(p[0]) | code(p[1]) << 8);
            *(uint16_t *) (out + HD + dim()) = (uint16_t) (code(n[0]) | code(n[1]) << 8);
        }
    }
};

// pages that the row sees
__device__ __forceinline__ int see_of(const cache_select_args & a, const seq_view & v, int64_t row, int page_shift) {
    return (cache_visible(v.len - v.rows + (int32_t) (row - v.row0), v.len, a.block) + a.page_size - 1) >> page_shift;
}

// Place i of a row's list: the first pages, those found (n, in `found`), the last ones, -1; or all that the row sees
__device__ __forceinline__ int32_t entry(const cache_select_args & a, int i, int see, const uint32_t * found, int n) {
    if (see <= a.take) return i < see ? i : -1;
    return i < a.first ? i : i < a.first + n ? (int32_t) found[i - a.first] : i < a.first + n + a.last ? see - a.last + (i - a.first - n) : -1;
}

// ---------------------------------------------------------------------------------------------- a row a workgroup
struct row_lds {
    uint32_t keys[CAP], pages[CAP], hist[256];
    int32_t count[2][CAP / 64];
    uint32_t range[2][WAVES];
};

// The `keep` largest of 64 WAVES PER keys in registers (key e 64 WAVES + thread in k[e]; 0: none), ties to the first, to the front of l.keys and l.pages in their
// order; by the workgroup. Returns how many.
template <int PER>
__device__ __forceinline__ int best_of(row_lds & l, const uint32_t * k, const uint32_t * p, int keep) {
    const int lane = (int) threadIdx.x & 63, tid = (int) threadIdx.x, wv = uniform(tid >> 6);
    auto clear = [&] { if (tid < 256) l.hist[tid] = 0; };
    // the smallest and largest key, and how many there are
    uint32_t most = 0, least = 0xffffffffu;
    int n = 0;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        most = max(most, k[e]);
        least = min(least, k[e] - 1);      // (0 becomes the largest)
        n += (int) __popcll(__ballot(k[e] != 0));
    }
#define DPP(x, ctrl, rows) (uint32_t) __builtin_amdgcn_update_dpp((int) x, (int) x, ctrl, rows, 0xf, false)
#define JOIN(ctrl, rows) most = max(most, DPP(most, ctrl, rows)); least = min(least, DPP(least, ctrl, rows))
    JOIN(0x111, 0xf); JOIN(0x112, 0xf); JOIN(0x114, 0xf); JOIN(0x118, 0xf); JOIN(0x142, 0xa); JOIN(0x143, 0xc);
#undef JOIN
#undef DPP
    most = (uint32_t) __builtin_amdgcn_readlane((int) most, 63);
    least = (uint32_t) __builtin_amdgcn_readlane((int) least, 63);
    clear();
    if (lane == 0) { l.range[0][wv] = most; l.range[1][wv] = least; l.count[0][wv] = n; }
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        most = max(most, l.range[0][w]);
        least = min(least, l.range[1][w]);
        n += l.count[0][w];
    }
    least++;
    // the last one taken lies in [least, most], `need` of those are taken
    int need = keep;
    if (n <= keep) {      // all of them
        need = n;
    } else {
        for (;;) {
            const int shift = most == least ? 0 : max(0, 24 - __builtin_clz(most - least));
#pragma unroll
            for (int e = 0; e < PER; e++)
                if (k[e] >= least && k[e] <= most) atomicAdd(&l.hist[(k[e] - least) >> shift], 1u);
            __syncthreads();
            // every wave: four bins a lane, from the last
            const int b0 = 255 - lane * 4;
            int c[4], all = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) all += c[j] = (int) l.hist[b0 - j];
            const int upto = wave_scan(all);
            const int at = __builtin_ctzll(__ballot(upto >= need));      // (some lane's: all of the range's are need or more)
            int above = upto - all, bin = b0;
#pragma unroll
            for (int j = 0; j < 3; j++)
                if (bin == b0 - j && above + c[j] < need) { above += c[j]; bin--; }
            const int in = bin == b0 ? c[0] : bin == b0 - 1 ? c[1] : bin == b0 - 2 ? c[2] : c[3];
            need -= __builtin_amdgcn_readlane(above, at);
            const uint32_t from = least + ((uint32_t) __builtin_amdgcn_readlane(bin, at) << shift);
            least = from;
            most = most - from < 1u << shift ? most : from + ((1u << shift) - 1);
            if (need == __builtin_amdgcn_readlane(in, at) || shift == 0) break;
            __syncthreads();
            clear();
            __syncthreads();
        }
    }
    // more than `most`: all; in the range: the first `need`. A group is 64 consecutive keys, of a wave
    uint64_t eq[PER], gt[PER];
    __syncthreads();      // (l.count has been read)
#pragma unroll
    for (int e = 0; e < PER; e++) {
        eq[e] = __ballot(k[e] >= least && k[e] <= most);
        gt[e] = __ballot(k[e] > most);
        if (lane == 0) { l.count[0][e * WAVES + wv] = (int) __popcll(eq[e]); l.count[1][e * WAVES + wv] = (int) __popcll(gt[e]); }
    }
    __syncthreads();
    static_assert(PER * WAVES <= 64, "a group a lane");
    const int of = min(lane, PER * WAVES - 1), mine_eq = lane < PER * WAVES ? l.count[0][of] : 0, mine_gt = lane < PER * WAVES ? l.count[1][of] : 0;
    const int eq_before = wave_scan(mine_eq) - mine_eq, ties = min(max(need - eq_before, 0), mine_eq);
    const int upto = wave_scan(mine_gt + ties), before = upto - mine_gt - ties;
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const int t = __builtin_amdgcn_readlane(ties, e * WAVES + wv), at = __builtin_amdgcn_readlane(before, e * WAVES + wv);
        const bool mine = (gt[e] >> lane & 1) || ((eq[e] >> lane & 1) && (int) __popcll(eq[e] & below) < t);
        const uint64_t in = __ballot(mine);
        if (mine) {
            const int i = at + (int) __popcll(in & below);
            l.keys[i] = k[e];
            l.pages[i] = p[e];
        }
    }
    __syncthreads();
    return __builtin_amdgcn_readlane(upto, 63);
}

// the same of n keys that `of` gives by their number, those of a thread before all threads are past this
template <int PER, typename OF>
__device__ __forceinline__ int best_from(row_lds & l, int keep, OF of) {
    uint32_t k[PER], p[PER];
#pragma unroll
    for (int e = 0; e < PER; e++) of(e * 64 * WAVES + (int) threadIdx.x, k[e], p[e]);
    return best_of<PER>(l, k, p, keep);
}
template <typename OF>
__device__ __forceinline__ int best(row_lds & l, int n, int keep, OF of) {
    static_assert(CAP == 4 * 64 * WAVES, "up to four keys a thread");
    return n <= 64 * WAVES ? best_from<1>(l, keep, of) : n <= 2 * 64 * WAVES ? best_from<2>(l, keep, of) : best_from<4>(l, keep, of);
}

// `work`: a counter for each (row, K/V head) of several pieces, SPLIT_UNITS of them, then [row][K/V head][piece] what they found: keys [take] (0 behind the
// last), pages [take]
struct pieces_view {
    static constexpr int SC1 = 16;
    const brsrc r;
    const uint32_t bytes;
    __device__ pieces_view(const cache_select_args & a, int64_t unit)
        : r(make_brsrc((unsigned char *) a.work + SPLIT_UNITS * 8 + unit * a.pieces * (8 * a.take), (int64_t) a.pieces * (8 * a.take))), bytes(8 * a.take) {}
    __device__ void put(int piece, int i, uint32_t key, uint32_t page) const {
        __builtin_amdgcn_raw_buffer_store_b64(word2_t{key, page}, r, piece * bytes + i * 8, 0, SC1);
    }
    __device__ word2_t get(int piece, int i) const { return __builtin_amdgcn_raw_buffer_load_b64(r, piece * bytes + i * 8, 0, SC1); }
};

template <typename T, int HD>
__global__ __launch_bounds__(64 * WAVES, 4) void k_select_row(cache_select_args a) {
    constexpr int NK = 2 * HD / 64, THREADS = 64 * WAVES, AT_ONCE = (CAP - MOST) / THREADS * THREADS;
    __shared__ __attribute__((aligned(16))) unsigned char codes[2 * HD];
    __shared__ row_lds l;
    const int tid = (int) threadIdx.x, lane = tid & 63, l15 = lane & 15, g = lane >> 4, wv = uniform(tid >> 6);
    const int group = a.n_head / a.n_kv_head, kvh = (int) (blockIdx.x % (unsigned) a.n_kv_head);
    const unsigned at_block = blockIdx.x / (unsigned) a.n_kv_head;
    const int piece = (int) (at_block % (unsigned) a.pieces);
    const int64_t row = at_block / (unsigned) a.pieces;
    const int page_shift = __builtin_ctz((unsigned) a.page_size);
    int seq;
    seq_view v;
    if (!place_of(a, (int32_t) row, seq, v)) return;
    const int see = see_of(a, v, row, page_shift), keep = a.take - a.first - a.last;
    int32_t * const out = a.selected + (row * a.n_kv_head + kvh) * a.take;
    if (see <= a.take || keep == 0) {      // nothing to choose
        if (piece == 0 && tid < a.take) out[tid] = entry(a, tid, see, nullptr, 0);
        return;
    }
    const int p0 = a.first + piece * a.piece, p1 = min(see - a.last, p0 + a.piece);
    int n = 0;
    if (p0 < p1) {
        const int32_t * table = a.table + (int64_t) seq * a.width;
        // a lane's page of 64: the one whose score the matrix tiles will leave in it (tile l15 / 4, its page 4 g + l15 % 4)
        const int mine = (l15 >> 2) * 16 + g * 4 + (l15 & 3);
        const unsigned char * const heads = a.digest + (int64_t) kvh * cache_digest_bytes(HD);
        const int64_t per = a.n_kv_head * cache_digest_bytes(HD);
        int4_t y[4][NK];
        float scale;
        bool bad;
        auto load_page = [&](int p) { return table[min(p + mine, p1 - 1)]; };
        auto load = [&](int32_t next) {
            bad = next < 0 || next >= a.n_pages;
            const int32_t page = bad ? 0 : next;
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const int32_t of = __builtin_amdgcn_ds_bpermute(((l15 >> 2) * 16 + t * 4 + (l15 & 3)) * 4, page);      // the lane of the tile's page l15
                const unsigned char * d = heads + of * per + g * 16;
#pragma unroll
                for (int k = 0; k < NK; k++) y[t][k] = *(const int4_t *) (d + k * 64);
            }
            scale = *(const float *) (heads + page * per + 2 * HD);
        };
        const int32_t first_page = load_page(p0 + wv * 64);
        int32_t next = load_page(p0 + wv * 64 + THREADS);
        const T * q = (const T *) a.q + row * a.ldq + (int64_t) kvh * group * HD;
        row_queries<T, HD> queries;
        if (wv == 0) queries.fetch(q, group);
        load(first_page);      // (on their way while the queries' codes are made)
        if (wv == 0) queries.codes(q, group, codes);
        __syncthreads();
        int4_t b[NK];
#pragma unroll
        for (int k = 0; k < NK; k++) b[k] = *(const int4_t *) (codes + k * 64 + g * 16);      // (every column is the row)
        for (int c0 = p0; c0 < p1; c0 += AT_ONCE) {
            const int c1 = min(c0 + AT_ONCE, p1);
            for (int s0 = c0 + wv * 64; s0 < c1; s0 += THREADS) {
                int dot = 0;
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    int4_t x = {0, 0, 0, 0};
#pragma unroll
                    for (int k = 0; k < NK; k++) x = __builtin_amdgcn_mfma_i32_16x16x64_i8(y[t][k], b[k], x, 0, 0, 0);
                    const int r = l15 & 3, of = r == 0 ? x[0] : r == 1 ? x[1] : r == 2 ? x[2] : x[3];
                    if (l15 >> 2 == t) dot = of;
                }
                const int p = s0 + mine;
                if (p < c1) {
                    l.keys[n + p - c0] = bad ? KEY_LOWEST : key_of((float) dot * scale);
                    l.pages[n + p - c0] = (uint32_t) p;
                }
                if (s0 + THREADS < p1) {      // (the next chunk's begin behind this one's: chunks are whole THREADS)
                    load(next);
                    next = load_page(s0 + 2 * THREADS);
                }
            }
            const int all = n + c1 - c0;
            __syncthreads();
            if (all > keep) {
                auto of = [&](int i, uint32_t & key, uint32_t & page) {
                    key = i < all ? l.keys[i] : 0u;
                    page = i < all ? l.pages[i] : 0u;
                };
                n = best(l, all, keep, of);
            } else {
                n = all;
            }
        }
    }
    if (a.pieces > 1) {
        const int64_t unit = row * a.n_kv_head + kvh;
        const pieces_view w(a, unit);
        static_assert(MOST <= THREADS, "a page a thread");
        if (tid < keep) w.put(piece, tid, tid < n ? l.keys[tid] : 0u, tid < n ? l.pages[tid] : 0u);
        if (!last_to_arrive(a.work, unit, a.pieces)) return;
        // all pieces' in their order, as many pieces at once as fit behind what is kept
        n = 0;
        for (int k0 = 0; k0 < a.pieces;) {
            const int pieces = min((CAP - n) / keep, a.pieces - k0), all = n + pieces * keep;
            auto of = [&](int i, uint32_t & key, uint32_t & page) {
                key = page = 0;
                if (i < n) {
                    key = l.keys[i];
                    page = l.pages[i];
                } else if (i < all) {
                    const word2_t x = w.get(k0 + (i - n) / keep, (i - n) % keep);
                    key = x[0];
                    page = x[1];
                }
            };
            n = best(l, all, keep, of);
            k0 += pieces;
        }
    }
    if (wv == 0)
        for (int i = lane; i < a.take; i += 64) out[i] = entry(a, i, see, l.pages, n);
}

// ---------------------------------------------------------------------------------------------- 16 rows a workgroup
// Lane l15 of each group of 16 has row l15 of the tile, as the matrix instruction leaves the scores, in every wave: its keys of 16 pages of each tile of scores stay in
// registers, what belongs to a row as a whole is in all its lanes, and the rows go through the search in step.
constexpr int TILES = CHUNK / (16 * WAVES);          // tiles of scores of a wave
constexpr int KEPT_KEYS = MOST / (4 * WAVES);        // keys that a lane takes of those that its row has kept
constexpr int SLOTS = 4 * WAVES * (1 + TILES);       // groups of keys of one lane, in the keys' order: the kept ones, then each tile's
constexpr int BINS = 257;                            // of a row, a word between rows
struct rows_lds {
    uint32_t hist[ROWS * BINS];                      // (the slots' counts lie here afterwards)
    __attribute__((aligned(16))) uint32_t edge[3][ROWS][WAVES];
    __attribute__((aligned(16))) uint32_t found[ROWS][4];
    __attribute__((aligned(16))) float scales[CHUNK];
};
static_assert(SLOTS * ROWS <= ROWS * BINS && SLOTS <= 192, "the counts in the histograms' place, three slots a lane");

template <typename T, int HD>
__global__ __launch_bounds__(64 * WAVES, 4) void k_select_rows(cache_select_args a) {
    constexpr int NK = 2 * HD / 64, QS = 2 * HD + 16, EACH = ROWS / WAVES, THREADS = 64 * WAVES;
    __shared__ __attribute__((aligned(16))) unsigned char codes[ROWS * QS];
    __shared__ rows_lds l;
    extern __shared__ __attribute__((aligned(16))) uint32_t lists[];      // what rows keep: keys [ROWS][take], pages [ROWS][take]
    const int tid = (int) threadIdx.x, lane = tid & 63, l15 = lane & 15, g = lane >> 4, wv = uniform(tid >> 6);
    const int group = a.n_head / a.n_kv_head, kvh = (int) (blockIdx.x % (unsigned) a.n_kv_head), page_shift = __builtin_ctz((unsigned) a.page_size);
    const int64_t t0 = (int64_t) (blockIdx.x / (unsigned) a.n_kv_head) * ROWS, t1 = min(t0 + ROWS, a.n_rows);
    const int keep = a.take - a.first - a.last;
    uint32_t * const keys = lists + l15 * a.take, * const pages = lists + (ROWS + l15) * a.take;
    for (int64_t r0 = t0; r0 < t1;) {      // the sequences of the tile's rows
        int seq;
        seq_view v;
        if (!place_of(a, (int32_t) r0, seq, v)) {
            if (r0 >= a.row_start[0]) break;
            r0 = min((int64_t) a.row_start[0], t1);
            continue;
        }
        const int64_t r1 = min(t1, (int64_t) v.row0 + v.rows);
        const int rows = (int) (r1 - r0), see_all = see_of(a, v, r1 - 1, page_shift);      // (the last row sees the most)
        int kept = 0;      // of the lane's row
        if (see_all > a.take && keep > 0) {
            const int p0 = a.first, p1 = see_all - a.last, see = see_of(a, v, min(r0 + l15, r1 - 1), page_shift);
            const int end = l15 < rows && see > a.take ? see - a.last : 0;      // the row's own
            const int32_t * table = a.table + (int64_t) seq * a.width;
            int32_t next[TILES];
            auto load_pages = [&](int c0) {
#pragma unroll
                for (int i = 0; i < TILES; i++) next[i] = table[min(c0 + (wv * TILES + i) * 16 + l15, p1 - 1)];
            };
            load_pages(p0);
            auto q_of = [&](int i) { return (const T *) a.q + min(r0 + wv * EACH + i, r1 - 1) * a.ldq + (int64_t) kvh * group * HD; };
            row_queries<T, HD> queries[EACH];
#pragma unroll
            for (int i = 0; i < EACH; i++) queries[i].fetch(q_of(i), group);
            int4_t y[TILES][NK];
            float scale[TILES];
            auto load = [&] {
#pragma unroll
                for (int i = 0; i < TILES; i++) {
                    const bool bad = next[i] < 0 || next[i] >= a.n_pages;
                    const unsigned char * d = a.digest + ((bad ? 0 : (int64_t) next[i]) * a.n_kv_head + kvh) * cache_digest_bytes(HD);
#pragma unroll
                    for (int k = 0; k < NK; k++) y[i][k] = *(const int4_t *) (d + k * 64 + g * 16);
                    scale[i] = bad ? -1.0f : *(const float *) (d + 2 * HD);
                }
            };
            load();      // (on their way while the queries' codes are made)
#pragma unroll
            for (int i = 0; i < EACH; i++) queries[i].codes(q_of(i), group, codes + (wv * EACH + i) * QS);
            uint32_t pass = 0;      // what a key of the row has to be more than
            // a chunk's pages and, but for the first, those that rows have kept of the ones before
            auto chunk = [&](int c0, auto first) {
                constexpr bool FIRST = decltype(first)::value;
                constexpr int KEPT = FIRST ? 0 : KEPT_KEYS;
                if constexpr (!FIRST) load();
                load_pages(c0 + CHUNK);
                for (int i = tid; i < ROWS * BINS; i += THREADS) l.hist[i] = 0;
                if (g == 0) {
#pragma unroll
                    for (int i = 0; i < TILES; i++) l.scales[(wv * TILES + i) * 16 + l15] = scale[i];
                }
                __syncthreads();
                // keys in their order: KEPT of the row's list, then 4 pages of each tile
                uint32_t k[KEPT + 4 * TILES], kp[KEPT + 1];
#pragma unroll
                for (int j = 0; j < KEPT; j++) {
                    const int at = (wv * 4 + g) * KEPT + j;
                    k[j] = at < kept ? keys[at] : 0u;
                    kp[j] = at < kept ? pages[at] : 0u;
                }
                const int base = c0 + wv * TILES * 16 + g * 4;      // + 16 i + r
                uint32_t most = 0, least = 0xffffffffu;
                int n = 0;
#pragma unroll
                for (int i = 0; i < TILES; i++) {
                    int4_t x = {0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < NK; j++)
                        x = __builtin_amdgcn_mfma_i32_16x16x64_i8(y[i][j], *(const int4_t *) (codes + l15 * QS + j * 64 + g * 16), x, 0, 0, 0);
                    const float4_t f = *(const float4_t *) (l.scales + (wv * TILES + i) * 16 + g * 4);
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const uint32_t key = f[r] < 0.0f ? KEY_LOWEST : key_of((float) x[r] * f[r]);
                        k[KEPT + 4 * i + r] = base + 16 * i + r < end && key > pass ? key : 0u;
                    }
                }
#pragma unroll
                for (int j = 0; j < KEPT + 4 * TILES; j++) {
                    most = max(most, k[j]);
                    least = min(least, k[j] - 1);      // (0 becomes the largest)
                    n += k[j] != 0;
                }
                // the row's: over the four groups, then over the waves
                auto over_groups = [](uint32_t x, auto f) {
                    auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
                    x = f((uint32_t) r[0], (uint32_t) r[1]);
                    r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
                    return f((uint32_t) r[0], (uint32_t) r[1]);
                };
                auto larger = [](uint32_t x, uint32_t y) { return max(x, y); };
                auto smaller = [](uint32_t x, uint32_t y) { return min(x, y); };
                auto sum = [](uint32_t x, uint32_t y) { return x + y; };
                auto over_waves = [&](int which, auto f) {
                    const word4_t x = *(const word4_t *) l.edge[which][l15], z = *(const word4_t *) (l.edge[which][l15] + 4);
                    return f(f(f(x[0], x[1]), f(x[2], x[3])), f(f(z[0], z[1]), f(z[2], z[3])));
                };
                static_assert(WAVES == 8, "two words of four");
                most = over_groups(most, larger);
                least = over_groups(least, smaller);
                n = (int) over_groups((uint32_t) n, sum);
                if (g == 0) {
                    l.edge[0][l15][wv] = most;
                    l.edge[1][l15][wv] = least;
                    l.edge[2][l15][wv] = (uint32_t) n;
                }
                __syncthreads();
                most = over_waves(0, larger);
                least = over_waves(1, smaller) + 1;
                n = (int) over_waves(2, sum);
                // the last one taken lies in [least, most], `need` of those are taken (of no more than `keep` keys: all)
                int need = min(keep, n);
                bool done = n <= keep;
                while (__any(!done)) {      // (the same in every wave)
                    const int shift = most == least ? 0 : max(0, 24 - __builtin_clz(most - least));
#pragma unroll
                    for (int j = 0; j < KEPT + 4 * TILES; j++)
                        if (!done && k[j] >= least && k[j] <= most) atomicAdd(&l.hist[l15 * BINS + ((k[j] - least) >> shift)], 1u);
                    __syncthreads();
#pragma unroll
                    for (int i = 0; i < EACH; i++) {      // a wave finds its rows' bins: four a lane, from the last
                        const int row = wv * EACH + i, b0 = row * BINS + 255 - lane * 4;
                        int c[4], all = 0;
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            all += c[j] = (int) l.hist[b0 - j];
                            l.hist[b0 - j] = 0;
                        }
                        const int want = __builtin_amdgcn_readlane(need, row);
                        const int upto = wave_scan(all);
                        const uint64_t reach = __ballot(upto >= want);
                        if (!reach) continue;      // (a row that is done)
                        const int at = __builtin_ctzll(reach);
                        int above = upto - all, bin = 0;
#pragma unroll
                        for (int j = 0; j < 3; j++)
                            if (bin == j && above + c[j] < want) { above += c[j]; bin++; }
                        const int in = bin == 0 ? c[0] : bin == 1 ? c[1] : bin == 2 ? c[2] : c[3];
                        if (lane == at) *(word4_t *) l.found[row] = word4_t{(uint32_t) (255 - lane * 4 - bin), (uint32_t) (want - above), (uint32_t) in, 0};
                    }
                    __syncthreads();
                    if (!done) {
                        const word4_t f = *(const word4_t *) l.found[l15];
                        least += f[0] << shift;
                        most = most - least < 1u << shift ? most : least + ((1u << shift) - 1);
                        need = (int) f[1];
                        done = f[1] == f[2] || shift == 0;
                    }
                }
                // more than `most`: all; in the range: the first `need`. Counts of every lane's groups of keys (in the range, more << 16), then their sums before each
                uint32_t * const counts = l.hist;
                auto place = [&](int s) { return l15 * SLOTS + s; };
                auto count = [&](int j0, int m) {
                    uint32_t c = 0;
#pragma unroll
                    for (int j = j0; j < j0 + m; j++) c += k[j] > most ? 0x10000u : k[j] >= least && k[j] != 0 ? 1u : 0u;
                    return c;
                };
                if constexpr (!FIRST) counts[place(wv * 4 + g)] = count(0, KEPT);
                else counts[place(wv * 4 + g)] = 0;
#pragma unroll
                for (int i = 0; i < TILES; i++) counts[place(4 * WAVES + (wv * TILES + i) * 4 + g)] = count(KEPT + 4 * i, 4);
                __syncthreads();
#pragma unroll
                for (int i = 0; i < EACH; i++) {
                    uint32_t * const row = counts + (wv * EACH + i) * SLOTS;
                    uint32_t c[3], all = 0;
#pragma unroll
                    for (int j = 0; j < 3; j++) all += c[j] = lane * 3 + j < SLOTS ? row[min(lane * 3 + j, SLOTS - 1)] : 0u;
                    uint32_t before = wave_scan(all) - all;
#pragma unroll
                    for (int j = 0; j < 3; j++) {
                        if (lane * 3 + j < SLOTS) row[lane * 3 + j] = before;
                        before += c[j];
                    }
                }
                __syncthreads();
                auto put = [&](int j0, int m, int slot, auto page_of) {
                    const uint32_t before = counts[place(slot)];
                    int in = (int) (before & 0xffffu), above = (int) (before >> 16);
#pragma unroll
                    for (int j = 0; j < m; j++) {
                        const uint32_t key = k[j0 + j];
                        const bool more = key > most, eq = !more && key >= least && key != 0;
                        if (more || (eq && in < need)) {
                            keys[above + min(in, need)] = key;
                            pages[above + min(in, need)] = page_of(j);
                        }
                        above += more;
                        in += eq;
                    }
                };
                if constexpr (!FIRST) put(0, KEPT, wv * 4 + g, [&](int j) { return kp[j]; });
#pragma unroll
                for (int i = 0; i < TILES; i++) put(KEPT + 4 * i, 4, 4 * WAVES + (wv * TILES + i) * 4 + g, [&](int r) { return (uint32_t) (base + 16 * i + r); });
                kept = min(keep, n);
                if (n > keep) pass = least - 1;
                __syncthreads();
            };
            chunk(p0, std::true_type{});
            for (int c0 = p0 + CHUNK; c0 < p1; c0 += CHUNK) chunk(c0, std::false_type{});
        }
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            const int at = wv * EACH + i;
            if (at >= rows) continue;
            const int see = see_of(a, v, r0 + at, page_shift), n = __builtin_amdgcn_readlane(kept, at);
            int32_t * out = a.selected + ((r0 + at) * a.n_kv_head + kvh) * a.take;
            for (int j = lane; j < a.take; j += 64) out[j] = entry(a, j, see, lists + (ROWS + at) * a.take, n);
        }
        __syncthreads();
        r0 = r1;
    }
}

// A workgroup a row takes time by the rows (some 7 us for 512 rows and K/V heads, after the first), a tile of 16 some 13 us for each sequence that it has rows of, however
// few there are. So tiles where sequences have four rows or more and the rows are worth it. Measured, us of a call with a row / with tiles, rows times K/V heads in
// brackets: 1 sequence of 14000 tokens in pages of 64, 128 rows (512) 12.2 / 13.3, 256 (1024) 16.8 / 13.2, 1024 (4096) 53.0 / 14.6; sequences of 200 to 8000
// in pages of 16: 64 of 1 row (512) 15.6 / 214, of 4 (2048) 38.4 / 65.2, of 8 (4096) 67.4 / 40.5; 16 of 8 (1024) 23.2 / 36.6, of 16 (2048) 35.1 / 22.0.
// These are sequences of equal rows; the rule knows only what the call is sized for. Single tokens beside a prompt, or in a captured call with room for one, come into tiles of
// up to 16 sequences: a token of 63 requests 14.8 us, in a call of 2000 rows 190, beside a prompt of 1000 rows (28.6 by itself) 195.
bool tiles_of(const cache_shape & c, int64_t n_seq, int64_t n_rows) {
    return n_rows >= 4 * n_seq && (double) n_rows * c.n_kv_head * n_rows >= 700.0 * (double) (n_rows + ROWS * n_seq);
}
int pieces_of(const cache_shape & c, int64_t n_seq, int64_t n_rows, int64_t width) {
    if (tiles_of(c, n_seq, n_rows)) return 1;
    return (int) std::clamp<int64_t>(std::min((width + PIECE - 1) / PIECE, SPLIT_UNITS / (n_rows * c.n_kv_head)), 1, MOST_PIECES);
}

int64_t blocks_of(const cache_shape & c, int64_t n_seq, int64_t n_rows, int64_t width) {
    const int rows = tiles_of(c, n_seq, n_rows) ? ROWS : 1;
    return (n_rows + rows - 1) / rows * pieces_of(c, n_seq, n_rows, width) * c.n_kv_head;
}

template <typename T, int HD>
hipError_t select(const cache_shape & c, const cache_select_args & a, hipStream_t s) {
    cache_select_args args = a;
    void * p[] = {&args};
    const bool tiles = tiles_of(c, a.n_seq, a.n_rows);
    args.pieces = pieces_of(c, a.n_seq, a.n_rows, a.width);
    args.piece = (a.width + args.pieces - 1) / args.pieces;
    return hipLaunchKernel(tiles ? (const void *) k_select_rows<T, HD> : (const void *) k_select_row<T, HD>, dim3((unsigned) blocks_of(c, a.n_seq, a.n_rows, a.width)),
                           dim3(64 * WAVES), p, tiles ? (unsigned) (2 * ROWS * a.take * 4) : 0, s);
}

template <typename T>
hipError_t by_head(const cache_shape & c, const cache_select_args & a, hipStream_t s) {
    return c.hd == 32 ? select<T, 32>(c, a, s) : c.hd == 64 ? select<T, 64>(c, a, s) : c.hd == 96 ? select<T, 96>(c, a, s) : select<T, 128>(c, a, s);
}

}  // namespace

// workgroups of 256 threads that the launch's are worth
int64_t cache_select_blocks(const cache_shape & c, int64_t n_seq, int64_t n_rows, int64_t width) {
    return blocks_of(c, n_seq, n_rows, width) * (64 * WAVES / NT);
}

// What any call of no more rows, pages and pages taken needs
int64_t cache_select_work_bytes(const cache_shape & c, int64_t n_rows, int64_t width, int take) {
    const int64_t most = std::min<int64_t>((width + PIECE - 1) / PIECE, MOST_PIECES);
    return most > 1 ? SPLIT_UNITS * 8 + std::min<int64_t>(n_rows * c.n_kv_head * most, SPLIT_UNITS) * 8 * (int64_t) take : 0;
}

hipError_t launch_cache_select(const cache_shape & c, int type, const cache_select_args & a, hipStream_t s) {
    return type == T_F32 ? by_head<float>(c, a, s) : type == T_F16 ? by_head<_Float16>(c, a, s) : by_head<__bf16>(c, a, s);
}
