// cache_attention.hip - attention of packed query rows over the 4-bit paged cache on gfx950.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp2(c (q . k_j) - mu),  k_j[n] = dk_jb (ck_jn - 8), v_j[n] = dv_jb (cv_jn - 8)
//
// Columns are the query rows times the heads of one K/V head ("group"): column = row * group + head. S^T = K Q^T puts one
// column in a lane (16x16x32 f16 MFMA, 16 keys x 16 columns), so the softmax is lane work and P^T feeds the second product,
// O^T += V^T P^T, from its registers.
//
// Numerics. 4-bit codes are exact in f16:
//   - the first product runs on K's codes: the MFMA's depth (32) is one q4_0 block, whose sum is multiplied by dk in f32 and added over
//     the blocks of a head;
//   - q is scaled by a power of two (exact) to a largest value in [2^14, 2^15), so that f16's subnormals begin at 2^-28 of it, and taken as
//     one f16 (f16 and bf16 rows: as they are, to 2^-39 of the row's largest value) or as the sum of two (f32 rows: 22 bits, to the same);
//   - a value dv (cv - 8) has 15 bits at most and is the sum of two f16, exactly (the second one's last bit is dv's, 2^-24 or more). That is half
//     as many MFMAs again as one f16 and, for 2000 f16 rows over 16000 tokens, 8 % of the time of scaled weights on V's codes; but a weight times a
//     scale needs a range that follows V, and then values of other tokens and blocks take its bits;
//   - weights are rounded to one f16 (16-bit rows: half a step of f16, 2^-11 relative at most, as the output's own rounding is or finer,
//     and averaged over the keys) or to the sum of two (f32 rows; the product of both second terms, 2^-22, is left out). mu is the running
//     maximum of the scores less 10, and moves when a tile passes it by more than 2^15: so the largest weight is between 2^10 and 2^15, and
//     f16's smallest step is 2^-34 of it or less. Nothing of V takes part in that: a token that a row must not read cannot change
//     the row, and the blocks of a head may differ in size;
//   - the sum of the weights is that of the rounded ones, by the same instructions (a row of ones beside V^T): the result is a mean
//     of the values, never past the largest, which f16 might not hold.
// Scores, maxima, sums and accumulators are f32.
//
// Few columns (k_cache_attention). The four waves of a workgroup share 16 columns and split the keys, a wave sweeping its tiles of 64
// (4 strips) by itself: no barrier in the loop, the waves' sums are joined in LDS at the end. K codes go from memory to the registers
// of the MFMA's A operand (the strip's layout is the operand's); V codes and scales go through the wave's own LDS, because V^T needs
// 16 keys of one dimension in a lane: ds_read_b64_tr_b4 turns 16 x 16 nibbles around. The next tile's loads (and the page numbers of
// the one after) are in flight while a tile is computed. Measured: 64 requests of 200 to 8000 tokens, f16, 32 heads over 8 of
// 128, 65.5 us (259 MB, 3.95 TB/s; a large copy reaches 5.2); 2 contexts of 90000 to 131000 tokens, bf16, 64 heads over 8, 62.3 us (253 MB,
// 4.05 TB/s). About 8 us of a call are its start (find_unit, the query, the first tile's way from memory, one after the other) and 2 its
// end, then memory bounds it, with the VALU at 57 % (unpacking codes, scales, softmax). With several tiles of columns a sequence
// the VALU bounds it: 8 sequences of 258 f32 rows, 78.5 us, 76 % of its time.
// Many columns (k_cache_prompt): see there.
//
// Work. A unit is (sequence, tile of columns, piece of its keys, K/V head). The piece length is the same for all sequences
// of a call and chosen on the device from the sum of their lengths, so that long sequences are split and short ones are not and
// the chip is filled evenly by ragged batches; the host knows only a bound on the units, and workgroups past the last one
// leave. Pieces of a column tile write their sums to `work`; the last one to arrive adds them in their order, so the result does not
// depend on which that is, and nothing waits for another workgroup.
#include "cache_attn_dev.h"
#include "common.h"

#include <algorithm>
#include <type_traits>

namespace {

constexpr int PIECE = 4 * TILE;      // pieces are multiples of this: one step of each of four waves
constexpr int piece_min(int c) { return c == 16 ? PIECE : 2 * PIECE; }      // many columns' sums are more to write and to join

// Workgroups that a CU holds, by its registers (512 of a SIMD lane) and LDS, of the kernel for column tiles of c; and the chip (256
// CUs). Calls whose column tiles alone are fewer are split into about as many units, or up to twice as many where that ends more
// evenly: of 64 requests of 200 to 8000 tokens, as many units as slots took 73 us, twice as many 67.
template <typename T> constexpr int groups_of(int hd, int c) { return c == 128 ? 2 : c == 64 ? (sizeof(T) == 4 && hd == 128 ? 3 : 4) : hd > 64 ? 3 : 4; }
template <typename T> constexpr int slots_of(int hd, int c) { return 256 * groups_of<T>(hd, c); }
// What a unit costs beside its keys, in keys; and how many units a call is split into at most, in slots
// (24 requests of 5 f16 rows, two column tiles each: 37.5 us, with 384 keys 42.1, with 1536 37.5; single tokens and frames do not change)
constexpr float UNIT_KEYS = 768.0f;
constexpr float MOST_UNITS = 1.9f;

// A piece of a column tile: keys [piece, piece + 1) * length of sequence v; part: the first piece's place in `work`
struct unit { seq_view v; int seq, tile, piece, pieces; int32_t length; int64_t part; };

// Column tiles of a sequence, and its pieces where pieces are to be about 1 / inv keys (the nearest number of equal ones)
template <int C> __device__ __forceinline__ uint32_t tiles_of(const seq_view & v, int group) {
    return ((uint32_t) v.rows * (uint32_t) group + C - 1) / C;      // (rows * heads are below 2^27)
}
__device__ __forceinline__ float pieces_of(const seq_view & v, float inv) { return fmaxf(floorf(__builtin_fmaf((float) v.len, inv, 0.5f)), 1.0f); }
// the inverse length of `units` equal pieces of `keys` keys (over all sequences, column tiles and K/V heads). Float sums and
// reciprocals will do: every workgroup makes the same ones of the same numbers.
template <int C> __device__ __forceinline__ float piece_inv(float keys, float units) {
    return __builtin_amdgcn_rcpf(fmaxf(keys * (1.0f / units), (float) piece_min(C)));
}

__device__ __forceinline__ float wave_max(float x) {      // (of values that are not negative)
#define DPP(ctrl, rows) __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), ctrl, rows, 0xf, true))
    x = fmaxf(x, DPP(0x111, 0xf));
    x = fmaxf(x, DPP(0x112, 0xf));
    x = fmaxf(x, DPP(0x114, 0xf));
    x = fmaxf(x, DPP(0x118, 0xf));
    x = fmaxf(x, DPP(0x142, 0xa));
    x = fmaxf(x, DPP(0x143, 0xc));
#undef DPP
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}
// Unit x of the call, for column tiles of C. Every thread gets it, in scalar registers; false past the last. Sequences whose rows overlap
// may have more units than the launch has workgroups: then nothing is computed, for a tile that only some of its pieces come to would
// leave its counter in `work` short.
// Up to 64 sequences each wave finds it by itself, a sequence a lane, and weighs a few piece lengths against each other; more are
// dealt to the workgroup's threads.
template <int C, int SLOTS>
__device__ __forceinline__ bool find_unit(const cache_attn_args & a, uint32_t x, unit & u) {
    const int tid = (int) threadIdx.x, lane = tid & 63, wv = tid >> 6, group = a.n_head / a.n_kv_head;
    auto set = [&](unit & f, const seq_view & v, int i, uint32_t tiles, uint32_t pieces, uint32_t at, uint32_t part) {
        f.v = v;
        f.seq = i;
        f.tile = (int) (tiles - 1 - at / pieces);      // a prompt's last rows read the most keys: they go first
        f.piece = (int) (at % pieces);
        f.pieces = (int) pieces;
        f.length = (int32_t) (((uint32_t) v.len + pieces * PIECE - 1) / (pieces * PIECE) * PIECE);
        f.part = (int64_t) part + (int64_t) f.tile * (int64_t) pieces;
    };
    if (a.n_seq <= 64) {
        seq_view v = {};
        if (lane < a.n_seq) v = view_of(a, lane);
        const uint32_t tiles = tiles_of<C>(v, group);
        const float heads = (float) a.n_kv_head, keys = wave_add((float) tiles * (float) v.len) * heads;
        float inv = 0.0f, least = INFINITY;
#pragma unroll
        for (int i = 0; i < 3; i++) {
            // so many units for each slot: the time of all, and of the longest while the last round is not full. A little less than one: the
            // rounding of pieces may not then add a second round (24 requests of 5 f16 rows 37.5 us, without it 41.8). Only the last would do
            // for ragged single tokens, but takes 71 us instead of 62 for two long contexts.
            constexpr float SHARE[3] = {1.0f, 0.93f, MOST_UNITS};
            const float x1 = piece_inv<C>(keys, SHARE[i] * SLOTS), n = pieces_of(v, x1);
            const float units = wave_add((float) tiles * n) * heads, rounds = units * (1.0f / SLOTS);
            const float longest = wave_max(tiles ? (float) v.len * __builtin_amdgcn_rcpf(n) : 0.0f) + UNIT_KEYS;
            const float time = fmaxf(__builtin_fmaf(units, UNIT_KEYS, keys) * (1.0f / SLOTS) + longest * (ceilf(rounds) - rounds), longest);
            if (time < least) { least = time; inv = x1; }
        }
        const uint32_t pieces = (uint32_t) pieces_of(v, inv), n = tiles * pieces, parts = pieces > 1 ? tiles * pieces : 0u;
        const uint32_t upto = wave_scan(n), parts_upto = wave_scan(parts);
        const uint64_t mine = __ballot(x >= upto - n && x < upto);
        if (!mine || (uint32_t) __builtin_amdgcn_readlane((int) upto, 63) > a.units) return false;
        const int i = __builtin_ctzll(mine);
        auto of = [&](uint32_t y) { return (uint32_t) __builtin_amdgcn_readlane((int) y, i); };
        set(u, {(int32_t) of((uint32_t) v.row0), (int32_t) of((uint32_t) v.rows), (int32_t) of((uint32_t) v.len)}, i, of(tiles), of(pieces),
            x - of(upto - n), of(parts_upto - parts));
        return true;
    }
    __shared__ float keys4[NT / 64], tiles4[NT / 64];
    __shared__ uint32_t sums[2][NT / 64];
    __shared__ struct { seq_view v; int seq; uint32_t tiles, pieces, at, part; } found;
    const int per = (a.n_seq + NT - 1) / NT, i0 = min(tid * per, a.n_seq), i1 = min(i0 + per, a.n_seq);
    float keys = 0.0f, all_tiles = 0.0f;
    for (int i = i0; i < i1; i++) {
        const seq_view v = view_of(a, i);
        const float tiles = (float) tiles_of<C>(v, group);
        keys += tiles * (float) v.len;
        all_tiles += tiles;
    }
    keys = wave_add(keys);
    all_tiles = wave_add(all_tiles);
    if (lane == 0) { keys4[wv] = keys; tiles4[wv] = all_tiles; }
    if (tid == 0) found.seq = -1;
    __syncthreads();
    if ((tiles4[0] + tiles4[1]) + (tiles4[2] + tiles4[3]) > 0x1p24f) return false;      // (more than any launch's; the sums below are 32 bits)
    const float inv = piece_inv<C>(((keys4[0] + keys4[1]) + (keys4[2] + keys4[3])) * (float) a.n_kv_head, MOST_UNITS * SLOTS);
    uint32_t mine = 0, parts = 0;
    for (int i = i0; i < i1; i++) {
        const seq_view v = view_of(a, i);
        const uint32_t tiles = tiles_of<C>(v, group), pieces = (uint32_t) pieces_of(v, inv);
        mine += tiles * pieces;
        parts += pieces > 1 ? tiles * pieces : 0;
    }
    uint32_t before = wave_scan(mine), parts_before = wave_scan(parts);
    if (lane == 63) { sums[0][wv] = before; sums[1][wv] = parts_before; }
    __syncthreads();
    if (sums[0][0] + sums[0][1] + sums[0][2] + sums[0][3] > a.units) return false;
    for (int w = 0; w < wv; w++) { before += sums[0][w]; parts_before += sums[1][w]; }
    before -= mine;
    parts_before -= parts;
    if (x >= before && x < before + mine) {
        uint32_t at = x - before;
        for (int i = i0; i < i1; i++) {
            const seq_view v = view_of(a, i);
            const uint32_t tiles = tiles_of<C>(v, group), pieces = (uint32_t) pieces_of(v, inv), n = tiles * pieces;
            if (at < n) {
                found = {v, i, tiles, pieces, at, parts_before};
                break;
            }
            at -= n;
            parts_before += pieces > 1 ? tiles * pieces : 0;
        }
    }
    __syncthreads();
    if (found.seq < 0) return false;
    set(u, {uniform(found.v.row0), uniform(found.v.rows), uniform(found.v.len)}, uniform(found.seq), (uint32_t) uniform((int) found.tiles),
        (uint32_t) uniform((int) found.pieces), (uint32_t) uniform((int) found.at), (uint32_t) uniform((int) found.part));
    return true;
}

// 16 dimensions x 32 keys of V as the A operand, from rows of f16 VS bytes apart: lane i of 16 names row i / 4, its 4 values i % 4
template <int VS>
__device__ __forceinline__ half8_t read_v(const unsigned char * at, int h) {
    typedef short short4_t __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) short4_t * lds4;
    const half4_t x = __builtin_bit_cast(half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4) (at + (2 * h) * 16 * VS)));
    const half4_t y = __builtin_bit_cast(half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4) (at + (2 * h + 1) * 16 * VS)));
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
}

template <int HD> constexpr int group_lds() {
    const int loop = 4 * wave_lds<HD>(), join = 4 * 16 * (HD + 4) * 4 + 4 * 16 * 8;
    return loop > join ? loop : join;
}

template <typename T, int HD>
__global__ __launch_bounds__(NT, groups_of<T>(HD, 16)) void k_cache_attention(cache_attn_args a) {
    constexpr int NB = HD / 32, ND = HD / 16, TERMS = sizeof(T) == 4 ? 2 : 1, C = 16;
    __shared__ __attribute__((aligned(16))) unsigned char lds[group_lds<HD>()];
    unit u;
    const int kvh = (int) (blockIdx.x % (unsigned) a.n_kv_head);
    if (!find_unit<C, slots_of<T>(HD, C)>(a, blockIdx.x / (unsigned) a.n_kv_head, u)) return;
    if (u.pieces > 1 && u.part + u.pieces > a.parts) return;      // (row_start that overlaps itself: more pieces than rows can have)
    const int tid = (int) threadIdx.x, lane = tid & 63, l15 = lane & 15, g = lane >> 4, wv = uniform(tid >> 6);
    const int seq = u.seq, group = a.n_head / a.n_kv_head;
    const seq_view sv = u.v;
    const int32_t n_cols = sv.rows * group;      // (below 2^27)
    const int32_t col0 = u.tile * C;
    auto query_at = [&](int32_t col) { return (const T *) a.q + (sv.row0 + (int64_t) ((uint32_t) col / (uint32_t) group)) * a.ldq + ((int64_t) kvh * group + (uint32_t) col % (uint32_t) group) * HD; };
    auto visible = [&](int32_t col) { return cache_visible(sv.len - sv.rows + (int32_t) ((uint32_t) col / (uint32_t) group), sv.len, a.block); };

    // the keys that the first and the last of the wave's columns read
    const int32_t lim_lo = visible(col0), lim_hi = visible(min(col0 + C, n_cols) - 1);

    // this wave's tiles of the unit's keys
    constexpr int STEP = 4 * TILE;
    const int32_t kend = (int32_t) min<int64_t>((int64_t) (u.piece + 1) * u.length, lim_hi);
    int32_t k0 = ((int32_t) min<int64_t>((int64_t) u.piece * u.length + wv * TILE, 0x7fffff00));
    const int last_strip = (kend - 1) / 16, strips_of_page = a.page_size / 16, page_shift = __builtin_ctz(strips_of_page);
    const int32_t * table = a.table + (int64_t) seq * a.width;
    auto load_pages = [&](int32_t key) { return table[min(key / 16 + (lane & 3), last_strip) >> page_shift]; };
    uint32_t kn[4][NB], vn[4][NB], sn[4], bad_n = 0;      // the tile's codes and scales, in flight
    int pages = k0 < kend ? load_pages(k0) : 0;            // page numbers of the next one, in lanes 0 to 3
    const int32_t col = min(col0 + l15, n_cols - 1), lim = visible(col);
    typename vec8<T>::t y[NB];      // the query row, fetched while the first page numbers are
    fetch_query<T, HD>(query_at(col), g, y);
    __builtin_amdgcn_sched_barrier(0);
    // a strip as a buffer resource (no bytes past the end of this wave's keys: such loads give 0 without a memory access)
    auto strip_of = [&](int32_t key, int pages, int t, uint32_t & bad) {
        const int strip = min(key / 16 + t, last_strip);
        int64_t page = __builtin_amdgcn_readlane(pages, t);
        if (page < 0 || page >= a.n_pages) { page = 0; bad |= 1u << t; }
        return make_brsrc(a.cache + ((page * a.n_kv_head + kvh) * strips_of_page + (strip & (strips_of_page - 1))) * (18 * HD), key < kend ? 18 * HD : 0);
    };
    brsrc strips[4];
    auto load_v = [&](int32_t key, int pages) {
        bad_n = 0;
#pragma unroll
        for (int t = 0; t < 4; t++) {
            strips[t] = strip_of(key, pages, t, bad_n);
            load_words<NB>(vn[t], strips[t], lane * (4 * NB), 8 * HD);
            load_words<1>(&sn[t], strips[t], 16 * HD + lane * 4, 0);      // (0 past the strip's scales, from lane HD / 2 on)
        }
    };
    auto load_k = [&] {      // of the tile whose load_v came last
#pragma unroll
        for (int t = 0; t < 4; t++) load_words<NB>(kn[t], strips[t], lane * (4 * NB), 0);
    };
    unsigned char * const mine = lds + wv * wave_lds<HD>();
    unsigned char * const scales = mine + ND * 528;
    // where this lane's V words go, [dimension tile][64 keys][8 bytes], and the row that it names for the transposed read
    const int e = (l15 & 3) * 2 + ((l15 & 7) >> 2);
    const int tr_at = (((l15 >> 3) * 2 + (e >> 2)) * 16 + g * 4 + (e & 3)) * 8;
    if (k0 < kend) {
        const int pages_after = load_pages(k0 + STEP);
        load_v(k0, pages);
        load_k();
        pages = pages_after;
    }
    float c;
    half8_t q[NB][TERMS];
    turn_query<T, HD, TERMS>(a.scale, y, q, c);
    float4_t o[ND + 1];      // the last: the weights' sum, four times
    float mu = -INFINITY;     // (before the first key)
    for (int d = 0; d <= ND; d++) o[d] = float4_t{0, 0, 0, 0};

    uint32_t k1024 = 0x64006400u;
    asm volatile("" : "+v"(k1024));
    // one tile: MASKED where it passes some column's last key, the end, or has a page that is none
    auto tile = [&](auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        const uint32_t bad = bad_n;
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
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const int w = (lane & 3) * NB + b;
                *(uint32_t *) (mine + (w >> 1) * 528 + (t * 16 + (lane >> 2)) * 8 + (w & 1) * 4) = vn[t][b];
            }
        }
        // in the order of their use: a wait for one load is a wait for all before it
        const int pages_after = load_pages(k0 + 2 * STEP);
        load_v(k0 + STEP, pages);
        wave_order();

        // scores
        float4_t s[4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const half4_t * dk = (const half4_t *) (scales + t * 2 * HD + g * (8 * NB));
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const half8_t kc = codes8(kn[t][b], k1024);
                const half4_t d = dk[b];
                float4_t x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, q[b][0], float4_t{0, 0, 0, 0}, 0, 0, 0);
                if constexpr (TERMS == 2) x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, q[b][1], x, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; r++) s[t][r] = __builtin_fmaf((float) d[r], x[r], b == 0 ? 0.0f : s[t][r]);
            }
            __builtin_amdgcn_sched_barrier(0x100);
        }
        load_k();
        pages = pages_after;
        softmax_step<MASKED, ND>(s, k0 + g * 4, lim, bad, c, mu, o);
        half8_t p[2][TERMS];
#pragma unroll
        for (int h = 0; h < 2; h++) turn_weights<TERMS>(s, h, p[h], o[ND]);
        // O^T += V^T P^T, block by block of the head
#pragma unroll
        for (int b = 0; b < NB; b++) {
#pragma unroll
            for (int dd = 0; dd < 2; dd++) {
                const int d = 2 * b + dd;
                const int2_t w = __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) int2_t *) (mine + d * 528 + tr_at));
#pragma unroll
                for (int h = 0; h < 2; h++)
                    o[d] = add_values<TERMS>(codes8((uint32_t) w[h], k1024), scales + HD + g * (8 * NB) + b * 8 + 2 * h * (2 * HD), 2 * HD, p[h], o[d]);
            }
            __builtin_amdgcn_sched_barrier(0x100);
        }
    };
    for (; k0 + TILE <= min(lim_lo, kend) && bad_n == 0; k0 += STEP) tile(std::false_type{});
    for (; k0 < kend; k0 += STEP) tile(std::true_type{});

    const parts_view<HD, C> part(a.work, a.parts, a.n_kv_head, u.part, kvh);
    auto out_at = [&](int32_t col) { return (T *) a.out + (sv.row0 + (int64_t) ((uint32_t) col / (uint32_t) group)) * a.ldo + ((int64_t) kvh * group + (uint32_t) col % (uint32_t) group) * HD; };
    // the four waves' sums at the largest of their maxima
    float * const stat = (float *) (lds + 4 * C * (HD + 4) * 4), * const sum = (float *) lds;
    __syncthreads();      // the loop's LDS is read out
    if (g == 0) {
        stat[(wv * C + l15) * 2] = mu;
        stat[(wv * C + l15) * 2 + 1] = o[ND][0];
    }
#pragma unroll
    for (int d = 0; d < ND; d++) *(float4_t *) (sum + (wv * C + l15) * (HD + 4) + d * 16 + g * 4) = o[d];
    __syncthreads();
    for (int i = tid; i < C * (HD / 4); i += NT) {
        const int at = i / (HD / 4), n = i % (HD / 4) * 4;
        if (col0 + at >= n_cols) break;
        float top = -INFINITY, all = 0.0f;
        for (int w = 0; w < 4; w++) top = fmaxf(top, stat[(w * C + at) * 2]);
        const float m = top == -INFINITY ? 0.0f : top;
        float4_t x = {0, 0, 0, 0};
        for (int w = 0; w < 4; w++) {
            const float f = __builtin_amdgcn_exp2f(stat[(w * C + at) * 2] - m);
            all += stat[(w * C + at) * 2 + 1] * f;
            x += *(const float4_t *) (sum + (w * C + at) * (HD + 4) + n) * f;
        }
        if (u.pieces > 1) {
            if (n == 0) part.put_stat(u.piece, at, top, all);
            part.put(u.piece, at, n, x);
        } else {
            store4(out_at(col0 + at) + n, x * (all == 0.0f ? 0.0f : 1.0f / all));
        }
    }
    if (u.pieces > 1 && last_to_arrive(a.work, u.part * a.n_kv_head + kvh, u.pieces)) join_pieces<T>(part, u.pieces, n_cols - col0, [&](int at) { return out_at(col0 + at); });
}

// Prompts: many columns for each key, so what a key costs is paid once a workgroup. Its four waves have 16 or 32 columns each; a
// tile's codes are turned into f16 once, by all four (a strip each), into LDS, K as rows for the A operand and V as rows that
// ds_read_b64_tr_b16 turns around. The next tile's codes are in flight meanwhile.
// For bf16 rows the scales go in with the codes (K and V rounded to f16, 2^-11 relative, against bf16's half step of 2^-8): no
// work per score is left but the softmax, and two column tiles a wave with two LDS buffers (one barrier a tile, two
// workgroups a CU) are best: 17.6k prompt rows of 32 x 128 take 0.80 ms, one column tile took 1.04 (then 0.81).
// f16 and f32 rows keep codes in LDS and the arithmetic above, K's scales in 32 bits and V as two f16, more than twice the work per score; what
// hides its latencies best is four workgroups a CU, of one column tile a wave and one buffer: 2000 f16 rows over 16000 tokens take 1.03 ms,
// two column tiles 1.12, with two buffers 1.14.
// Rows of both are padded by 32 bytes: of 16, 32 and 48 for either this has the fewest bank conflicts (f16, with scaled weights, 954 us; 16 and
// 32 971, 32 and 48 966, 48 and 32 970).
// Rates: 865 TFLOP/s for bf16 (three quarters of an 8192^3 product's 1130; the LDS reads of K and V take as many cycles as the MFMAs)
// and 475 for f16 (32 heads over 4: the VALU 63 % of the time, 8 instructions for each MFMA, most of them scales, the LDS 55 %, the MFMAs 30 %).
template <typename T> struct prompt {
    static constexpr bool scaled = std::is_same<T, __bf16>::value;
    static constexpr int tiles = scaled ? 2 : 1, bufs = scaled ? 2 : 1, columns = 64 * tiles;
};
template <typename T, int HD>
__global__ __launch_bounds__(NT, groups_of<T>(HD, prompt<T>::columns)) void k_cache_prompt(cache_attn_args a) {
    constexpr bool SCALED = prompt<T>::scaled;
    constexpr int CT = prompt<T>::tiles, BUFS = prompt<T>::bufs, NB = HD / 32, ND = HD / 16, TERMS = sizeof(T) == 4 ? 2 : 1, WC = 16 * CT, C = 4 * WC;
    constexpr int KS = 2 * HD + 32, VS = 2 * HD + 32, SCALES = TILE * (KS + VS), BUF = SCALES + (SCALED ? 0 : 8 * HD);
    __shared__ __attribute__((aligned(16))) unsigned char lds[BUFS * BUF];
    __shared__ uint32_t tile_bad[BUFS][4];
    unit u;
    const int kvh = (int) (blockIdx.x % (unsigned) a.n_kv_head);
    if (!find_unit<C, slots_of<T>(HD, C)>(a, blockIdx.x / (unsigned) a.n_kv_head, u)) return;
    if (u.pieces > 1 && u.part + u.pieces > a.parts) return;
    const int tid = (int) threadIdx.x, lane = tid & 63, l15 = lane & 15, g = lane >> 4, wv = uniform(tid >> 6);
    const int seq = u.seq, group = a.n_head / a.n_kv_head;
    const seq_view sv = u.v;
    const int32_t n_cols = sv.rows * group;      // (below 2^27)
    const int32_t first = u.tile * C, col0 = first + wv * WC;
    auto query_at = [&](int32_t col) { return (const T *) a.q + (sv.row0 + (int64_t) ((uint32_t) col / (uint32_t) group)) * a.ldq + ((int64_t) kvh * group + (uint32_t) col % (uint32_t) group) * HD; };
    auto out_at = [&](int32_t col) { return (T *) a.out + (sv.row0 + (int64_t) ((uint32_t) col / (uint32_t) group)) * a.ldo + ((int64_t) kvh * group + (uint32_t) col % (uint32_t) group) * HD; };
    auto visible = [&](int32_t col) { return cache_visible(sv.len - sv.rows + (int32_t) ((uint32_t) col / (uint32_t) group), sv.len, a.block); };
    const bool has = col0 < n_cols;
    const int32_t lim_lo = has ? visible(col0) : 0, lim_hi = has ? visible(min(col0 + WC, n_cols) - 1) : 0;
    const int32_t kend = (int32_t) min<int64_t>((int64_t) (u.piece + 1) * u.length, visible(min(first + C, n_cols) - 1));      // the workgroup's
    int32_t k0 = ((int32_t) min<int64_t>((int64_t) u.piece * u.length, 0x7fffff00));

    // this wave's strip of a tile: codes and scales on their way to LDS
    const int last_strip = (kend - 1) / 16, strips_of_page = a.page_size / 16, page_shift = __builtin_ctz(strips_of_page);
    const int32_t * table = a.table + (int64_t) seq * a.width;
    auto load_page = [&](int32_t key) { return table[min(key / 16 + wv, last_strip) >> page_shift]; };
    uint32_t kx[NB], vx[NB], sx[SCALED ? NB + 2 : 1], bad = 0;
    int32_t page_n = k0 < kend ? load_page(k0) : 0;
    const int vb0 = g * NB >> 2, vb1 = (g * NB + NB - 1) >> 2;      // blocks of the lane's first and last V word
    auto load = [&](int32_t key) {
        const int strip = min(key / 16 + wv, last_strip);
        int64_t page = __builtin_amdgcn_readfirstlane(page_n);
        bad = page < 0 || page >= a.n_pages;
        if (bad) page = 0;
        const brsrc s = make_brsrc(a.cache + ((page * a.n_kv_head + kvh) * strips_of_page + (strip & (strips_of_page - 1))) * (18 * HD), key < kend ? 18 * HD : 0);
        load_words<NB>(kx, s, lane * (4 * NB), 0);
        load_words<NB>(vx, s, l15 * (16 * NB) + g * (4 * NB), 8 * HD);
        if constexpr (SCALED) {
#pragma unroll
            for (int b = 0; b < NB; b++) sx[b] = __builtin_amdgcn_raw_buffer_load_b16(s, cache_k_scale(l15, b, HD), 0, 0);
            sx[NB] = __builtin_amdgcn_raw_buffer_load_b16(s, cache_v_scale(l15, vb0, HD), 0, 0);
            sx[NB + 1] = NB == 3 ? (uint32_t) __builtin_amdgcn_raw_buffer_load_b16(s, cache_v_scale(l15, vb1, HD), 0, 0) : sx[NB];
        } else {
            load_words<1>(sx, s, 16 * HD + lane * 4, 0);      // (0 past the strip's scales, from lane HD / 2 on)
        }
        page_n = load_page(key + TILE);
    };
    uint32_t k1024 = 0x64006400u;
    asm volatile("" : "+v"(k1024));
    auto scale2 = [](half8_t x, uint32_t d) {
        const _Float16 h = __builtin_bit_cast(_Float16, (uint16_t) d);
        return x * half8_t{h, h, h, h, h, h, h, h};
    };
    auto stage = [&](int32_t key, int buf) {      // the strip that load(key) brought
        unsigned char * const l = lds + buf * BUF;
        const bool ok = key + wv * 16 + l15 < kend && !bad;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            half8_t x = codes8(kx[b], k1024);
            if constexpr (SCALED) x = scale2(x, ok ? sx[b] : 0u);
            *(half8_t *) (l + (wv * 16 + l15) * KS + b * 64 + g * 16) = x;
        }
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const int w = g * NB + b;
            half8_t x = codes8(vx[b], k1024);
            x = half8_t{x[0], x[2], x[4], x[6], x[1], x[3], x[5], x[7]};      // dims in order
            if constexpr (SCALED) x = scale2(x, !ok ? 0u : w >> 2 == vb0 ? sx[NB] : sx[NB + 1]);
            *(half8_t *) (l + TILE * KS + (wv * 16 + l15) * VS + w * 16) = x;
        }
        if constexpr (!SCALED) {
            const int d = lane % (HD / 4);
            const int32_t at = key + wv * 16 + d / (2 * NB) * 4 + (d & 1) * 2;
            const uint32_t sc = at >= kend || bad ? 0u : at + 1 >= kend ? sx[0] & 0xffffu : sx[0];
            if (lane < HD / 2) *(uint32_t *) (l + SCALES + wv * 2 * HD + lane * 4) = sc;
        }
        if (lane == 0) tile_bad[buf][wv] = bad;
    };

    float c[CT];
    half8_t q[CT][NB][TERMS];
    int32_t lim[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        typename vec8<T>::t y[NB];
        fetch_query<T, HD>(query_at(min(col0 + ct * 16 + l15, n_cols - 1)), g, y);
        turn_query<T, HD, TERMS>(a.scale, y, q[ct], c[ct]);
    }
#pragma unroll
    for (int ct = 0; ct < CT; ct++) lim[ct] = visible(min(col0 + ct * 16 + l15, n_cols - 1));
    float4_t o[CT][ND + 1];
    float mu[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        mu[ct] = -INFINITY;
        for (int d = 0; d <= ND; d++) o[ct][d] = float4_t{0, 0, 0, 0};
    }

    int buf = 0;
    const int tr_at = TILE * KS + (g * 4 + (l15 >> 2)) * VS + (lane & 3) * 8;
    auto tile = [&](auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        const unsigned char * const m = lds + buf * BUF, * const scales = m + SCALES;
        uint32_t hidden = 0;
        if constexpr (MASKED) hidden = tile_bad[buf][0] | tile_bad[buf][1] << 1 | tile_bad[buf][2] << 2 | tile_bad[buf][3] << 3;
        float4_t s[CT][4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
#pragma unroll
            for (int ct = 0; ct < CT; ct++) s[ct][t] = float4_t{0, 0, 0, 0};
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const half8_t kc = *(const half8_t *) (m + (t * 16 + l15) * KS + b * 64 + g * 16);
                if constexpr (SCALED) {
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) s[ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, q[ct][b][0], s[ct][t], 0, 0, 0);
                } else {
                    const half4_t d = *(const half4_t *) (scales + t * 2 * HD + g * (8 * NB) + b * 8);
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) {
                        float4_t x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, q[ct][b][0], float4_t{0, 0, 0, 0}, 0, 0, 0);
                        if constexpr (TERMS == 2) x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, q[ct][b][1], x, 0, 0, 0);
#pragma unroll
                        for (int r = 0; r < 4; r++) s[ct][t][r] = __builtin_fmaf((float) d[r], x[r], s[ct][t][r]);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0x100);
        }
#pragma unroll
        for (int ct = 0; ct < CT; ct++) softmax_step<MASKED, ND>(s[ct], k0 + g * 4, lim[ct], hidden, c[ct], mu[ct], o[ct]);
        half8_t p[CT][2][TERMS];
#pragma unroll
        for (int ct = 0; ct < CT; ct++)
#pragma unroll
            for (int h = 0; h < 2; h++) turn_weights<TERMS>(s[ct], h, p[ct][h], o[ct][ND]);
#pragma unroll
        for (int d = 0; d < ND; d++) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const half8_t v = read_v<VS>(m + tr_at + d * 32, h);
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
                    if constexpr (SCALED) o[ct][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[ct][h][0], o[ct][d], 0, 0, 0);
                    else o[ct][d] = add_values<TERMS>(v, scales + HD + g * (8 * NB) + (d >> 1) * 8 + 2 * h * (2 * HD), 2 * HD, p[ct][h], o[ct][d]);
                }
            }
            if (d & 1) __builtin_amdgcn_sched_barrier(0x100);
        }
    };
    if (k0 < kend) {
        load(k0);
        stage(k0, 0);
        load(k0 + TILE);
    }
    __syncthreads();
    auto step = [&](auto masked) {
        if constexpr (BUFS == 2) {
            if (k0 + TILE < kend) stage(k0 + TILE, buf ^ 1);
            load(k0 + 2 * TILE);
            if (k0 < lim_hi) tile(masked);
            buf ^= 1;
        } else {
            if (k0 < lim_hi) tile(masked);
            __syncthreads();
            if (k0 + TILE < kend) stage(k0 + TILE, 0);
            load(k0 + 2 * TILE);
        }
        __syncthreads();
    };
    auto no_bad = [&] { return (tile_bad[buf][0] | tile_bad[buf][1] | tile_bad[buf][2] | tile_bad[buf][3]) == 0; };
    for (; k0 + TILE <= min(lim_lo, kend) && no_bad(); k0 += TILE) step(std::false_type{});
    for (; k0 < kend; k0 += TILE) step(std::true_type{});

    if (u.pieces == 1) {
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            const int32_t col = col0 + ct * 16 + l15;
            if (col >= n_cols) continue;
            const float l = o[ct][ND][0], inv = l == 0.0f ? 0.0f : 1.0f / l;
            T * p = out_at(col);
            for (int d = 0; d < ND; d++) store4(p + d * 16 + g * 4, o[ct][d] * inv);
        }
        return;
    }
    const parts_view<HD, C> part(a.work, a.parts, a.n_kv_head, u.part, kvh);
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        const int32_t at = wv * WC + ct * 16 + l15;
        if (first + at >= n_cols) continue;
        if (g == 0) part.put_stat(u.piece, at, mu[ct], o[ct][ND][0]);
        for (int d = 0; d < ND; d++) part.put(u.piece, at, d * 16 + g * 4, o[ct][d]);
    }
    if (last_to_arrive(a.work, u.part * a.n_kv_head + kvh, u.pieces)) join_pieces<T>(part, u.pieces, n_cols - first, [&](int at) { return out_at(first + at); });
}

// Column tiles: 16 (the four waves split the keys) or the prompts'. A prompt's workgroup does more for each key that it stages, so
// it is the faster one where sequences have many columns, and with fewer where the call's columns over all K/V heads (its heads of
// rows) fill the chip, less what its last tiles leave empty; else 16 columns are, split into fewer pieces. Measured, us of a call,
// 16 columns / prompts', rows of 8 K/V heads of 128:
//   1 sequence of 16000 tokens: 256 columns bf16 65 / 99, f16 58 / 106, f32 68 / 86; 1024 columns 190 / 102, 189 / 163, 224 / 204;
//   16 of 1500 (128 columns are 16k heads of rows): 128 columns 49 / 55, 48 / 51, 57 / 58; 256 columns 89 / 65, 89 / 91, 105 / 94;
//   64 of 700 (64 columns are 33k): 32 columns 30 / 32, 30 / 38, 34 / 44; 64 columns 51 / 39, 51 / 42, 59 / 50; 96 columns 76 / 45,
//   76 / 62, 88 / 80; 256 of 500: 16 columns 55 / 92, 55 / 63, 60 / 86; 32 columns 92 / 94, 92 / 77, 104 / 102;
// and of 16 K/V heads of 64:
//   1 of 16000: 256 columns 63 / 52, 63 / 63, 73 / 74; 1024 columns 219 / 124, 219 / 190, 262 / 239;
//   16 of 1500: 128 columns 54 / 44, 54 / 58, 62 / 68; 258 columns 109 / 67, 110 / 118, 128 / 146;
//   64 of 700: 32 columns 36 / 40, 36 / 34, 40 / 40; 64 columns 62 / 45, 62 / 42, 70 / 52;
//   8 of 1806 (33k, 20 % of five tiles empty): 258 columns 69 / 60, 70 / 72, 80 / 89.
// The rule knows neither the width nor the number of keys. Of these it takes the slower kernel for 1 of 16000 with 256 columns of width 64 in bf16
// (by 24 %), 16 of 1500 with 128 columns in bf16 (14 %), in f16 and f32 of width 64 (7, 9 %) and with 258 there (7, 15 %), 64 of 700 with 32
// f16 columns of width 64 (8 %); two more are within 3 %.
template <typename T> struct column_rule {
    static constexpr int64_t C = prompt<T>::columns, full = prompt<T>::scaled ? 16000 : 32000, least = 24, many = prompt<T>::scaled ? 256 : 768;
};
template <typename T> int columns_of(const cache_shape & c, int64_t n_seq, int64_t n_rows) {
    typedef column_rule<T> R;
    const int64_t columns = n_rows * (c.n_head / c.n_kv_head), of_tiles = std::max<int64_t>(n_seq, 1) * R::C, with_empty = (columns + of_tiles - 1) / of_tiles * of_tiles;
    const bool prompts = columns > R::many * n_seq || (columns > R::least * n_seq && (double) n_rows * c.n_head * columns > (double) R::full * with_empty);
    return prompts ? (int) R::C : 16;
}
// whether columns_of can be the prompts' for this many rows or fewer, of any number of sequences
template <typename T> bool prompts_within(const cache_shape & c, int64_t n_rows) {
    typedef column_rule<T> R;
    const int64_t columns = n_rows * (c.n_head / c.n_kv_head);
    return columns > R::many || (columns > R::least && n_rows * c.n_head > R::full);
}

// bounds on the column tiles of all sequences, and on the pieces that the ones split into several have
int64_t tiles_bound(const cache_shape & c, int C, int64_t n_seq, int64_t n_rows) { return n_rows * (c.n_head / c.n_kv_head) / C + n_seq; }
// A tile's pieces are keys of its sequence / length rounded, length at least the keys of all tiles and K/V heads over MOST_UNITS
// slots: without the rounding all are that / K/V heads at most, and where there are two or more (1.5 before rounding) it adds a third
// at most. (A half is counted: the device's sums are floats.)
template <typename T> int64_t parts_bound(const cache_shape & c, int C, int64_t n_seq, int64_t n_rows, int64_t width) {
    const int64_t most = (width * c.page_size + piece_min(C) / 2) / piece_min(C), units = (int64_t) (1.5f * MOST_UNITS * slots_of<T>(c.hd, C));
    if (most < 2) return 0;
    static_assert(1.5f * MOST_UNITS * 1024 + 4096 <= COUNTERS, "a counter for each part: units and a round-up to K/V heads, of which there are 4096 at most");
    return std::min(tiles_bound(c, C, n_seq, n_rows) * most, (units + c.n_kv_head - 1) / c.n_kv_head);
}
// (what any call of no more rows, sequences and pages needs: a program asks once, for its largest step)
template <typename T> int64_t work_bytes(const cache_shape & c, int64_t n_seq, int64_t n_rows, int64_t width) {
    auto bytes = [&](int C) { return parts_bound<T>(c, C, n_seq, n_rows, width) * c.n_kv_head * C * (c.hd + 2) * 4; };
    return COUNTERS * 8 + std::max(bytes(16), prompts_within<T>(c, n_rows) ? bytes(prompt<T>::columns) : 0);
}

template <typename T> int64_t blocks_of(const cache_shape & c, int64_t n_seq, int64_t n_rows, int64_t width) {
    const int C = columns_of<T>(c, n_seq, n_rows);
    return (tiles_bound(c, C, n_seq, n_rows) + parts_bound<T>(c, C, n_seq, n_rows, width)) * c.n_kv_head;
}

template <typename T, int HD, int C>
hipError_t attend(const cache_shape & c, const cache_attn_args & a, hipStream_t s, const void * kernel) {
    cache_attn_args args = a;
    void * p[] = {&args};
    const int64_t tiles = tiles_bound(c, C, a.n_seq, a.n_rows), parts = parts_bound<T>(c, C, a.n_seq, a.n_rows, a.width);
    args.parts = parts;
    args.units = (uint32_t) (tiles + parts);
    return hipLaunchKernel(kernel, dim3((unsigned) ((tiles + parts) * c.n_kv_head)), dim3(NT), p, 0, s);
}

template <typename T, int HD>
hipError_t by_columns(const cache_shape & c, const cache_attn_args & a, hipStream_t s) {
    return columns_of<T>(c, a.n_seq, a.n_rows) == 16 ? attend<T, HD, 16>(c, a, s, (const void *) k_cache_attention<T, HD>)
                                                     : attend<T, HD, prompt<T>::columns>(c, a, s, (const void *) k_cache_prompt<T, HD>);
}

template <typename T>
hipError_t by_head(const cache_shape & c, const cache_attn_args & a, hipStream_t s) {
    return c.hd == 32 ? by_columns<T, 32>(c, a, s) : c.hd == 64 ? by_columns<T, 64>(c, a, s) : c.hd == 96 ? by_columns<T, 96>(c, a, s) : by_columns<T, 128>(c, a, s);
}

}  // namespace

int64_t cache_attention_work_bytes(const cache_shape & c, int64_t n_seq, int64_t n_rows, int64_t width) {      // (rows of any type)
    return std::max({work_bytes<float>(c, n_seq, n_rows, width), work_bytes<_Float16>(c, n_seq, n_rows, width), work_bytes<__bf16>(c, n_seq, n_rows, width)});
}

int64_t cache_attention_blocks(const cache_shape & c, int type, int64_t n_seq, int64_t n_rows, int64_t width) {
    return type == T_F32 ? blocks_of<float>(c, n_seq, n_rows, width) : type == T_F16 ? blocks_of<_Float16>(c, n_seq, n_rows, width) : blocks_of<__bf16>(c, n_seq, n_rows, width);
}

hipError_t launch_cache_attention(const cache_shape & c, int type, const cache_attn_args & a, hipStream_t s) {
    return type == T_F32 ? by_head<float>(c, a, s) : type == T_F16 ? by_head<_Float16>(c, a, s) : by_head<__bf16>(c, a, s);
}
