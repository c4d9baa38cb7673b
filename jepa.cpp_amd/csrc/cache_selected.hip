// cache_selected.hip - attention of packed rows over pages that each row and K/V head selects from the 4-bit paged cache.
//
// The arithmetic is k_cache_attention's (scales in f32, weights of one f16 or two, V as two f16) but for two things: 16-bit rows take K's codes as f16 subnormals
// without their offset, which the sum begins with instead (raw8: 64 instructions of a tile's 650 less), and many bf16 rows take V rounded to one f16, as there (64 more). f32
// rows take K as there, for the offset costs the sum two bits. Few bf16 rows keep V's bits, for 2 to 5 % of their time (a call, V as one f16 / as two: one token over 512 of
// 16 heads of 64 6.9 / 7.0 us, 30 requests of 32 heads over 8 of 128 over 1024 tokens each 12.8 / 13.5, 64 of them 19.4 / 20.4). f16 weights of two terms were measured: 14 %
// slower for many rows, 10 % for few, for an error of 2.1e-4 instead of 2.6e-4, of which 2.0e-4 is the output's own rounding.
// A row's columns are the heads that share a K/V head, its keys the tokens of its own pages, so nothing is shared between rows but the caches that hold
// the pages: with the K/V head in the workgroup's low bits an XCD's L2 sees one head of the cache (or a few).
//
// A list is brought in first, without the entries that are no page of the row's (-1, past its last token, not the cache's): pages and places in LDS,
// so that the loop has no such cases, and masks only strips that the row's last token ends.
//   many rows (WHOLE)   a wave has a row and K/V head by itself and writes its result from its registers
//   few rows            the four waves of a workgroup have 64 keys each in turn and join in LDS; fewer still: several workgroups a row, the
//                       last of which joins their sums
// Measured, 32 heads over 4 or 8 of 128: 2000 bf16 rows over 16 pages of 64 each 140 us (1.18 GB from the L2s, 8.4 TB/s; the VALU 76 % of its time, 510 instructions a
// tile of 64 keys; half of the 16 columns are empty with 8 heads), f16 172, f32 207; 64 f16 requests, 64 pages of 16 each, 19.8 us (72 MB, 3.7 TB/s; 5.1 between the first
// tile, 3.4 us after the start by the chain of sequence, list, page numbers and codes, and the tail of 4); one f32 token over 32 pages of 16, 16 heads of 64, 8.1 us, that chain.
#include "cache_attn_dev.h"
#include "common.h"

#include <algorithm>
#include <type_traits>

namespace {

constexpr int C = 16;                     // columns
constexpr int MOST = CACHE_MOST_SELECTED;
constexpr int groups_of(int hd) { return hd > 64 ? 3 : 4; }      // workgroups of a CU

template <int HD> constexpr int split_lds() {
    const int loop = 4 * wave_lds<HD>(), join = 4 * C * (HD + 4) * 4 + 4 * C * 8;
    return loop > join ? loop : join;
}

template <typename T, int HD, bool WHOLE>
__global__ __launch_bounds__(NT, groups_of(HD)) void k_cache_selected(cache_selected_args a) {
    constexpr int NB = HD / 32, ND = HD / 16, TERMS = sizeof(T) == 4 ? 2 : 1, LISTS = WHOLE ? 4 : 1;
    constexpr bool RAW = TERMS == 1, EXACT = !(WHOLE && std::is_same<T, __bf16>::value);
    __shared__ __attribute__((aligned(16))) unsigned char lds[WHOLE ? 4 * wave_lds<HD>() : split_lds<HD>()];
    __shared__ int2_t lists[LISTS][MOST];      // a page of the cache, the token it begins with
    const int tid = (int) threadIdx.x, lane = tid & 63, l15 = lane & 15, g = lane >> 4, wv = uniform(tid >> 6), group = a.n_head / a.n_kv_head;
    const int kvh = (int) (blockIdx.x % (unsigned) a.n_kv_head);
    // the unit: (row, tile of 16 heads, piece of the keys)
    const unsigned at = blockIdx.x / (unsigned) a.n_kv_head;
    const int64_t unit = WHOLE ? (int64_t) at * 4 + wv : at / (unsigned) a.pieces;
    const int piece = WHOLE ? 0 : (int) (at % (unsigned) a.pieces);
    const int64_t row = unit / a.tiles;
    if (row >= a.n_rows) return;      // (WHOLE: of a wave; no barrier follows)
    const int col0 = (int) (unit % a.tiles) * C;
    int seq;
    seq_view v;
    if (!place_of(a, (int32_t) row, seq, v)) return;
    const int32_t lim = cache_visible(v.len - v.rows + (int32_t) (row - v.row0), v.len, a.block);
    const int col = min(col0 + l15, group - 1);
    typename vec8<T>::t y[NB];
    fetch_query<T, HD>((const T *) a.q + row * a.ldq + ((int64_t) kvh * group + col) * HD, g, y);

    // the list
    const int strips_of_page = a.page_size / 16, page_shift = __builtin_ctz((unsigned) strips_of_page), tokens_shift = page_shift + 4;
    int2_t * const list = lists[WHOLE ? wv : 0];
    int n_pages = 0;
    {
        const int32_t * chosen = a.selected + (row * a.n_kv_head + kvh) * a.take, * table = a.table + (int64_t) seq * a.width;
        const int see = (lim + a.page_size - 1) >> tokens_shift;
        int32_t p[MOST / 64], page[MOST / 64];
#pragma unroll
        for (int e = 0; e < MOST / 64; e++) p[e] = e * 64 + lane < a.take ? chosen[e * 64 + lane] : -1;
#pragma unroll
        for (int e = 0; e < MOST / 64; e++) page[e] = p[e] >= 0 && p[e] < see ? table[p[e]] : -1;
#pragma unroll
        for (int e = 0; e < MOST / 64; e++) {
            const bool ok = page[e] >= 0 && page[e] < a.n_pages;
            const uint64_t in = __ballot(ok);
            if (ok && (WHOLE || wv == 0)) list[n_pages + (int) __popcll(in & ((1ull << lane) - 1))] = int2_t{page[e], p[e] << tokens_shift};
            n_pages += (int) __popcll(in);
        }
        n_pages = uniform(n_pages);
        if constexpr (WHOLE) wave_order();
        else __syncthreads();
    }

    // this wave's tiles of 4 strips
    const int n_strips = n_pages << page_shift, last_strip = n_strips - 1, n_tiles = (n_strips + 3) / 4;
    constexpr int STEP = WHOLE ? 1 : 4;
    int tile_at = WHOLE ? 0 : piece * a.piece_tiles + wv;
    const int tile_end = WHOLE ? n_tiles : min(n_tiles, (piece + 1) * a.piece_tiles);
    // strips in lanes 0 to 3: their page, and how many of their tokens are read
    auto load_pages = [&](int t) {
        const int strip = t * 4 + (lane & 3), in = min(strip, max(last_strip, 0));
        const int2_t x = list[in >> page_shift];
        const int left = lim - (x[1] + (in & (strips_of_page - 1)) * 16);
        return int2_t{x[0], strip > last_strip ? 0 : min(max(left, 0), 16)};
    };
    uint32_t kn[4][NB], vn[4][NB], sn[4];
    int2_t pages = {0, 0}, cur = {0, 0};      // of the next tile, and of the one in flight
    brsrc strips[4];
    auto load_v = [&](int t, int2_t pages) {
#pragma unroll
        for (int s = 0; s < 4; s++) {
            const int strip = min(t * 4 + s, last_strip);
            const int64_t page = __builtin_amdgcn_readlane(pages[0], s);
            strips[s] = make_brsrc(a.cache + ((page * a.n_kv_head + kvh) * strips_of_page + (strip & (strips_of_page - 1))) * (18 * HD), t < tile_end ? 18 * HD : 0);
            load_words<NB>(vn[s], strips[s], lane * (4 * NB), 8 * HD);
            load_words<1>(&sn[s], strips[s], 16 * HD + lane * 4, 0);      // (0 past the strip's scales, from lane HD / 2 on)
        }
    };
    auto load_k = [&] {
#pragma unroll
        for (int s = 0; s < 4; s++) load_words<NB>(kn[s], strips[s], lane * (4 * NB), 0);
    };
    unsigned char * const mine = lds + wv * wave_lds<HD>();
    unsigned char * const scales = mine + ND * 528;
    const int e = (l15 & 3) * 2 + ((l15 & 7) >> 2);
    const int tr_at = (((l15 >> 3) * 2 + (e >> 2)) * 16 + g * 4 + (e & 3)) * 8;
    if (tile_at < tile_end) {
        cur = load_pages(tile_at);
        load_v(tile_at, cur);
        load_k();
        pages = load_pages(tile_at + STEP);
    }
    float c;
    half8_t q[NB][TERMS];
    turn_query<T, HD, TERMS>(a.scale, y, q, c);
    float offset[NB];      // what the product with the raw codes of a block begins with
    if constexpr (RAW) {
#pragma unroll
        for (int b = 0; b < NB; b++) {
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (j & 2) q[b][0][j] *= (_Float16) 0.0625f;
                sum = __builtin_fmaf((float) q[b][0][j], j & 2 ? 16.0f : 1.0f, sum);
            }
            offset[b] = col_sum(sum) * -0x1p-21f;
        }
    }
    // (held where scores times it stay finite for the largest queries of f32 and bf16: there all weight is on the largest scores, of c as of this)
    c = RAW ? fminf(c * 0x1p24f, 0x1p100f) : fminf(c, 0x1p76f);
    float4_t o[ND + 1];
    float mu = -INFINITY;
    for (int d = 0; d <= ND; d++) o[d] = float4_t{0, 0, 0, 0};
    uint32_t k1024 = 0x64006400u;
    asm volatile("" : "+v"(k1024));
    // one tile: MASKED where a strip is not read to its end
    auto tile = [&](auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        int read[4];
#pragma unroll
        for (int t = 0; t < 4; t++) read[t] = MASKED ? __builtin_amdgcn_readlane(cur[1], t) : 16;
        wave_order();
#pragma unroll
        for (int t = 0; t < 4; t++) {
            uint32_t sc = sn[t];
            if constexpr (MASKED) {      // scales of tokens that nobody reads are 0: what lies there does not matter
                const int d = lane % (HD / 4), token = d / (2 * NB) * 4 + (d & 1) * 2;
                if (token >= read[t]) sc = 0;
                else if (token + 1 >= read[t]) sc &= 0xffffu;
            }
            if (lane < HD / 2) *(uint32_t *) (scales + t * 2 * HD + lane * 4) = sc;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const int w = (lane & 3) * NB + b;
                *(uint32_t *) (mine + (w >> 1) * 528 + (t * 16 + (lane >> 2)) * 8 + (w & 1) * 4) = vn[t][b];
            }
        }
        const int2_t after = load_pages(tile_at + 2 * STEP);
        load_v(tile_at + STEP, pages);
        wave_order();
        float4_t s[4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const half4_t * dk = (const half4_t *) (scales + t * 2 * HD + g * (8 * NB));
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const half8_t kc = RAW ? raw8(kn[t][b]) : codes8(kn[t][b], k1024);
                const half4_t d = dk[b];
                const float z = RAW ? offset[b] : 0.0f;
                float4_t x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, q[b][0], float4_t{z, z, z, z}, 0, 0, 0);
                if constexpr (TERMS == 2) x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, q[b][1], x, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; r++) s[t][r] = __builtin_fmaf((float) d[r], x[r], b == 0 ? 0.0f : s[t][r]);
            }
            if constexpr (MASKED) {
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (g * 4 + r >= read[t]) s[t][r] = -INFINITY;
            }
            __builtin_amdgcn_sched_barrier(0x100);
        }
        load_k();
        cur = pages;
        pages = after;
        softmax_weights<MASKED, ND>(s, c, mu, o);
        half8_t p[2][TERMS];
#pragma unroll
        for (int h = 0; h < 2; h++) turn_weights<TERMS>(s, h, p[h], o[ND]);
#pragma unroll
        for (int b = 0; b < NB; b++) {
#pragma unroll
            for (int dd = 0; dd < 2; dd++) {
                const int d = 2 * b + dd;
                const int2_t w = __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) int2_t *) (mine + d * 528 + tr_at));
#pragma unroll
                for (int h = 0; h < 2; h++)
                    o[d] = add_values<TERMS, EXACT>(codes8((uint32_t) w[h], k1024), scales + HD + g * (8 * NB) + b * 8 + 2 * h * (2 * HD), 2 * HD, p[h], o[d]);
            }
            __builtin_amdgcn_sched_barrier(0x100);
        }
    };
    // (in a list as _cache_select makes it, the last page alone ends before its last token)
    for (; tile_at < tile_end && __all(cur[1] == 16); tile_at += STEP) tile(std::false_type{});
    for (; tile_at < tile_end; tile_at += STEP) tile(std::true_type{});

    auto out_at = [&](int col) { return (T *) a.out + row * a.ldo + ((int64_t) kvh * group + col) * HD; };
    if constexpr (WHOLE) {
        if (col0 + l15 >= group) return;
        const float l = o[ND][0], inv = l == 0.0f ? 0.0f : 1.0f / l;
        T * p = out_at(col0 + l15);
#pragma unroll
        for (int d = 0; d < ND; d++) store4(p + d * 16 + g * 4, o[d] * inv);
    } else {
        // the four waves' sums at the largest of their maxima
        float * const stat = (float *) (lds + 4 * C * (HD + 4) * 4), * const sum = (float *) lds;
        const parts_view<HD, C> part(a.work, a.parts, a.n_kv_head, unit * a.pieces, kvh);
        __syncthreads();      // the loop's LDS is read out
        if (g == 0) {
            stat[(wv * C + l15) * 2] = mu;
            stat[(wv * C + l15) * 2 + 1] = o[ND][0];
        }
#pragma unroll
        for (int d = 0; d < ND; d++) *(float4_t *) (sum + (wv * C + l15) * (HD + 4) + d * 16 + g * 4) = o[d];
        __syncthreads();
        for (int i = tid; i < C * (HD / 4); i += NT) {
            const int of = i / (HD / 4), n = i % (HD / 4) * 4;
            if (col0 + of >= group) break;
            float top = -INFINITY, all = 0.0f;
            for (int w = 0; w < 4; w++) top = fmaxf(top, stat[(w * C + of) * 2]);
            const float m = top == -INFINITY ? 0.0f : top;
            float4_t x = {0, 0, 0, 0};
            for (int w = 0; w < 4; w++) {
                const float f = __builtin_amdgcn_exp2f(stat[(w * C + of) * 2] - m);
                all += stat[(w * C + of) * 2 + 1] * f;
                x += *(const float4_t *) (sum + (w * C + of) * (HD + 4) + n) * f;
            }
            if (a.pieces > 1) {
                if (n == 0) part.put_stat(piece, of, top, all);
                part.put(piece, of, n, x);
            } else {
                store4(out_at(col0 + of) + n, x * (all == 0.0f ? 0.0f : 1.0f / all));
            }
        }
        if (a.pieces > 1 && last_to_arrive(a.work, unit * a.n_kv_head + kvh, a.pieces))
            join_pieces<T>(part, a.pieces, group - col0, [&](int at) { return out_at(col0 + at); });
    }
}

// A wave for each unit where there are two for each SIMD; else a workgroup, or as many as there are CUs, if each has a step of its waves to do. Measured, us of
// a call with a workgroup / a wave a unit: f16 rows of 32 heads over 8 of 128, 1024 tokens each, 512 units 21.4 / 37.1, 1024 36.2 / 37.7, 1536 49.0 / 52.4,
// 2048 60.5 / 58.1, 4096 110 / 105; bf16 rows of 16 heads of 64, 512 tokens each (a workgroup with V as two f16, a wave as one), 512 units 9.7 / 13.9, 1024 14.3 / 14.3,
// 1536 19.7 / 18.2, 2040 24.2 / 18.9. The rows are those that the call is sized for: a token of 63 f16 requests, 32 heads over 8 of 128, 1024 tokens each, 20.3, in a call of
// 2000 rows 35.9.
// Pieces of 240 units into 480 or 720 workgroups 16.2, whole 14.5; of 128 units (2048 tokens each) whole 21.2, 256 workgroups 15.9, 512 15.8, 768 16.0.
constexpr int64_t WAVE_UNITS = 2048, SLOTS = 256;
int64_t steps_of(const cache_shape & c, int take) { return ((int64_t) take * c.page_size + 4 * TILE - 1) / (4 * TILE); }
struct split { int tiles; bool whole; int pieces, piece_tiles; };
split split_of(const cache_shape & c, int64_t n_rows, int take) {
    split s;
    s.tiles = (c.n_head / c.n_kv_head + C - 1) / C;
    const int64_t units = n_rows * s.tiles * c.n_kv_head, steps = steps_of(c, take);
    s.whole = units >= WAVE_UNITS;
    s.pieces = s.whole ? 1 : (int) std::clamp<int64_t>(SLOTS / std::max<int64_t>(units, 1), 1, steps);
    const int64_t each = (steps + s.pieces - 1) / s.pieces;
    s.piece_tiles = (int) each * 4;
    s.pieces = (int) ((steps + each - 1) / each);
    return s;
}

template <typename T, int HD>
hipError_t selected(const cache_shape & c, const cache_selected_args & a, hipStream_t s) {
    cache_selected_args args = a;
    void * p[] = {&args};
    const split f = split_of(c, a.n_rows, a.take);
    args.tiles = f.tiles;
    args.pieces = f.pieces;
    args.piece_tiles = f.piece_tiles;
    args.parts = a.n_rows * f.tiles * f.pieces;
    return hipLaunchKernel(f.whole ? (const void *) k_cache_selected<T, HD, true> : (const void *) k_cache_selected<T, HD, false>,
                           dim3((unsigned) cache_selected_blocks(c, a.n_rows, a.take)), dim3(NT), p, 0, s);
}

template <typename T>
hipError_t by_head(const cache_shape & c, const cache_selected_args & a, hipStream_t s) {
    return c.hd == 32 ? selected<T, 32>(c, a, s) : c.hd == 64 ? selected<T, 64>(c, a, s) : c.hd == 96 ? selected<T, 96>(c, a, s) : selected<T, 128>(c, a, s);
}

}  // namespace

int64_t cache_selected_blocks(const cache_shape & c, int64_t n_rows, int take) {
    const split f = split_of(c, n_rows, take);
    const int64_t units = n_rows * f.tiles;
    return (f.whole ? (units + 3) / 4 : units * f.pieces) * c.n_kv_head;
}

// What any call of no more rows and pages needs: of units in several pieces there are half the slots or fewer, and no more pieces than slots
int64_t cache_selected_work_bytes(const cache_shape & c, int64_t n_rows, int take) {
    static_assert(SLOTS <= COUNTERS, "a counter for each unit of several pieces");
    const int64_t units = n_rows * ((c.n_head / c.n_kv_head + C - 1) / C) * c.n_kv_head, steps = steps_of(c, take);
    return steps > 1 ? COUNTERS * 8 + std::min(units * steps, SLOTS) * C * (c.hd + 2) * 4 : 0;
}

hipError_t launch_cache_selected(const cache_shape & c, int type, const cache_selected_args & a, hipStream_t s) {
    return type == T_F32 ? by_head<float>(c, a, s) : type == T_F16 ? by_head<_Float16>(c, a, s) : by_head<__bf16>(c, a, s);
}
