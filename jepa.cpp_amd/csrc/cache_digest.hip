// cache_digest.hip - the digests of the cache's pages: what box the keys of a page and K/V head lie in.
//
//   hi_n = max_t k_tn, lo_n = min_t k_tn over the page's tokens t (none that is NaN), s = max_n max(|hi_n|, |lo_n|)
//   codes rint(hi_n * fl(127 / s)), rint(lo_n * fl(127 / s)), scale fl(s / 127); all zero where s is below 2^-100
//
// A wave has one K/V head of the pages that some rows lie in, mostly one. A lane takes 8 dimensions (a word of codes) of a few tokens of each strip, so that
// most of the largest and smallest are found in its registers and the few lanes of the same dimensions are joined by DPP. AHEAD strips, up to four of a page, are
// in flight (all four for pages of one strip were 35 us for 41000 tokens of 8 x 128, one was 21).
//
// Measured: 41000 prompt tokens of 8 x 128 in pages of 16, 18.2 us: the VALU's instructions, 380 for each of 20.9 thousand waves, are 13 us of every SIMD's time. A wave is ready and
// waits to issue for 45 % of its life, waits for memory for 30 % of it, and 4.6 are on a SIMD on average. A third of the instructions lie before and behind the tokens, but several pages
// or heads a wave, which share them, took no less (two pages 18.3, four 19.2, two heads 21.6 instead of 21.7 then); why not is not known. One token of 64 requests in pages of 64,
// 4.8 us: one chain of loads.
#include "cache_attn_dev.h"
#include "common.h"

#include <algorithm>

namespace {

constexpr float LEAST = 0x1p-100f;

// The largest over aligned groups of N lanes (pairs, quads, halves of 16 mirrored, 16 mirrored) of eight values that are no NaN, in place. In one block, for
// the compiler would make each of them canonical first: a DPP operand has to be two instructions old, which the others of the eight see to.
#define STEP(how)                                                                                                                                                       \
    asm volatile("s_nop 1\n\tv_max_f32_dpp %0, %0, %0 " how "\n\tv_max_f32_dpp %1, %1, %1 " how "\n\tv_max_f32_dpp %2, %2, %2 " how "\n\tv_max_f32_dpp %3, %3, %3 " how  \
                 "\n\tv_max_f32_dpp %4, %4, %4 " how "\n\tv_max_f32_dpp %5, %5, %5 " how "\n\tv_max_f32_dpp %6, %6, %6 " how "\n\tv_max_f32_dpp %7, %7, %7 " how "\n\ts_nop 1"  \
                 : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]), "+v"(x[4]), "+v"(x[5]), "+v"(x[6]), "+v"(x[7]))
template <int N>
__device__ __forceinline__ void max_of(float * x) {
    STEP("quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf");
    STEP("quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf");
    if constexpr (N >= 8) STEP("row_half_mirror row_mask:0xf bank_mask:0xf");
    if constexpr (N >= 16) STEP("row_mirror row_mask:0xf bank_mask:0xf");
}
#undef STEP

// rint of four values of magnitude 127 at most, as bytes: what an addition of 1.5 * 2^23 leaves in the lowest bits
__device__ __forceinline__ uint32_t bytes_of(const float * x) {
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; j++) u[j] = __float_as_uint(x[j] + 0x1.8p23f);
    const uint32_t lo = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(u[3], u[2], 0x04000c0cu);
    return lo | hi;
}

template <int HD, int AHEAD>
__global__ __launch_bounds__(NT) void k_cache_digest(cache_digest_args a) {
    // lanes of the same dimensions, tokens of each: 64 lanes are 4 NB words of codes (of 8 dimensions) times TL (48 of 64 for three blocks)
    constexpr int NB = HD / 32, TL = HD == 32 ? 16 : HD == 64 ? 8 : 4, TOKENS = 16 / TL;
    const int lane = (int) threadIdx.x & 63, tl = lane % TL, word = min(lane / TL, 4 * NB - 1), g = word / NB, b = word % NB;
    const uint32_t unit = blockIdx.x * 4 + (uint32_t) uniform((int) threadIdx.x >> 6);      // (below 2^26)
    const int kvh = (int) (unit % (uint32_t) a.n_kv_head);
    const int64_t r0 = (int64_t) (unit / (uint32_t) a.n_kv_head) * a.rows_per, r1 = min(r0 + a.rows_per, a.n_rows);
    const int page_shift = __builtin_ctz((unsigned) a.page_size), strips_of_page = a.page_size / 16;
    uint32_t k1024 = 0x64006400u;
    asm volatile("" : "+v"(k1024));
    for (int64_t r = r0; r < r1;) {
        int i;
        seq_view v;
        if (!place_of(a, (int32_t) r, i, v)) {      // before the first sequence, or behind the last
            if (r >= a.row_start[0]) break;
            r = min((int64_t) a.row_start[0], r1);
            continue;
        }
        const int64_t end = min(r1, (int64_t) v.row0 + v.rows);
        // the pages that begin within these rows, and the sequence's first
        const int64_t pos = (int64_t) v.len - v.rows + (r - v.row0), pos_end = pos + (end - r);
        auto page_from = [&](int64_t t) { return (int32_t) (((t < 0 ? 0 : t) + a.page_size - 1) >> page_shift); };      // the first one that begins at t or later
        const int32_t p0 = r == v.row0 ? (int32_t) ((pos < 0 ? 0 : pos) >> page_shift) : page_from(pos), p1 = page_from(pos_end);
        for (int32_t p = p0; p < p1; p++) {
            const int64_t page = uniform(a.table[(int64_t) i * a.width + p]);
            if (page < 0 || page >= a.n_pages) continue;
            const int tokens = min(a.page_size, v.len - (p << page_shift));
            const unsigned char * strips = a.cache + (page * a.n_kv_head + kvh) * strips_of_page * (18 * HD);
            float hi[8], lo[8];      // the largest value, and the largest of the values' negatives
#pragma unroll
            for (int j = 0; j < 8; j++) hi[j] = lo[j] = -INFINITY;
            for (int t0 = 0; t0 * 16 < tokens; t0 += AHEAD) {
                uint32_t w[AHEAD][TOKENS], d[AHEAD][(TOKENS + 1) / 2];
#pragma unroll
                for (int t = 0; t < AHEAD; t++) {
                    const brsrc s = make_brsrc(strips + (t0 + t) * (18 * HD), (t0 + t) * 16 < tokens ? 18 * HD : 0);
#pragma unroll
                    for (int k = 0; k < TOKENS; k++) w[t][k] = __builtin_amdgcn_raw_buffer_load_b32(s, cache_k_word(tl * TOKENS + k, g, b, HD), 0, 0);
                    if constexpr (TOKENS == 1) d[t][0] = __builtin_amdgcn_raw_buffer_load_b16(s, cache_k_scale(tl, b, HD), 0, 0);
                    else load_words<TOKENS / 2>(d[t], s, cache_k_scale(tl * TOKENS, b, HD), 0);      // (of consecutive tokens of four)
                }
#pragma unroll
                for (int t = 0; t < AHEAD; t++) {
#pragma unroll
                    for (int k = 0; k < TOKENS; k++) {
                        const uint16_t bits = (uint16_t) (d[t][k / 2] >> (16 * (k & 1)));
                        const float scale = (t0 + t) * 16 + tl * TOKENS + k < tokens ? (float) __builtin_bit_cast(_Float16, bits) : __builtin_nanf("");      // (no number: not counted)
                        const half8_t c = codes8(w[t][k], k1024);
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const float x = __builtin_fmaf((float) c[j], scale, 0.0f);      // (takes the f16 as it is)
                            hi[j] = fmaxf(hi[j], x);
                            lo[j] = fmaxf(lo[j], -x);
                        }
                    }
                }
            }
            max_of<TL>(hi);
            max_of<TL>(lo);
            if (__any(hi[0] == -INFINITY)) {      // no token of this block of the head is a number
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (hi[j] == -INFINITY) hi[j] = lo[j] = 0.0f;
            }
            float top = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) top = fmaxf(top, fmaxf(fabsf(hi[j]), fabsf(lo[j])));
            top = col_max(row_max16(top));
            const float inv = top >= LEAST ? 127.0f / top : 0.0f, scale = top >= LEAST ? top / 127.0f : 0.0f;
            // the first lane of the same dimensions writes the largest, the second the smallest
            unsigned char * out = a.digest + (page * a.n_kv_head + kvh) * cache_digest_bytes(HD);
            float x[8];
            const float by = tl == 0 ? inv : -inv;
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = (tl == 0 ? hi[j] : lo[j]) * by;
            const word2_t codes = {bytes_of(x), bytes_of(x + 4)};
            if (tl < 2 && lane < 4 * NB * TL) *(word2_t *) (out + tl * HD + 32 * b + 8 * g) = codes;
            if (lane < 4) *(uint32_t *) (out + 2 * HD + lane * 4) = lane == 0 ? __float_as_uint(scale) : 0u;
        }
        r = end;
    }
}

// the bounds [n][n_kv_head][2][HD] of pages; zeros for a page that is none
__global__ __launch_bounds__(NT) void k_cache_digest_read(const unsigned char * digest, const int32_t * pages, int64_t n, int64_t n_pages, int n_kv_head, int hd, float * bounds) {
    const uint32_t words = (uint32_t) hd / 2, at = blockIdx.x * NT + threadIdx.x, of = at / words, w = at % words, i = of / (uint32_t) n_kv_head;      // (words of a page and head)
    if (i >= n) return;
    const int64_t page = pages[i];
    float4_t x = {0, 0, 0, 0};
    if (page >= 0 && page < n_pages) {
        const unsigned char * d = digest + (page * n_kv_head + of % (uint32_t) n_kv_head) * cache_digest_bytes(hd);
        const int32_t word = *(const int32_t *) (d + w * 4);
        const float scale = *(const float *) (d + 2 * hd);
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = (float) (word << (24 - 8 * j) >> 24) * scale;
    }
    *(float4_t *) (bounds + (int64_t) at * 4) = x;
}

}  // namespace

// A wave has some consecutive rows: one where sequences get a row or so each, up to a page of a prompt's. That goes by the mean of what the call is sized for: single tokens
// beside a prompt, or in a captured call with room for one, share a wave, which takes their sequences one after the other (a token of 63 requests in pages of 16 3.2 us, in a
// call of 2000 rows or beside a prompt of 1000 24.5).
static int rows_per_of(int page_size, int64_t n_seq, int64_t n_rows) {
    int n = 1;
    while (n < page_size && 2 * n * n_seq <= n_rows) n *= 2;
    return n;
}
int64_t cache_digest_blocks(const cache_shape & c, int64_t n_seq, int64_t n_rows) {
    const int n = rows_per_of(c.page_size, n_seq, n_rows);
    return ((n_rows + n - 1) / n * c.n_kv_head + 3) / 4;
}
hipError_t launch_cache_digest(const cache_shape & c, const cache_digest_args & a, hipStream_t s) {
    cache_digest_args args = a;
    args.rows_per = rows_per_of(a.page_size, a.n_seq, a.n_rows);
    void * p[] = {&args};
#define OF(HD) (c.page_size == 16 ? (const void *) k_cache_digest<HD, 1> : c.page_size == 32 ? (const void *) k_cache_digest<HD, 2> : (const void *) k_cache_digest<HD, 4>)
    const void * k = c.hd == 32 ? OF(32) : c.hd == 64 ? OF(64) : c.hd == 96 ? OF(96) : OF(128);
#undef OF
    return hipLaunchKernel(k, dim3((unsigned) cache_digest_blocks(c, a.n_seq, a.n_rows)), dim3(NT), p, 0, s);
}

hipError_t launch_cache_digest_read(const unsigned char * digest, const int32_t * page, int64_t n, int64_t n_pages, int n_kv_head, int hd, float * bounds, hipStream_t s) {
    void * p[] = {&digest, &page, &n, &n_pages, &n_kv_head, &hd, &bounds};
    return hipLaunchKernel((const void *) k_cache_digest_read, dim3((unsigned) ((n * n_kv_head * (hd / 2) + NT - 1) / NT)), dim3(NT), p, 0, s);
}
