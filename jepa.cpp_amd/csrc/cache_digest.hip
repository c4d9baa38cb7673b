// cache_digest.hip - the digests of the cache's pages: what box the keys of a page and K/V head lie in.
//
//   hi_n = max_t k_tn, lo_n = min_t k_tn over the page's tokens t (none that is NaN), s = max_n max(|hi_n|, |lo_n|)
//   codes rint(hi_n * fl(127 / s)), rint(lo_n * fl(127 / s)), scale fl(s / 127); all zero where s is below 2^-100
//
// A wave has one page and K/V head. Its lanes read K's codes as the attention does (lane 16 g + token: dims 32 b + 8 g .. + 7 of
// every block b), multiply them by the token's scale (f32, exact: 4 bits times 11), keep the largest and smallest over the strips and join the 16 tokens' lanes.
#include "cache_attn_dev.h"
#include "common.h"

#include <algorithm>

namespace {

constexpr float LEAST = 0x1p-100f;

template <int HD>
__global__ __launch_bounds__(NT) void k_cache_digest(cache_digest_args a) {
    constexpr int NB = HD / 32, WORDS = 2 * HD / 4;      // of codes
    __shared__ __attribute__((aligned(16))) float box[4][2 * HD];
    const int tid = (int) threadIdx.x, lane = tid & 63, l15 = lane & 15, g = lane >> 4, wv = uniform(tid >> 6), kvh = (int) (blockIdx.x % (unsigned) a.n_kv_head);
    const int64_t r0 = (int64_t) (blockIdx.x / (unsigned) a.n_kv_head) * a.rows_per, r1 = min(r0 + a.rows_per, a.n_rows);
    const int page_shift = __builtin_ctz((unsigned) a.page_size), strips_of_page = a.page_size / 16;
    int at = 0;      // pages of the workgroup so far, dealt to its waves
    for (int64_t r = r0; r < r1;) {
        const int i = seq_of_row(a.row_start, a.n_seq, (int32_t) r);
        if (i < 0) {      // before the first sequence, or behind the last
            if (r >= a.row_start[0]) break;
            r = min((int64_t) a.row_start[0], r1);
            continue;
        }
        const seq_view v = view_of(a, i);
        const int64_t end = min(r1, (int64_t) v.row0 + v.rows);
        if (end <= r) { r++; continue; }      // (row_start that does not ascend)
        // the pages that begin within these rows, and the sequence's first
        const int64_t pos = (int64_t) v.len - v.rows + (r - v.row0), pos_end = pos + (end - r);
        auto page_from = [&](int64_t t) { return (int32_t) (((t < 0 ? 0 : t) + a.page_size - 1) >> page_shift); };      // the first one that begins at t or later
        const int32_t p0 = r == v.row0 ? (int32_t) ((pos < 0 ? 0 : pos) >> page_shift) : page_from(pos), p1 = page_from(pos_end);
        for (int32_t p = p0; p < p1; p++) {
            if ((at++ & 3) != wv) continue;
            const int64_t page = uniform(a.table[(int64_t) i * a.width + p]);
            if (page < 0 || page >= a.n_pages) continue;
            const int tokens = min(a.page_size, v.len - (p << page_shift));
            float hi[NB * 8], lo[NB * 8];
#pragma unroll
            for (int j = 0; j < NB * 8; j++) { hi[j] = -INFINITY; lo[j] = INFINITY; }
            uint32_t k1024 = 0x64006400u;
            asm volatile("" : "+v"(k1024));
            for (int t = 0; t * 16 < tokens; t++) {
                const brsrc s = make_brsrc(a.cache + ((page * a.n_kv_head + kvh) * strips_of_page + t) * (18 * HD), 18 * HD);
                uint32_t w[NB];
                load_words<NB>(w, s, lane * (4 * NB), 0);
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const uint32_t d = __builtin_amdgcn_raw_buffer_load_b16(s, cache_k_scale(l15, b, HD), 0, 0);
                    const float scale = t * 16 + l15 < tokens ? (float) __builtin_bit_cast(_Float16, (uint16_t) d) : __builtin_nanf("");      // (no number: not counted)
                    const half8_t c = codes8(w[b], k1024);
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const float x = (float) c[j] * scale;
                        hi[b * 8 + j] = fmaxf(hi[b * 8 + j], x);
                        lo[b * 8 + j] = fminf(lo[b * 8 + j], x);
                    }
                }
            }
            float top = 0.0f;
#pragma unroll
            for (int j = 0; j < NB * 8; j++) {
                const float h = row_max16(hi[j]), l = -row_max16(-lo[j]);
                hi[j] = h == -INFINITY ? 0.0f : h;
                lo[j] = l == INFINITY ? 0.0f : l;
                top = fmaxf(top, fmaxf(fabsf(hi[j]), fabsf(lo[j])));
            }
            top = col_max(top);
            const float inv = top >= LEAST ? 127.0f / top : 0.0f, scale = top >= LEAST ? top / 127.0f : 0.0f;
            if (l15 == 0) {
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        box[wv][b * 32 + g * 8 + j] = hi[b * 8 + j];
                        box[wv][HD + b * 32 + g * 8 + j] = lo[b * 8 + j];
                    }
            }
            wave_order();
            unsigned char * out = a.digest + (page * a.n_kv_head + kvh) * cache_digest_bytes(HD);
            if (lane < WORDS) {
                const float4_t x = *(const float4_t *) &box[wv][lane * 4];
                uint32_t word = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) word |= ((uint32_t) (int) rintf(x[j] * inv) & 255u) << (8 * j);
                *(uint32_t *) (out + lane * 4) = word;
            }
            if (lane < 4) *(uint32_t *) (out + 2 * HD + lane * 4) = lane == 0 ? __float_as_uint(scale) : 0u;
            wave_order();
        }
        r = end;
    }
}

// the bounds [n][n_kv_head][2][HD] of pages; zeros for a page that is none
__global__ __launch_bounds__(NT) void k_cache_digest_read(const unsigned char * digest, const int32_t * pages, int64_t n, int64_t n_pages, int n_kv_head, int hd, float * bounds) {
    const int64_t words = n * n_kv_head * (hd / 2), at = (int64_t) blockIdx.x * NT + threadIdx.x;
    if (at >= words) return;
    const int64_t of = at / (hd / 2);      // (page, head)
    const int w = (int) (at % (hd / 2));
    const int64_t page = pages[of / n_kv_head];
    float4_t x = {0, 0, 0, 0};
    if (page >= 0 && page < n_pages) {
        const unsigned char * d = digest + (page * n_kv_head + of % n_kv_head) * cache_digest_bytes(hd);
        const int32_t word = *(const int32_t *) (d + w * 4);
        const float scale = *(const float *) (d + 2 * hd);
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = (float) (word << (24 - 8 * j) >> 24) * scale;
    }
    *(float4_t *) (bounds + at * 4) = x;
}

}  // namespace

// A workgroup has some consecutive rows: one where sequences get a row or so each, up to a page of a prompt's
static int rows_per_of(int page_size, int64_t n_seq, int64_t n_rows) {
    int n = 1;
    while (n < page_size && 2 * n * n_seq <= n_rows) n *= 2;
    return n;
}
int64_t cache_digest_blocks(const cache_shape & c, int64_t n_seq, int64_t n_rows) {
    const int n = rows_per_of(c.page_size, n_seq, n_rows);
    return (n_rows + n - 1) / n * c.n_kv_head;
}
hipError_t launch_cache_digest(const cache_digest_args & a, int hd, hipStream_t s) {
    cache_digest_args args = a;
    args.rows_per = rows_per_of(a.page_size, a.n_seq, a.n_rows);
    void * p[] = {&args};
    const void * k = hd == 32 ? (const void *) k_cache_digest<32> : hd == 64 ? (const void *) k_cache_digest<64> : hd == 96 ? (const void *) k_cache_digest<96> : (const void *) k_cache_digest<128>;
    return hipLaunchKernel(k, dim3((unsigned) ((a.n_rows + args.rows_per - 1) / args.rows_per * a.n_kv_head)), dim3(NT), p, 0, s);
}

hipError_t launch_cache_digest_read(const unsigned char * digest, const int32_t * page, int64_t n, int64_t n_pages, int n_kv_head, int hd, float * bounds, hipStream_t s) {
    void * p[] = {&digest, &page, &n, &n_pages, &n_kv_head, &hd, &bounds};
    return hipLaunchKernel((const void *) k_cache_digest_read, dim3((unsigned) ((n * n_kv_head * (hd / 2) + NT - 1) / NT)), dim3(NT), p, 0, s);
}
