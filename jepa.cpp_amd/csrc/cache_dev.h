// cache_dev.h - the 4-bit paged key/value cache: where its bytes lie, and how lengths map to pages.
//
// A page holds page_size tokens of every K/V head, as [kv head][strip of 16 tokens]. A strip of one head is
// 18 * hd bytes; with NB = hd / 32 ggml q4_0 blocks per row (value = (code - 8) * d, d an f16):
//   K codes  [4 g][16 tokens][NB words]: word (g, token, b) is dims 32 b + 8 g .. + 7, which is what lane
//            16 g + token of the QK MFMA (A operand, 16 keys x 32 dims) reads of block b, so a wave reads the
//            codes of 16 keys as one contiguous piece. Nibble n of the word is element (n % 4) * 2 + n / 4:
//            two nibbles 16 bits apart are one register of two f16 after a mask, an or and an add.
//   V codes  [16 tokens][hd / 2 bytes], dims in order: LDS reads them transposed, 4 bits a lane.
//   scales   f16 [4 tokens / 4][NB][4 tokens % 4] of K, then of V: the accumulator of 16 keys x 16 queries
//            has 4 consecutive keys in a lane, whose scales of one block are 8 bytes.
// Everything is a multiple of 16 bytes, and a strip's address does not depend on the page size.
#pragma once
#include <cstdint>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define CACHE_HD __host__ __device__ __forceinline__
#else
#define CACHE_HD inline
#endif

constexpr int CACHE_STRIP = 16;              // tokens of a strip
constexpr int CACHE_MAX_SEQ = 4096;          // sequences of one step (the planner's LDS)

CACHE_HD int64_t cache_strip_bytes(int hd) { return 18 * (int64_t) hd; }
CACHE_HD int64_t cache_page_bytes(int n_kv_head, int page_size, int hd) { return (int64_t) n_kv_head * (page_size / CACHE_STRIP) * cache_strip_bytes(hd); }
// byte offset of the strip of token `in_page` of a page
CACHE_HD int64_t cache_strip_at(int64_t page, int head, int in_page, int n_kv_head, int page_size, int hd) {
    return ((page * n_kv_head + head) * (page_size / CACHE_STRIP) + in_page / CACHE_STRIP) * cache_strip_bytes(hd);
}
// offsets in a strip: the K word (token, g, b), the V word of dims 8 t .. 8 t + 7, the K scale (token, b)
CACHE_HD int cache_k_word(int token, int g, int b, int hd) { return ((g * 16 + token) * (hd / 32) + b) * 4; }
CACHE_HD int cache_v_word(int token, int t, int hd) { return 8 * hd + token * (hd / 2) + t * 4; }
CACHE_HD int cache_k_scale(int token, int b, int hd) { return 16 * hd + 2 * ((token / 4 * (hd / 32) + b) * 4 + token % 4); }
CACHE_HD int cache_v_scale(int token, int b, int hd) { return cache_k_scale(token, b, hd) + hd; }

// What a step does to one sequence: `have` tokens are cached, `come` > 0 tokens are added or -come dropped.
struct cache_seq_step {
    uint32_t rows, need, give;     // rows in the step's packed arrays; pages taken, pages given back
    int32_t held, len;             // pages and tokens before (held) and after (len), if it is admitted
    bool bad;                      // lengths that the table cannot hold: refused whatever the pool has
};
CACHE_HD cache_seq_step cache_step_of(int32_t have, int32_t come, int32_t width, int32_t page_size) {
    cache_seq_step s;
    const int64_t cap = (int64_t) width * page_size;
    const int64_t keep = (int64_t) have + come > 0 ? (int64_t) have + come : 0;
    const int shift = __builtin_ctz((unsigned) page_size);
    s.rows = come > 0 ? (uint32_t) come : 0u;
    s.bad = have < 0 || have > cap || keep > cap;
    s.held = s.bad ? 0 : (int32_t) ((have + (int64_t) page_size - 1) >> shift);
    const int32_t kept = s.bad ? 0 : (int32_t) ((keep + page_size - 1) >> shift);
    s.need = kept > s.held ? (uint32_t) (kept - s.held) : 0u;
    s.give = kept < s.held ? (uint32_t) (s.held - kept) : 0u;
    s.len = s.bad ? (int32_t) (have < 0 ? 0 : have > cap ? cap : have) : (int32_t) keep;
    return s;
}
CACHE_HD uint32_t cache_add_sat(uint32_t a, uint32_t b) { return a + b < a ? 0xffffffffu : a + b; }
// first index of the ascending ends[n] that is greater than x (n if none)
CACHE_HD int cache_find(const uint32_t * ends, int n, uint32_t x) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ends[mid] > x) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}
// keys that the row at position pos of a sequence of len tokens reads: block 0 all, else those of its own and earlier
// blocks of `block` positions (1: causal). block is at most 2^30 (cache_block_of), as is len.
CACHE_HD int32_t cache_visible(int32_t pos, int32_t len, int32_t block) {
    if (block == 0) return len;
    if (pos < 0) return 0;
    const uint32_t end = block == 1 ? (uint32_t) pos + 1 : ((uint32_t) pos / (uint32_t) block + 1) * (uint32_t) block;
    return end < (uint32_t) len ? (int32_t) end : len;
}
// a caller's block in 32 bits: 2^30 positions are all that a sequence has
CACHE_HD int32_t cache_block_of(int64_t block) { return block < 1 << 30 ? (int32_t) block : 1 << 30; }
