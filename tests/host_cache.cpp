// Test program of cache_dev.h (the paged cache's layout and its arithmetic on lengths) on the host. Exit status 0: as it should be.
#include "cache_dev.h"

#include <cstdio>
#include <vector>

#define CHECK(x) do { if (!(x)) { fprintf(stderr, "line %d: %s\n", __LINE__, #x); return 1; } } while (0)

// every byte of a strip belongs to exactly one word or scale
static int layout() {
    for (int hd : {32, 64, 96, 128}) {
        std::vector<int> seen((size_t) cache_strip_bytes(hd), 0);
        auto mark = [&](int at, int n) { for (int i = 0; i < n; i++) seen.at((size_t) (at + i))++; };
        for (int t = 0; t < 16; t++) {
            for (int b = 0; b < hd / 32; b++) {
                for (int g = 0; g < 4; g++) mark(cache_k_word(t, g, b, hd), 4);
                mark(cache_k_scale(t, b, hd), 2);
                mark(cache_v_scale(t, b, hd), 2);
            }
            for (int w = 0; w < hd / 8; w++) mark(cache_v_word(t, w, hd), 4);
        }
        for (int n : seen) CHECK(n == 1);
        for (int ps : {16, 32, 64, 128, 256}) {      // strips follow each other, heads and pages too
            const int64_t sb = cache_strip_bytes(hd);
            CHECK(sb % 16 == 0 && cache_page_bytes(3, ps, hd) == 3 * (ps / 16) * sb);
            int64_t next = 0;
            for (int64_t page = 0; page < 3; page++)
                for (int h = 0; h < 3; h++)
                    for (int t = 0; t < ps; t += 16, next += sb) CHECK(cache_strip_at(page, h, t + 5, 3, ps, hd) == next);
            const int64_t far = 0x7ffffffeLL;        // past 32 bits
            CHECK(cache_strip_at(far, 2, ps - 1, 3, ps, hd) == far * cache_page_bytes(3, ps, hd) + cache_page_bytes(3, ps, hd) - sb);
        }
    }
    return 0;
}

static int steps() {
    auto s = cache_step_of(0, 0, 4, 16);
    CHECK(!s.bad && s.rows == 0 && s.need == 0 && s.give == 0 && s.len == 0 && s.held == 0);
    s = cache_step_of(16, 1, 4, 16);
    CHECK(!s.bad && s.rows == 1 && s.need == 1 && s.held == 1 && s.len == 17);
    s = cache_step_of(15, 1, 4, 16);
    CHECK(!s.bad && s.need == 0 && s.len == 16);
    s = cache_step_of(0, 64, 4, 16);
    CHECK(!s.bad && s.need == 4 && s.len == 64);
    s = cache_step_of(0, 65, 4, 16);
    CHECK(s.bad && s.rows == 65 && s.need == 0 && s.len == 0);
    s = cache_step_of(33, -1, 4, 16);
    CHECK(!s.bad && s.rows == 0 && s.give == 1 && s.held == 3 && s.len == 32);
    s = cache_step_of(33, -100, 4, 16);      // more than there are: all of them
    CHECK(!s.bad && s.give == 3 && s.len == 0);
    s = cache_step_of(-1, 5, 4, 16);
    CHECK(s.bad && s.rows == 5 && s.need == 0 && s.give == 0 && s.len == 0);
    s = cache_step_of(65, -5, 4, 16);        // a length that the table cannot hold
    CHECK(s.bad && s.give == 0 && s.len == 64);
    s = cache_step_of(0x7fffffff, 0x7fffffff, 0x7fffffff / 16, 16);
    CHECK(s.bad && s.need == 0);
    s = cache_step_of(0x7ffffff0, -0x7fffffff - 1, 0x7fffffff / 16, 16);
    CHECK(!s.bad && s.len == 0 && s.give == 0x7ffffffu);
    CHECK(cache_add_sat(0xffffffffu, 1) == 0xffffffffu && cache_add_sat(5, 6) == 11);
    return 0;
}

static int views() {
    const uint32_t e[] = {0, 3, 3, 7};
    CHECK(cache_find(e, 4, 0) == 1 && cache_find(e, 4, 2) == 1 && cache_find(e, 4, 3) == 3 && cache_find(e, 4, 6) == 3 && cache_find(e, 4, 7) == 4);
    CHECK(cache_find(e, 0, 0) == 0);
    CHECK(cache_visible(0, 10, 0) == 10 && cache_visible(3, 10, 1) == 4 && cache_visible(-1, 10, 1) == 0 && cache_visible(-1, 10, 0) == 10);
    CHECK(cache_visible(5, 10, 4) == 8 && cache_visible(9, 10, 4) == 10 && cache_visible(0, 10, cache_block_of((int64_t) 1 << 40)) == 10);
    CHECK(cache_visible(0x3fffffff, 0x40000000, 0x40000000) == 0x40000000 && cache_visible(0x3ffffffe, 0x40000000, 1) == 0x3fffffff && cache_visible(0x3fffffff, 0x40000000, 3) == 0x40000000);
    CHECK(cache_block_of(0) == 0 && cache_block_of(1) == 1 && cache_block_of(1 << 30) == 1 << 30);
    return 0;
}

int main() { return layout() || steps() || views(); }
