// cache_api.cpp - the 4-bit paged key/value cache's entry points of include/jepa_amd.h: argument checks, then one or two
// launches on the caller's stream. Nothing is allocated and nothing waits, so the calls can be captured into a graph.
#include "../../include/jepa_amd.h"
#include "cache_dev.h"
#include "kernels.h"
#include "model.h"

#include <cmath>

namespace {

constexpr int64_t I31 = 0x7fffffff;
constexpr int64_t MAX_TOKENS = 1 << 30;      // of a table row: positions and the steps past them stay in 32 bits

// the shape, checked; who: the entry point for the message
bool shape_of(const char * who, const jepa_amd_cache_shape * s, cache_shape & c) {
    if (!s) { jepa_log("jepa: %s: no shape\n", who); return false; }
    const bool page = s->page_size == 16 || s->page_size == 32 || s->page_size == 64 || s->page_size == 128 || s->page_size == 256;
    const bool hd = s->head_dim == 32 || s->head_dim == 64 || s->head_dim == 96 || s->head_dim == 128;
    if (!page || !hd || s->n_kv_head < 1 || s->n_head < 1 || s->n_head > 4096 || s->n_head % s->n_kv_head || s->n_pages < 1 || s->n_pages > I31) {
        jepa_log("jepa: %s: %d heads over %d of width %d, %lld pages of %d tokens not supported (heads a multiple of the K/V heads, up to 4096; "
                 "width 32, 64, 96 or 128; pages of 16, 32, 64, 128 or 256)\n",
                 who, s->n_head, s->n_kv_head, s->head_dim, (long long) s->n_pages, s->page_size);
        return false;
    }
    c.n_head = s->n_head; c.n_kv_head = s->n_kv_head; c.hd = s->head_dim; c.page_size = s->page_size; c.n_pages = s->n_pages;
    return true;
}

bool sizes_ok(const char * who, const cache_shape & c, int64_t n_seq, int64_t n_rows, int64_t width) {
    if (n_seq < 0 || n_seq > CACHE_MAX_SEQ || n_rows < 0 || n_rows >= I31 || width < 1 || width > MAX_TOKENS / c.page_size) {
        jepa_log("jepa: %s: %lld sequences, %lld rows, tables of %lld pages not supported (up to %d sequences, 2^31 rows, 2^30 tokens of a table row)\n",
                 who, (long long) n_seq, (long long) n_rows, (long long) width, CACHE_MAX_SEQ);
        return false;
    }
    return true;
}

// packed rows of n_heads heads: an element type, a 16-byte aligned start and a stride in whole 16 bytes
bool rows_ok(const char * who, const char * what, int type, const void * p, int64_t ld, int64_t width, int64_t n_rows) {
    const int64_t size = type == T_F32 ? 4 : 2;
    if (type != T_F32 && type != T_F16 && type != T_BF16) { jepa_log("jepa: %s: type %d not supported (0 f32, 1 f16, 30 bf16)\n", who, type); return false; }
    if (!p && n_rows) { jepa_log("jepa: %s: %s is NULL\n", who, what); return false; }
    if ((uintptr_t) p % 16 || ld * size % 16 || ld < width || ld > ((int64_t) 1 << 40)) {
        jepa_log("jepa: %s: %s rows of %lld elements, %lld apart: start and stride must be whole 16 bytes, the stride at least the row\n", who, what,
                 (long long) width, (long long) ld);
        return false;
    }
    return true;
}

// heads of rows that one launch takes (its threads are below 2^32, 16 of them for a head of a row, or 64 for one of a few rows)
bool grid_ok(const char * who, int64_t n) {
    if (n < (int64_t) 1 << 27) return true;
    jepa_log("jepa: %s: %lld heads of rows in one call (below 2^27)\n", who, (long long) n);
    return false;
}

bool cache_ok(const char * who, const void * cache) {
    if (cache && (uintptr_t) cache % 16 == 0) return true;
    jepa_log("jepa: %s: the cache must be 16-byte aligned device memory\n", who);
    return false;
}

bool all(const char * who, std::initializer_list<const void *> ps) {
    for (const void * p : ps)
        if (!p) { jepa_log("jepa: %s: a pointer is NULL\n", who); return false; }
    return true;
}

// `f` with `device` current, which it is no longer afterwards if it was not before
template <typename F>
int on_device(const char * who, int device, F f) {
    if (!dev_check(device)) return -1;
    int prev = 0;
    if (hipGetDevice(&prev) != hipSuccess || (prev != device && hipSetDevice(device) != hipSuccess)) {
        jepa_log("jepa: cannot use HIP device %d\n", device);
        return -1;
    }
    const hipError_t e = f();
    if (prev != device) hipSetDevice(prev);
    if (e == hipSuccess) return 0;
    (void) hipGetLastError();      // reported here, not by the thread's next call
    jepa_log("jepa: %s: launch failed: %s\n", who, hipGetErrorString(e));
    return -1;
}

}  // namespace

extern "C" int64_t jepa_amd_cache_page_bytes(const jepa_amd_cache_shape * shape) {
    cache_shape c;
    if (!shape_of("jepa_amd_cache_page_bytes", shape, c)) return -1;
    return cache_page_bytes(c.n_kv_head, c.page_size, c.hd);
}

extern "C" int64_t jepa_amd_cache_work_bytes(const jepa_amd_cache_shape * shape, int64_t n_seq, int64_t n_rows, int64_t table_width) {
    cache_shape c;
    if (!shape_of("jepa_amd_cache_work_bytes", shape, c) || !sizes_ok("jepa_amd_cache_work_bytes", c, n_seq, n_rows, table_width)) return -1;
    return cache_attention_work_bytes(c, n_seq, n_rows, table_width);
}

extern "C" int jepa_amd_cache_plan(int device, const jepa_amd_cache_shape * shape, int64_t n_seq, int64_t n_rows, const int32_t * len,
                                   const int32_t * n_new, int32_t * table, int64_t table_width, int32_t * ring, const int32_t * free_in,
                                   int32_t * free_out, int32_t * kv_len, int32_t * row_start, int64_t * slot, int32_t * refused, void * stream) {
    const char * who = "jepa_amd_cache_plan";
    cache_shape c;
    if (!shape_of(who, shape, c) || !sizes_ok(who, c, n_seq, n_rows, table_width) || !all(who, {ring, free_in, free_out, row_start}) ||
        (n_seq && !all(who, {len, n_new, table, kv_len, refused})) || (n_rows && !all(who, {slot})))
        return -1;
    cache_plan_args a;
    a.n_seq = (int) n_seq; a.width = (int) table_width; a.page_size = c.page_size; a.n_rows = n_rows; a.n_pages = c.n_pages;
    a.len = len; a.come = n_new; a.free_in = free_in;
    a.table = table; a.ring = ring; a.free_out = free_out; a.kv_len = kv_len; a.row_start = row_start; a.refused = refused; a.slot = slot;
    return on_device(who, device, [&] { return launch_cache_plan(a, (hipStream_t) stream); });
}

extern "C" int jepa_amd_cache_store(int device, const jepa_amd_cache_shape * shape, void * cache, int type, const void * k, int64_t k_stride,
                                    const void * v, int64_t v_stride, int64_t n_rows, const int64_t * slot, void * stream) {
    const char * who = "jepa_amd_cache_store";
    cache_shape c;
    if (!shape_of(who, shape, c) || !sizes_ok(who, c, 0, n_rows, 1)) return -1;
    const int64_t width = (int64_t) c.n_kv_head * c.hd;
    if (!cache_ok(who, cache) || !rows_ok(who, "k", type, k, k_stride, width, n_rows) ||
        !rows_ok(who, "v", type, v, v_stride, width, n_rows) || (n_rows && !all(who, {slot})) || !grid_ok(who, n_rows * c.n_kv_head))
        return -1;
    return on_device(who, device, [&] {
        return n_rows ? launch_cache_store(c, cache, type, k, k_stride, v, v_stride, n_rows, slot, (hipStream_t) stream) : hipSuccess;
    });
}

extern "C" int jepa_amd_cache_read(int device, const jepa_amd_cache_shape * shape, const void * cache, const int64_t * slot, int64_t n_rows, int type,
                                   void * k, int64_t k_stride, void * v, int64_t v_stride, void * stream) {
    const char * who = "jepa_amd_cache_read";
    cache_shape c;
    if (!shape_of(who, shape, c) || !sizes_ok(who, c, 0, n_rows, 1)) return -1;
    const int64_t width = (int64_t) c.n_kv_head * c.hd;
    if (!cache_ok(who, cache) || !rows_ok(who, "k", type, k, k_stride, width, n_rows) ||
        !rows_ok(who, "v", type, v, v_stride, width, n_rows) || (n_rows && !all(who, {slot})) || !grid_ok(who, n_rows * c.n_kv_head))
        return -1;
    return on_device(who, device, [&] {
        return n_rows ? launch_cache_read(c, cache, slot, n_rows, type, k, k_stride, v, v_stride, (hipStream_t) stream) : hipSuccess;
    });
}

extern "C" int jepa_amd_cache_attention(int device, const jepa_amd_cache_shape * shape, const void * cache, int type, const void * q, int64_t q_stride,
                                        int64_t n_seq, int64_t n_rows, const int32_t * row_start, const int32_t * kv_len, const int32_t * table,
                                        int64_t table_width, float scale, int64_t causal_block, void * out, int64_t out_stride, void * work,
                                        int64_t work_bytes, void * stream) {
    const char * who = "jepa_amd_cache_attention";
    cache_shape c;
    if (!shape_of(who, shape, c) || !sizes_ok(who, c, n_seq, n_rows, table_width)) return -1;
    const int64_t width = (int64_t) c.n_head * c.hd;
    if (!cache_ok(who, cache) || !rows_ok(who, "q", type, q, q_stride, width, n_rows) ||
        !rows_ok(who, "out", type, out, out_stride, width, n_rows) || !grid_ok(who, n_rows * c.n_head))
        return -1;
    if (!std::isfinite(scale) || causal_block < 0) {
        jepa_log("jepa: %s: scale %g, causal block %lld\n", who, (double) scale, (long long) causal_block);
        return -1;
    }
    const int64_t blocks = cache_attention_blocks(c, type, n_seq, n_rows, table_width);
    if (n_rows && n_seq && blocks >= 1 << 24) {      // (threads of a launch are below 2^32)
        jepa_log("jepa: %s: %lld rows of %d heads in %lld sequences over %d K/V heads: %lld workgroups in one call (below 2^24)\n", who, (long long) n_rows, c.n_head,
                 (long long) n_seq, c.n_kv_head, (long long) blocks);
        return -1;
    }
    const int64_t need = cache_attention_work_bytes(c, n_seq, n_rows, table_width);
    if (n_rows && n_seq && (!all(who, {row_start, kv_len, table, work}))) return -1;
    if (n_rows && n_seq && ((uintptr_t) work % 16 || work_bytes < need)) {
        jepa_log("jepa: %s: %lld bytes of work space, %lld needed (16-byte aligned)\n", who, (long long) work_bytes, (long long) need);
        return -1;
    }
    cache_attn_args a;
    a.cache = (const unsigned char *) cache; a.q = q; a.out = out; a.ldq = q_stride; a.ldo = out_stride; a.n_rows = n_rows; a.n_pages = c.n_pages;
    a.block = cache_block_of(causal_block); a.row_start = row_start; a.kv_len = kv_len; a.table = table; a.n_seq = (int) n_seq; a.width = (int) table_width;
    a.n_head = c.n_head; a.n_kv_head = c.n_kv_head; a.page_size = c.page_size; a.scale = scale; a.work = (float *) work;
    return on_device(who, device, [&] { return n_rows && n_seq ? launch_cache_attention(c, type, a, (hipStream_t) stream) : hipSuccess; });
}
