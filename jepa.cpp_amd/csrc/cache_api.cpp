// cache_api.cpp - entry points of include/jepa_amd.h for rotary positions and the 4-bit paged key/value cache: argument checks, then one or two
// launches on the caller's stream. Nothing is allocated and nothing waits, so the calls can be captured into a graph.
#include "../../include/jepa_amd.h"
#include "cache_dev.h"
#include "kernels.h"
#include "model.h"

#include <algorithm>
#include <cmath>
#include <iterator>

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

// the description of a rotation, checked; frequencies in more than 64 bits, each rounded once
bool rope_of(const char * who, const jepa_amd_rope_axes * r, rope_map & m) {
    if (!r) { jepa_log("jepa: %s: no rotation\n", who); return false; }
    bool ok = r->head_dim >= 8 && r->head_dim <= 256 && r->head_dim % 8 == 0 && r->form >= 0 && r->form <= 3 && r->n_axes >= 1 && r->n_axes <= 4 &&
              std::isfinite(r->theta) && r->theta > 0.0;
    int rot = 0;
    for (int a = 0; ok && a < r->n_axes; a++) {
        ok = r->dims[a] >= 2 && r->dims[a] <= 256 && r->dims[a] % (r->form == 2 ? 16 : 2) == 0 && std::isfinite(r->scale[a]);
        rot += r->dims[a];
    }
    if (!ok || rot > r->head_dim || (r->form == 3 && rot % 16)) {
        jepa_log("jepa: %s: rotation of form %d over %d axes of heads of %d not supported (forms 0 to 3; 1 to 4 axes of an even number of dims each, of whole 16 "
                 "in form 2, whole 16 together in form 3, no more than the head; heads of 8 to 256, whole 8; theta above 0, scales finite)\n",
                 who, r->form, r->n_axes, r->head_dim);
        return false;
    }
    m.form = r->form; m.hd = r->head_dim; m.rot = rot; m.n_axes = r->n_axes;
    const bool halves = r->form >= 2;
    std::fill(std::begin(m.rev), std::end(m.rev), 0.0);
    std::fill(std::begin(m.axis), std::end(m.axis), (uint8_t) 0);
    std::fill(std::begin(m.delta), std::end(m.delta), (int16_t) 0);
    const long double two_pi = 6.283185307179586476925286766559L;
    auto step_of = [&](int width) { return powl((long double) r->theta, -2.0L / width); };
    auto put = [&](int e, int axis, long double f) { m.rev[e] = (double) (f * r->scale[axis] / two_pi); m.axis[e] = (uint8_t) axis; };
    long double f = 1.0L, step = r->form == 3 ? step_of(rot) : 0.0L;
    for (int a = 0, at = 0; a < r->n_axes; at += r->dims[a++]) {
        const int w = r->dims[a], h = w / 2;
        if (r->form != 3) { f = 1.0L; step = step_of(w); }
        for (int i = 0; i < h; i++, f *= step) {
            if (r->form == 0) { put(at + i, a, f); put(at + i + h, a, f); }      // the frequencies run twice through the section, across its pairs
            if (r->form == 1) { put(at + 2 * i, a, f); put(at + 2 * i + 1, a, f); }
            if (r->form == 2) { put(at + i, a, f); put(at + i + h, a, f); }
            if (r->form == 3) { put(at / 2 + i, a, f); put(at / 2 + i + rot / 2, a, f); }
        }
        for (int i = 0; r->form == 2 && i < w / 8; i++) m.delta[at / 8 + i] = (int16_t) (i < w / 16 ? h : -h);
    }
    for (int i = 0; r->form == 3 && i < rot / 8; i++) m.delta[i] = (int16_t) (i < rot / 16 ? rot / 2 : -(rot / 2));
    for (int e = 0; e < rot; e++)
        if (!(std::fabs(m.rev[e]) <= 0x1p990)) {      // (times a position of 32 bits, still finite)
            jepa_log("jepa: %s: theta %g, axis %d scaled by %g: angles past 64 bits\n", who, r->theta, m.axis[e], r->scale[m.axis[e]]);
            return false;
        }
    int leads = 0;
    std::fill(std::begin(m.lead), std::end(m.lead), (uint8_t) 0);
    for (int i = 0; i < m.hd / 8; i++)
        if (!halves || m.delta[i] >= 0) m.lead[leads++] = (uint8_t) i;
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

bool digest_ok(const char * who, const void * digest) {
    if (digest && (uintptr_t) digest % 16 == 0) return true;
    jepa_log("jepa: %s: the digests must be 16-byte aligned device memory\n", who);
    return false;
}

bool take_ok(const char * who, int64_t first, int64_t last, int64_t take) {
    if (take >= 1 && take <= CACHE_MOST_SELECTED && first >= 0 && first <= take && last >= 0 && last <= take - first) return true;
    jepa_log("jepa: %s: %lld pages of a row, %lld first and %lld last ones among them, not supported (1 to %d pages)\n", who, (long long) take, (long long) first,
             (long long) last, CACHE_MOST_SELECTED);
    return false;
}

// (threads of a launch are below 2^32)
bool blocks_ok(const char * who, int64_t blocks) {
    if (blocks < 1 << 24) return true;
    jepa_log("jepa: %s: %lld workgroups in one call (below 2^24)\n", who, (long long) blocks);
    return false;
}

bool work_ok(const char * who, const void * work, int64_t bytes, int64_t need) {
    if (need == 0 || (work && (uintptr_t) work % 16 == 0 && bytes >= need)) return true;
    jepa_log("jepa: %s: %lld bytes of work space, %lld needed (16-byte aligned)\n", who, (long long) bytes, (long long) need);
    return false;
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

extern "C" int jepa_amd_rope_rows(int device, const jepa_amd_rope_axes * rope, int type, const void * x, int64_t x_stride, int64_t n_rows, int n_head,
                                  const int32_t * pos, int backward, void * out, int64_t out_stride, void * stream) {
    const char * who = "jepa_amd_rope_rows";
    rope_map m;
    if (!rope_of(who, rope, m)) return -1;
    if (n_head < 1 || n_head > 4096 || n_rows < 0 || n_rows >= I31 || n_rows * n_head >= (int64_t) 1 << 26) {
        jepa_log("jepa: %s: %lld rows of %d heads not supported (up to 4096 heads, below 2^26 heads of rows)\n", who, (long long) n_rows, n_head);
        return -1;
    }
    const int64_t width = (int64_t) n_head * m.hd;
    if (!rows_ok(who, "x", type, x, x_stride, width, n_rows) || !rows_ok(who, "out", type, out, out_stride, width, n_rows) || (n_rows && !all(who, {pos}))) return -1;
    if (x == out && x_stride != out_stride) { jepa_log("jepa: %s: rows in place must keep their stride\n", who); return -1; }
    rope_args a;
    a.x = x; a.out = out; a.ldx = x_stride; a.ldo = out_stride; a.n_rows = n_rows; a.pos = pos; a.n_head = n_head; a.hd = m.hd; a.back = backward != 0;
    return on_device(who, device, [&] { return n_rows ? launch_rope_axes(a, m, type, (hipStream_t) stream) : hipSuccess; });
}

extern "C" int jepa_amd_cache_append(int device, const jepa_amd_cache_shape * shape, const jepa_amd_rope_axes * rope, void * cache, int type, const void * q,
                                     int64_t q_stride, const void * k, int64_t k_stride, const void * v, int64_t v_stride, int64_t n_rows, const int32_t * pos,
                                     const int64_t * slot, void * q_out, int64_t q_out_stride, void * stream) {
    const char * who = "jepa_amd_cache_append";
    cache_shape c;
    rope_map m;
    if (!shape_of(who, shape, c) || !sizes_ok(who, c, 0, n_rows, 1) || !rope_of(who, rope, m)) return -1;
    if (m.hd != c.hd) { jepa_log("jepa: %s: a rotation of heads of %d for a cache of %d\n", who, m.hd, c.hd); return -1; }
    const int64_t width = (int64_t) c.n_kv_head * c.hd, q_width = (int64_t) c.n_head * c.hd;
    if (!cache_ok(who, cache) || !rows_ok(who, "k", type, k, k_stride, width, n_rows) || !rows_ok(who, "v", type, v, v_stride, width, n_rows) ||
        (q && (!rows_ok(who, "q", type, q, q_stride, q_width, n_rows) || !rows_ok(who, "q_out", type, q_out, q_out_stride, q_width, n_rows))) ||
        (n_rows && !all(who, {pos, slot})))
        return -1;
    if (n_rows * c.n_head >= (int64_t) 1 << 26) { jepa_log("jepa: %s: %lld heads of rows in one call (below 2^26)\n", who, (long long) (n_rows * c.n_head)); return -1; }
    if (q && q == q_out && q_stride != q_out_stride) { jepa_log("jepa: %s: rows in place must keep their stride\n", who); return -1; }
    append_args a;
    a.cache = (unsigned char *) cache; a.k = k; a.v = v; a.ldk = k_stride; a.ldv = v_stride; a.n_rows = n_rows; a.n_slots = c.n_pages * c.page_size; a.pos = pos;
    a.slots = slot; a.n_kv_head = c.n_kv_head; a.page_shift = __builtin_ctz((unsigned) c.page_size);
    rope_args r;
    r.x = q; r.out = q_out; r.ldx = q_stride; r.ldo = q_out_stride; r.n_rows = n_rows; r.pos = pos; r.n_head = c.n_head; r.hd = c.hd;
    return on_device(who, device, [&] { return n_rows ? launch_cache_append(a, r, m, type, (hipStream_t) stream) : hipSuccess; });
}

extern "C" int64_t jepa_amd_cache_digest_bytes(const jepa_amd_cache_shape * shape) {
    cache_shape c;
    if (!shape_of("jepa_amd_cache_digest_bytes", shape, c)) return -1;
    return c.n_kv_head * cache_digest_bytes(c.hd);
}

extern "C" int jepa_amd_cache_digest(int device, const jepa_amd_cache_shape * shape, const void * cache, int64_t n_seq, int64_t n_rows, const int32_t * row_start,
                                     const int32_t * kv_len, const int32_t * table, int64_t table_width, void * digest, void * stream) {
    const char * who = "jepa_amd_cache_digest";
    cache_shape c;
    if (!shape_of(who, shape, c) || !sizes_ok(who, c, n_seq, n_rows, table_width) || !cache_ok(who, cache) || !digest_ok(who, digest)) return -1;
    const bool some = n_seq && n_rows;
    if (some && (!all(who, {row_start, kv_len, table}) || !blocks_ok(who, cache_digest_blocks(c, n_seq, n_rows)))) return -1;
    cache_digest_args a;
    a.cache = (const unsigned char *) cache; a.digest = (unsigned char *) digest; a.row_start = row_start; a.kv_len = kv_len; a.table = table; a.n_rows = n_rows;
    a.n_pages = c.n_pages; a.n_seq = (int) n_seq; a.width = (int) table_width; a.n_kv_head = c.n_kv_head; a.page_size = c.page_size;
    return on_device(who, device, [&] { return some ? launch_cache_digest(c, a, (hipStream_t) stream) : hipSuccess; });
}

extern "C" int jepa_amd_cache_digest_read(int device, const jepa_amd_cache_shape * shape, const void * digest, const int32_t * page, int64_t n, float * bounds, void * stream) {
    const char * who = "jepa_amd_cache_digest_read";
    cache_shape c;
    if (!shape_of(who, shape, c) || !digest_ok(who, digest)) return -1;
    if (n < 0 || n >= I31 || n * c.n_kv_head >= 1 << 25) { jepa_log("jepa: %s: %lld pages of %d heads in one call (below 2^25 heads)\n", who, (long long) n, c.n_kv_head); return -1; }
    if (n && (!all(who, {page, bounds}))) return -1;
    if ((uintptr_t) bounds % 16) { jepa_log("jepa: %s: the bounds must be 16-byte aligned\n", who); return -1; }
    return on_device(who, device, [&] {
        return n ? launch_cache_digest_read((const unsigned char *) digest, page, n, c.n_pages, c.n_kv_head, c.hd, bounds, (hipStream_t) stream) : hipSuccess;
    });
}

extern "C" int64_t jepa_amd_cache_select_work_bytes(const jepa_amd_cache_shape * shape, int64_t n_seq, int64_t n_rows, int64_t table_width, int64_t n_select) {
    const char * who = "jepa_amd_cache_select_work_bytes";
    cache_shape c;
    if (!shape_of(who, shape, c) || !sizes_ok(who, c, n_seq, n_rows, table_width) || !take_ok(who, 0, 0, n_select)) return -1;
    return cache_select_work_bytes(c, n_rows, table_width, (int) n_select);
}

extern "C" int jepa_amd_cache_select(int device, const jepa_amd_cache_shape * shape, const void * digest, int type, const void * q, int64_t q_stride, int64_t n_seq,
                                     int64_t n_rows, const int32_t * row_start, const int32_t * kv_len, const int32_t * table, int64_t table_width,
                                     int64_t causal_block, int64_t n_first, int64_t n_last, int64_t n_select, int32_t * selected, void * work, int64_t work_bytes,
                                     void * stream) {
    const char * who = "jepa_amd_cache_select";
    cache_shape c;
    if (!shape_of(who, shape, c) || !sizes_ok(who, c, n_seq, n_rows, table_width) || !digest_ok(who, digest) ||
        !rows_ok(who, "q", type, q, q_stride, (int64_t) c.n_head * c.hd, n_rows) || !grid_ok(who, n_rows * c.n_head) || !take_ok(who, n_first, n_last, n_select))
        return -1;
    if (causal_block < 0 || n_last < 1) {
        jepa_log("jepa: %s: causal block %lld, %lld last pages (1 or more: the page that a row ends in is one)\n", who, (long long) causal_block, (long long) n_last);
        return -1;
    }
    const bool some = n_seq && n_rows;
    if (some && (!all(who, {row_start, kv_len, table, selected}) || !blocks_ok(who, cache_select_blocks(c, n_seq, n_rows, table_width)) ||
                 !work_ok(who, work, work_bytes, cache_select_work_bytes(c, n_rows, table_width, (int) n_select))))
        return -1;
    cache_select_args a;
    a.digest = (const unsigned char *) digest; a.q = q; a.selected = selected; a.ldq = q_stride; a.n_rows = n_rows; a.n_pages = c.n_pages; a.row_start = row_start;
    a.kv_len = kv_len; a.table = table; a.n_seq = (int) n_seq; a.width = (int) table_width; a.n_head = c.n_head; a.n_kv_head = c.n_kv_head; a.page_size = c.page_size;
    a.block = cache_block_of(causal_block); a.first = (int) n_first; a.last = (int) n_last; a.take = (int) n_select; a.work = (float *) work;
    return on_device(who, device, [&] { return some ? launch_cache_select(c, type, a, (hipStream_t) stream) : hipSuccess; });
}

extern "C" int64_t jepa_amd_cache_selected_work_bytes(const jepa_amd_cache_shape * shape, int64_t n_rows, int64_t n_select) {
    const char * who = "jepa_amd_cache_selected_work_bytes";
    cache_shape c;
    if (!shape_of(who, shape, c) || !sizes_ok(who, c, 0, n_rows, 1) || !take_ok(who, 0, 0, n_select)) return -1;
    return cache_selected_work_bytes(c, n_rows, (int) n_select);
}

extern "C" int jepa_amd_cache_attention_selected(int device, const jepa_amd_cache_shape * shape, const void * cache, int type, const void * q, int64_t q_stride,
                                                 int64_t n_seq, int64_t n_rows, const int32_t * row_start, const int32_t * kv_len, const int32_t * table,
                                                 int64_t table_width, const int32_t * selected, int64_t n_select, float scale, int64_t causal_block, void * out,
                                                 int64_t out_stride, void * work, int64_t work_bytes, void * stream) {
    const char * who = "jepa_amd_cache_attention_selected";
    cache_shape c;
    if (!shape_of(who, shape, c) || !sizes_ok(who, c, n_seq, n_rows, table_width)) return -1;
    const int64_t width = (int64_t) c.n_head * c.hd;
    if (!cache_ok(who, cache) || !rows_ok(who, "q", type, q, q_stride, width, n_rows) || !rows_ok(who, "out", type, out, out_stride, width, n_rows) ||
        !grid_ok(who, n_rows * c.n_head) || !take_ok(who, 0, 0, n_select))
        return -1;
    if (!std::isfinite(scale) || causal_block < 0) {
        jepa_log("jepa: %s: scale %g, causal block %lld\n", who, (double) scale, (long long) causal_block);
        return -1;
    }
    const bool some = n_seq && n_rows;
    if (some && (!all(who, {row_start, kv_len, table, selected}) || !blocks_ok(who, cache_selected_blocks(c, n_rows, (int) n_select)) ||
                 !work_ok(who, work, work_bytes, cache_selected_work_bytes(c, n_rows, (int) n_select))))
        return -1;
    cache_selected_args a;
    a.cache = (const unsigned char *) cache; a.q = q; a.out = out; a.ldq = q_stride; a.ldo = out_stride; a.n_rows = n_rows; a.n_pages = c.n_pages;
    a.row_start = row_start; a.kv_len = kv_len; a.table = table; a.selected = selected; a.n_seq = (int) n_seq; a.width = (int) table_width; a.n_head = c.n_head;
    a.n_kv_head = c.n_kv_head; a.page_size = c.page_size; a.block = cache_block_of(causal_block); a.take = (int) n_select; a.scale = scale; a.work = (float *) work;
    return on_device(who, device, [&] { return some ? launch_cache_selected(c, type, a, (hipStream_t) stream) : hipSuccess; });
}
