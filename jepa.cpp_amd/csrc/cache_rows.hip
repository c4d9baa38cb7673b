// cache_rows.hip - rows of keys and values into the 4-bit paged cache and back.
//
// A row of one head is hd / 32 ggml q4_0 blocks: m the block's first value of largest magnitude, d = m / -8,
// code = min(15, trunc(x / d + 8.5)) with x / d as fl(x * fl(1 / d)), value (code - 8) * f16(d): the arithmetic of
// k_quant_q4_0, so the values are those of jepa_amd_quantize_rows. Values beyond f16's range are held at its ends. A
// head of a row with a NaN or an infinity in its K or V is stored as K all NaN (the scales) and V all zero: a query
// that reads the key comes out NaN, as it would from the values, and no NaN can reach one that does not.
//
// Memory-bound: 32k bf16 rows of 8 x 128 are stored in 44 us (4.0 TB/s; the VALU is busy 70 % of it) and read in 26 (6.6 TB/s, the
// codes come from the last-level cache after a store). One thread takes 8 values of K and V (a 32-bit word of codes each), four threads a block (its maximum
// by two shuffles). A workgroup has 16 to 64 consecutive rows of one head (256 threads, 4 to 16 a row): of a prompt whole strips, which leave
// their L2 as whole lines (rows of all heads in a workgroup spread a strip over the L2s of all XCDs).
#include "cache_dev.h"
#include "common.h"
#include "kernels.h"

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));
typedef float float8 __attribute__((ext_vector_type(8)));
template <typename T> struct vec8;
template <> struct vec8<float> { typedef float8 t; };
template <> struct vec8<_Float16> { typedef half8 t; };
template <> struct vec8<__bf16> { typedef bhalf8 t; };

template <typename T> struct at16 { typedef typename vec8<T>::t t __attribute__((aligned(16))); };      // (rows lie at whole 16 bytes, f32's 8 values too)

template <typename T>
__device__ __forceinline__ float8 load8(const T * p) {
    return __builtin_convertvector(*(const typename at16<T>::t *) p, float8);
}
template <typename T>
__device__ __forceinline__ void store8(T * p, float8 x) {
    *(typename at16<T>::t *) p = __builtin_convertvector(x, typename vec8<T>::t);
}

__device__ __forceinline__ uint16_t f2h(float f) {
    asm volatile("" : "+v"(f));      // the f32 product is rounded first
    return __builtin_bit_cast(uint16_t, (_Float16) f);
}
__device__ __forceinline__ float h2f(uint16_t h) { return (float) __builtin_bit_cast(_Float16, h); }

// Codes of 8 of a block's 32 values (this thread's, of the four of a quad) and the block's f16 scale. Magnitudes are compared as their
// bits, held at f16's largest (a value beyond it gets the end code of its side as it would if it were held there itself).
__device__ __forceinline__ uint16_t quantize8(float8 x, int lane, uint32_t code[8], bool & finite) {
    constexpr uint32_t F16_MAX = 0x477fe000;      // 65504
    uint32_t most = 0, from = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) most = max(most, __float_as_uint(x[j]) & 0x7fffffffu);
    finite = most < 0x7f800000u;
    most = min(most, F16_MAX);
#pragma unroll
    for (int j = 7; j >= 0; j--)      // the first of equal magnitudes gives the sign
        if (min(__float_as_uint(x[j]) & 0x7fffffffu, F16_MAX) == most) from = __float_as_uint(x[j]);
    auto join = [&](uint32_t m, uint32_t f, bool second) {
        if (m > most || (m == most && second)) { most = m; from = f; }
    };
    // quad_perm 1 0 3 2, then 2 3 0 1: of equal magnitudes the lower lane's is the first
    join((uint32_t) __builtin_amdgcn_update_dpp(0, (int) most, 0xb1, 0xf, 0xf, true), (uint32_t) __builtin_amdgcn_update_dpp(0, (int) from, 0xb1, 0xf, 0xf, true), lane & 1);
    join((uint32_t) __builtin_amdgcn_update_dpp(0, (int) most, 0x4e, 0xf, 0xf, true), (uint32_t) __builtin_amdgcn_update_dpp(0, (int) from, 0x4e, 0xf, 0xf, true), lane & 2);
    const float d = __uint_as_float(most | (most ? from & 0x80000000u : 0u)) / -8.0f;      // (zeros of either sign: the format's -0)
    const float id = d != 0.0f ? 1.0f / d : 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) code[j] = (uint32_t) __builtin_amdgcn_fmed3f(x[j] * id + 8.5f, 0.0f, 15.0f);      // (an overflowing id: in range all the same)
    return f2h(d);
}

// lanes of a row of one head: hd / 8 threads work, the next power of two is the group
template <int HD> struct group { static constexpr int work = HD / 8, size = HD == 96 ? 16 : HD / 8, rows = 256 / size; };

template <typename T, int HD>
__global__ __launch_bounds__(256) void k_cache_store(unsigned char * __restrict__ cache, const T * __restrict__ k, int64_t ldk,
                                                     const T * __restrict__ v, int64_t ldv, int64_t n_rows, const int64_t * __restrict__ slots,
                                                     int n_kv_head, int page_shift, int64_t n_slots) {
    constexpr int GS = group<HD>::size, GW = group<HD>::work, ROWS = group<HD>::rows;
    const int tid = (int) threadIdx.x, lane = tid & 63, t = tid % GS, head = (int) (blockIdx.x % (unsigned) n_kv_head);
    const int64_t row = (int64_t) (blockIdx.x / (unsigned) n_kv_head) * ROWS + tid / GS;
    const bool has = row < n_rows && t < GW;
    const int64_t slot = has ? slots[row] : -1;
    float8 xk = {}, xv = {};
    if (has) {      // (whatever its slot: the loads do not wait for it)
        xk = load8(k + row * ldk + (int64_t) head * HD + 8 * t);
        xv = load8(v + row * ldv + (int64_t) head * HD + 8 * t);
    }
    uint32_t ck[8], cv[8];
    bool fk, fv;
    uint16_t dk = quantize8(xk, lane, ck, fk), dv = quantize8(xv, lane, cv, fv);
    const uint64_t odd = __ballot(!(fk && fv)) >> (lane & ~(GS - 1));
    if (slot < 0 || slot >= n_slots) return;
    if (odd & ((1ull << GS) - 1)) {
        dk = 0x7e00; dv = 0;
        for (int j = 0; j < 8; j++) ck[j] = cv[j] = 8;
    }
    uint32_t wk = 0, wv = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        wk |= ck[j] << (4 * ((j & 1) * 4 + (j >> 1)));
        wv |= cv[j] << (4 * j);
    }
    const int in_page = (int) slot & ((1 << page_shift) - 1), token = in_page % CACHE_STRIP, b = t / 4, g = t % 4;
    unsigned char * strip = cache + cache_strip_at(slot >> page_shift, head, in_page, n_kv_head, 1 << page_shift, HD);
    *(uint32_t *) (strip + cache_k_word(token, g, b, HD)) = wk;
    *(uint32_t *) (strip + cache_v_word(token, t, HD)) = wv;
    if (g == 0) {
        *(uint16_t *) (strip + cache_k_scale(token, b, HD)) = dk;
        *(uint16_t *) (strip + cache_v_scale(token, b, HD)) = dv;
    }
}

// rows whose slot is none of the cache's come out as zeros
template <typename T, int HD>
__global__ __launch_bounds__(256) void k_cache_read(const unsigned char * __restrict__ cache, const int64_t * __restrict__ slots, int64_t n_rows,
                                                    T * __restrict__ k, int64_t ldk, T * __restrict__ v, int64_t ldv, int n_kv_head,
                                                    int page_shift, int64_t n_slots) {
    constexpr int GS = group<HD>::size, GW = group<HD>::work, ROWS = group<HD>::rows;
    const int tid = (int) threadIdx.x, t = tid % GS, head = (int) (blockIdx.x % (unsigned) n_kv_head);
    const int64_t row = (int64_t) (blockIdx.x / (unsigned) n_kv_head) * ROWS + tid / GS;
    if (row >= n_rows || t >= GW) return;
    const int64_t slot = slots[row];
    float8 xk = {}, xv = {};
    if (slot >= 0 && slot < n_slots) {
        const int in_page = (int) slot & ((1 << page_shift) - 1), token = in_page % CACHE_STRIP, b = t / 4, g = t % 4;
        const unsigned char * strip = cache + cache_strip_at(slot >> page_shift, head, in_page, n_kv_head, 1 << page_shift, HD);
        const uint32_t wk = *(const uint32_t *) (strip + cache_k_word(token, g, b, HD)), wv = *(const uint32_t *) (strip + cache_v_word(token, t, HD));
        const float dk = h2f(*(const uint16_t *) (strip + cache_k_scale(token, b, HD))), dv = h2f(*(const uint16_t *) (strip + cache_v_scale(token, b, HD)));
#pragma unroll
        for (int j = 0; j < 8; j++) {
            xk[j] = (float) ((int) (wk >> (4 * ((j & 1) * 4 + (j >> 1))) & 15) - 8) * dk;
            xv[j] = (float) ((int) (wv >> (4 * j) & 15) - 8) * dv;
        }
    }
    store8(k + row * ldk + (int64_t) head * HD + 8 * t, xk);
    store8(v + row * ldv + (int64_t) head * HD + 8 * t, xv);
}

template <typename T, int HD>
hipError_t store(const cache_shape & c, void * cache, const void * k, int64_t ldk, const void * v, int64_t ldv, int64_t n_rows, const int64_t * slot, hipStream_t s) {
    int n_kv_head = c.n_kv_head, page_shift = __builtin_ctz((unsigned) c.page_size);
    int64_t n_slots = c.n_pages * c.page_size;
    const int64_t per = group<HD>::rows;
    void * p[] = {&cache, &k, &ldk, &v, &ldv, &n_rows, &slot, &n_kv_head, &page_shift, &n_slots};
    return hipLaunchKernel((const void *) k_cache_store<T, HD>, dim3((unsigned) ((n_rows + per - 1) / per * n_kv_head)), dim3(256), p, 0, s);
}

template <typename T, int HD>
hipError_t read(const cache_shape & c, const void * cache, const int64_t * slot, int64_t n_rows, void * k, int64_t ldk, void * v, int64_t ldv, hipStream_t s) {
    int n_kv_head = c.n_kv_head, page_shift = __builtin_ctz((unsigned) c.page_size);
    int64_t n_slots = c.n_pages * c.page_size;
    const int64_t per = group<HD>::rows;
    void * p[] = {&cache, &slot, &n_rows, &k, &ldk, &v, &ldv, &n_kv_head, &page_shift, &n_slots};
    return hipLaunchKernel((const void *) k_cache_read<T, HD>, dim3((unsigned) ((n_rows + per - 1) / per * n_kv_head)), dim3(256), p, 0, s);
}

}  // namespace

#define BY_HEAD(T, ...) (c.hd == 32 ? __VA_ARGS__(T, 32) : c.hd == 64 ? __VA_ARGS__(T, 64) : c.hd == 96 ? __VA_ARGS__(T, 96) : __VA_ARGS__(T, 128))
#define BY_TYPE(...) (type == T_F32 ? BY_HEAD(float, __VA_ARGS__) : type == T_F16 ? BY_HEAD(_Float16, __VA_ARGS__) : BY_HEAD(__bf16, __VA_ARGS__))

hipError_t launch_cache_store(const cache_shape & c, void * cache, int type, const void * k, int64_t ldk, const void * v, int64_t ldv,
                              int64_t n_rows, const int64_t * slot, hipStream_t s) {
#define CALL(T, HD) store<T, HD>(c, cache, k, ldk, v, ldv, n_rows, slot, s)
    return BY_TYPE(CALL);
#undef CALL
}

hipError_t launch_cache_read(const cache_shape & c, const void * cache, const int64_t * slot, int64_t n_rows, int type, void * k,
                             int64_t ldk, void * v, int64_t ldv, hipStream_t s) {
#define CALL(T, HD) read<T, HD>(c, cache, slot, n_rows, k, ldk, v, ldv, s)
    return BY_TYPE(CALL);
#undef CALL
}
