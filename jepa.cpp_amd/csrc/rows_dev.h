// rows_dev.h - 8 values of a row at a time, and their way into the 4-bit cache.
#pragma once
#include "cache_dev.h"
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

// 8 values of K and V, dims 8 t .. 8 t + 7 of one head of a row, quantized into the row's slot. All lanes of a wave come here.
template <int HD>
__device__ __forceinline__ void store_head(unsigned char * __restrict__ cache, float8 xk, float8 xv, int64_t slot, int lane, int t, int head, int n_kv_head, int page_shift,
                                           int64_t n_slots) {
    constexpr int GS = group<HD>::size, GW = group<HD>::work;
    uint32_t ck[8], cv[8];
    bool fk, fv;
    uint16_t dk = quantize8(xk, lane, ck, fk), dv = quantize8(xv, lane, cv, fv);
    const uint64_t odd = __ballot((GW == GS || t < GW) && !(fk && fv)) >> (lane & ~(GS - 1));      // (lanes without work may hold anything)
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

}  // namespace
