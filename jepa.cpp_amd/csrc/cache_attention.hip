// cache_attention.hip - attention of packed query rows over the 4-bit paged cache.
//
// One workgroup takes one row of one head: 256 keys at a time, a key a thread for the scores, then a dimension a thread
// for the weighted sum, with the running maximum and sum of the softmax.
#include "cache_dev.h"
#include "common.h"
#include "kernels.h"

namespace {

__device__ __forceinline__ float h2f(uint16_t h) { return (float) __builtin_bit_cast(_Float16, h); }

template <typename T, int HD>
__global__ __launch_bounds__(256) void k_cache_attention(cache_attn_args a) {
    constexpr int NB = HD / 32, PARTS = 256 / HD;
    __shared__ float q[HD], p[256], red[4], acc[PARTS][HD];
    __shared__ int64_t at[256];      // the strip of each of the 256 keys, -1: none
    const int tid = (int) threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int64_t row = blockIdx.x;
    const int head = (int) blockIdx.y, kvh = head / (a.n_head / a.n_kv_head);
    const int seq = cache_find((const uint32_t *) a.row_start + 1, a.n_seq, (uint32_t) row);
    if (seq >= a.n_seq || row < a.row_start[seq]) return;      // rows behind the last sequence are left as they are
    const int64_t cap = (int64_t) a.width * a.page_size;
    const int32_t len = (int32_t) min<int64_t>(max(a.kv_len[seq], 0), cap);
    const int32_t n = cache_visible((int64_t) len - (a.row_start[seq + 1] - row), len, a.block);
    if (tid < HD) q[tid] = (float) ((const T *) a.q)[row * a.ldq + (int64_t) head * HD + tid];
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    const int dim = tid % HD, part = tid / HD;
    for (int32_t k0 = 0; k0 < n; k0 += 256) {
        __syncthreads();
        const int32_t key = k0 + tid;
        float s = -INFINITY;
        at[tid] = -1;
        if (key < n) {
            const int32_t page = a.table[(int64_t) seq * a.width + key / a.page_size];
            if (page >= 0 && page < a.n_pages) {
                const int in_page = key % a.page_size;
                at[tid] = cache_strip_at(page, kvh, in_page, a.n_kv_head, a.page_size, HD);
                const unsigned char * strip = a.cache + at[tid];
                s = 0.0f;
                for (int b = 0; b < NB; b++) {
                    float x = 0.0f;
                    for (int g = 0; g < 4; g++) {
                        const uint32_t w = *(const uint32_t *) (strip + cache_k_word(key % 16, g, b, HD));
                        for (int j = 0; j < 8; j++) x += q[32 * b + 8 * g + j] * (float) ((int) (w >> (4 * ((j & 1) * 4 + (j >> 1))) & 15) - 8);
                    }
                    s += x * h2f(*(const uint16_t *) (strip + cache_k_scale(key % 16, b, HD)));
                }
                s *= a.scale;
            }
        }
        float mx = s;
        for (int k = 32; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor(mx, k, 64));
        if (lane == 0) red[wv] = mx;
        __syncthreads();
        mx = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
        const float mu = mx == -INFINITY ? 0.0f : mx;
        const float e = at[tid] < 0 ? 0.0f : expf(s - mu), back = expf(m - mu);
        m = mx;
        p[tid] = e;
        float sum = e;
        for (int k = 32; k > 0; k >>= 1) sum += __shfl_xor(sum, k, 64);
        __syncthreads();
        if (lane == 0) red[wv] = sum;
        __syncthreads();
        l = l * back + (red[0] + red[1]) + (red[2] + red[3]);
        o *= back;
        if (part < PARTS)
            for (int j = part; j < 256; j += PARTS) {
                if (at[j] < 0) continue;
                const unsigned char * strip = a.cache + at[j];
                const int token = (k0 + j) % 16;
                const int code = strip[8 * HD + token * (HD / 2) + dim / 2] >> (4 * (dim & 1)) & 15;
                o += p[j] * h2f(*(const uint16_t *) (strip + cache_v_scale(token, dim / 32, HD))) * (float) (code - 8);
            }
    }
    __syncthreads();
    if (part < PARTS) acc[part][dim] = o;
    __syncthreads();
    if (tid >= HD) return;
    float sum = 0.0f;
    for (int i = 0; i < PARTS; i++) sum += acc[i][tid];
    ((T *) a.out)[row * a.ldo + (int64_t) head * HD + tid] = (T) (l == 0.0f ? 0.0f : sum / l);
}

template <typename T, int HD>
hipError_t attend(const cache_attn_args & a, hipStream_t s) {
    cache_attn_args args = a;
    void * p[] = {&args};
    return hipLaunchKernel((const void *) k_cache_attention<T, HD>, dim3((unsigned) a.n_rows, (unsigned) a.n_head), dim3(256), p, 0, s);
}

template <typename T>
hipError_t by_head(int hd, const cache_attn_args & a, hipStream_t s) {
    return hd == 32 ? attend<T, 32>(a, s) : hd == 64 ? attend<T, 64>(a, s) : hd == 96 ? attend<T, 96>(a, s) : attend<T, 128>(a, s);
}

}  // namespace

int64_t cache_attention_work_bytes(const cache_shape &, int64_t, int64_t, int64_t) { return 16; }

hipError_t launch_cache_attention(const cache_shape & c, int type, const cache_attn_args & a, hipStream_t s) {
    return type == T_F32 ? by_head<float>(c.hd, a, s) : type == T_F16 ? by_head<_Float16>(c.hd, a, s) : by_head<__bf16>(c.hd, a, s);
}
