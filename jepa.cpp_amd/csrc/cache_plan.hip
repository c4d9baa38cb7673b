// cache_plan.hip - the bookkeeping of one step of the paged cache on the GPU: from each sequence's length and the
// tokens that come (or are dropped), its block table, its place in the packed rows, and the cache slot of every row.
//
// The pages that sequence i takes are entries [P(i-1), P(i)) behind the ring's head, P the inclusive sum of the pages
// needed; it is admitted while P(i) fits the free count. Everything is a prefix sum over the sequences and then
// independent work per page and per row, so one workgroup does it: sums in registers and LDS, 16 waves, and pages
// and rows dealt to threads by a binary search in the sums. Rows past PLAN_ROWS are left to a second launch, which
// needs only what the first one wrote.
#include "cache_dev.h"
#include "common.h"
#include "kernels.h"

namespace {

constexpr int NT = 1024;
constexpr int64_t PLAN_ROWS = 16 * NT;      // rows whose slots the first kernel writes itself

__device__ __forceinline__ uint32_t wave_scan(uint32_t x, int lane) {
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = (uint32_t) __shfl_up((int) x, o, 64);
        if (lane >= o) x = cache_add_sat(x, y);
    }
    return x;
}

__device__ __forceinline__ int64_t slot_of(const cache_plan_args & a, int i, int32_t pos) {
    const int32_t page = a.table[(int64_t) i * a.width + pos / a.page_size];
    return page < 0 || page >= a.n_pages ? -1 : (int64_t) page * a.page_size + pos % a.page_size;
}

__global__ __launch_bounds__(NT) void k_cache_plan(cache_plan_args a, bool slots) {
    __shared__ uint32_t row_end[CACHE_MAX_SEQ], need_end[CACHE_MAX_SEQ], give_end[CACHE_MAX_SEQ], wsum[3][NT / 64], s_taken;
    __shared__ int32_t held[CACHE_MAX_SEQ];
    const int tid = (int) threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int32_t np = (int32_t) a.n_pages;
    int32_t head = a.free_in[0], count = a.free_in[1];
    if (head < 0 || head >= np || count < 0 || count > np) head = count = 0;     // not a ring: nothing to give
    if (tid == 0) s_taken = 0;
    uint32_t total[3] = {0, 0, 0};
    for (int base = 0; base < a.n_seq; base += NT) {
        const int i = base + tid;
        cache_seq_step s = {};
        if (i < a.n_seq) s = cache_step_of(a.len[i], a.come[i], a.width, a.page_size);
        uint32_t sum[3] = {wave_scan(s.rows, lane), wave_scan(s.need, lane), wave_scan(s.give, lane)};
        __syncthreads();
        if (lane == 63)
            for (int k = 0; k < 3; k++) wsum[k][wv] = sum[k];
        __syncthreads();
        for (int k = 0; k < 3; k++) {
            uint32_t before = total[k], all = total[k];
            for (int w = 0; w < NT / 64; w++) {
                if (w == wv) before = all;
                all = cache_add_sat(all, wsum[k][w]);
            }
            sum[k] = cache_add_sat(before, sum[k]);
            total[k] = all;
        }
        if (i < a.n_seq) {
            // need that no sequence after the first refusal gets: its sums are past the count for all of them
            const bool refused = s.bad || (s.rows > 0 && sum[0] > (uint32_t) a.n_rows) || (s.need > 0 && sum[1] > (uint32_t) count);
            const int32_t have = a.len[i];
            const int64_t cap = (int64_t) a.width * a.page_size;
            row_end[i] = min(sum[0], (uint32_t) a.n_rows);
            need_end[i] = sum[1];
            give_end[i] = sum[2];
            held[i] = s.held;
            if (!refused && s.need > 0) atomicMax(&s_taken, sum[1]);
            a.kv_len[i] = refused ? (int32_t) (have < 0 ? 0 : have > cap ? cap : have) : s.len;
            a.row_start[i + 1] = (int32_t) row_end[i];
            a.refused[i] = refused;
        }
    }
    if (tid == 0) a.row_start[0] = 0;
    __syncthreads();
    const uint32_t taken = s_taken, given = min(total[2], (uint32_t) (np - count));
    for (uint32_t p = tid; p < taken; p += NT) {
        const int i = cache_find(need_end, a.n_seq, p);
        const uint32_t first = i ? need_end[i - 1] : 0u;
        a.table[(int64_t) i * a.width + held[i] + (p - first)] = a.ring[((int64_t) head + p) % np];
    }
    for (uint32_t p = tid; p < total[2]; p += NT) {
        const int i = cache_find(give_end, a.n_seq, p);
        const uint32_t first = i ? give_end[i - 1] : 0u;
        int32_t * t = a.table + (int64_t) i * a.width + held[i] - (give_end[i] - first) + (p - first);
        if (p < given) a.ring[((int64_t) head + count + p) % np] = *t;
        *t = -1;
    }
    if (tid == 0) {
        a.free_out[0] = (int32_t) (((int64_t) head + taken) % np);
        a.free_out[1] = count - (int32_t) taken + (int32_t) given;
    }
    if (!slots) return;
    __syncthreads();
    for (int64_t r = tid; r < a.n_rows; r += NT) {
        const int i = cache_find(row_end, a.n_seq, (uint32_t) r);
        int64_t slot = -1;
        if (i < a.n_seq && !a.refused[i]) slot = slot_of(a, i, a.kv_len[i] - (int32_t) (row_end[i] - r));
        a.slot[r] = slot;
    }
}

__global__ __launch_bounds__(256) void k_cache_slots(cache_plan_args a) {
    const int64_t r = (int64_t) blockIdx.x * 256 + threadIdx.x;
    if (r >= a.n_rows) return;
    const uint32_t * end = (const uint32_t *) a.row_start + 1;
    const int i = cache_find(end, a.n_seq, (uint32_t) r);
    int64_t slot = -1;
    if (i < a.n_seq && !a.refused[i]) slot = slot_of(a, i, a.kv_len[i] - (int32_t) (end[i] - r));
    a.slot[r] = slot;
}

}  // namespace

// (each launch's own status: hipGetLastError would also report what an earlier call left on the thread)
hipError_t launch_cache_plan(const cache_plan_args & a, hipStream_t s) {
    cache_plan_args args = a;
    bool one = a.n_rows <= PLAN_ROWS;
    void * p[] = {&args, &one};
    const hipError_t e = hipLaunchKernel((const void *) k_cache_plan, dim3(1), dim3(NT), p, 0, s);
    if (e != hipSuccess || one) return e;
    return hipLaunchKernel((const void *) k_cache_slots, dim3((unsigned) ((a.n_rows + 255) / 256)), dim3(256), p, 0, s);
}
