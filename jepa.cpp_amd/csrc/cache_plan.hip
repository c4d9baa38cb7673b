// cache_plan.hip - the bookkeeping of one step of the paged cache on the GPU: from each sequence's length and the
// tokens that come (or are dropped), its block table, its place in the packed rows, and the cache slot of every row.
//
// The pages that sequence i takes are entries [P(i-1), P(i)) behind the ring's head, P the inclusive sum of the pages
// needed; it is admitted while P(i) fits the free count. Everything is a prefix sum over the sequences and then
// independent work per page and per row, so one workgroup of 16 waves does it: sums in registers and LDS. What it costs is
// latency, one global load after another (256 sequences of one token 5 us; 238k rows of prompts 4.5 and 4.8 us), so the
// thread of a sequence also writes its rows' slots where every sequence has a few; else pages and rows are dealt to all
// threads by a binary search in the sums, and from PLAN_ROWS rows on to a second launch, which finds from what the first
// one wrote which page a row is in.
#include "cache_dev.h"
#include "common.h"
#include "kernels.h"

namespace {

constexpr int NT = 1024;
constexpr int64_t PLAN_ROWS = 4 * NT;      // rows whose pages and slots the first kernel writes itself
constexpr uint32_t FEW = 4;                // rows of a sequence that its own thread writes

// sums over the lanes up to this one, held at 2^32 - 1: within rows of 16 lanes, then across rows
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
#define DPP(ctrl, rows) (uint32_t) __builtin_amdgcn_update_dpp(0, (int) x, ctrl, rows, 0xf, true)
    x = cache_add_sat(x, DPP(0x111, 0xf));      // row_shr 1, 2, 4, 8
    x = cache_add_sat(x, DPP(0x112, 0xf));
    x = cache_add_sat(x, DPP(0x114, 0xf));
    x = cache_add_sat(x, DPP(0x118, 0xf));
    x = cache_add_sat(x, DPP(0x142, 0xa));      // row_bcast 15, 31
    x = cache_add_sat(x, DPP(0x143, 0xc));
#undef DPP
    return x;
}
// entry p of a ring of n behind `head` (both below n, n below 2^31)
__device__ __forceinline__ int32_t ring_at(int32_t head, uint32_t p, int32_t n) {
    const uint32_t i = (uint32_t) head + p;
    return (int32_t) (i >= (uint32_t) n ? i - (uint32_t) n : i);
}

struct plan_view {      // what both kernels do with a row
    const cache_plan_args & a;
    int shift;
    int32_t np;
    __device__ plan_view(const cache_plan_args & args) : a(args), shift(__builtin_ctz((unsigned) args.page_size)), np((int32_t) args.n_pages) {}
    __device__ int64_t slot_of(int32_t page, int32_t pos) const {
        return page < 0 || page >= np ? -1 : ((int64_t) page << shift) + (pos & (a.page_size - 1));
    }
    // the page of position pos of sequence i: a new one from the ring on, if the sequence held `held` and takes from entry `first` on
    __device__ int32_t page_of(int i, int32_t pos, int32_t held, int32_t head, uint32_t first) const {
        const int32_t j = pos >> shift;
        return j >= held ? a.ring[ring_at(head, first + (uint32_t) (j - held), np)] : a.table[(int64_t) i * a.width + j];
    }
};

__global__ __launch_bounds__(NT) void k_cache_plan(cache_plan_args a, bool rows_too) {
    __shared__ uint32_t row_end[CACHE_MAX_SEQ], need_end[CACHE_MAX_SEQ], give_end[CACHE_MAX_SEQ], wsum[3][NT / 64], s_taken;
    __shared__ int32_t held[CACHE_MAX_SEQ];
    const plan_view v(a);
    const int tid = (int) threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int32_t np = v.np;
    int32_t head = a.free_in[0], count = a.free_in[1];
    if (head < 0 || head >= np || count < 0 || count > np) head = count = 0;     // not a ring: nothing to give
    if (tid == 0) s_taken = 0;
    uint32_t total[3] = {0, 0, 0};
    bool many = false;
    for (int base = 0; base < a.n_seq; base += NT) {
        const int i = base + tid;
        cache_seq_step s = {};
        int32_t have = 0;
        if (i < a.n_seq) {
            have = a.len[i];
            s = cache_step_of(have, a.come[i], a.width, a.page_size);
        }
        uint32_t sum[3] = {wave_scan(s.rows), wave_scan(s.need), wave_scan(s.give)};
        __syncthreads();
        if (lane == 63)
            for (int k = 0; k < 3; k++) wsum[k][wv] = sum[k];
        many |= __syncthreads_or(s.rows > FEW) != 0;
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
            const uint32_t end = min(sum[0], (uint32_t) a.n_rows);
            row_end[i] = end;
            need_end[i] = sum[1];
            give_end[i] = sum[2];
            held[i] = s.held;
            if (!refused && s.need > 0) atomicMax(&s_taken, sum[1]);
            const int64_t cap = (int64_t) a.width * a.page_size;
            a.kv_len[i] = refused ? (int32_t) (have < 0 ? 0 : have > cap ? cap : have) : s.len;
            a.row_start[i + 1] = (int32_t) end;
            a.refused[i] = refused;
            if (rows_too && !many) {      // up to here every sequence has few rows: this one's, by its thread
                const uint32_t first = sum[1] - s.need;
                for (uint32_t k = 0; !refused && k < s.need; k++) a.table[(int64_t) i * a.width + s.held + k] = a.ring[ring_at(head, first + k, np)];
                const int64_t r0 = (int64_t) sum[0] - s.rows;
                for (uint32_t k = 0; k < s.rows && r0 + k < a.n_rows; k++)
                    a.slot[r0 + k] = refused ? -1 : v.slot_of(v.page_of(i, have + (int32_t) k, s.held, head, first), have + (int32_t) k);
            }
        }
    }
    if (tid == 0) a.row_start[0] = 0;
    __syncthreads();
    const uint32_t taken = s_taken, given = min(total[2], (uint32_t) (np - count));
    for (uint32_t p = tid; p < total[2]; p += NT) {
        const int i = cache_find(give_end, a.n_seq, p);
        const uint32_t first = i ? give_end[i - 1] : 0u;
        int32_t * t = a.table + (int64_t) i * a.width + held[i] - (give_end[i] - first) + (p - first);
        if (p < given) a.ring[ring_at(head, (uint32_t) count + p, np)] = *t;
        *t = -1;
    }
    if (tid == 0) {
        a.free_out[0] = ring_at(head, taken, np);
        a.free_out[1] = count - (int32_t) taken + (int32_t) given;
    }
    if (!rows_too) return;
    if (many) {
        for (uint32_t p = tid; p < taken; p += NT) {
            const int i = cache_find(need_end, a.n_seq, p);
            const uint32_t first = i ? need_end[i - 1] : 0u;
            a.table[(int64_t) i * a.width + held[i] + (p - first)] = a.ring[ring_at(head, p, np)];
        }
        __syncthreads();
    }
    const int64_t used = a.n_seq ? (int64_t) row_end[a.n_seq - 1] : 0;
    for (int64_t r = many ? tid : used + tid; r < a.n_rows; r += NT) {
        int64_t slot = -1;
        if (r < used) {
            const int i = cache_find(row_end, a.n_seq, (uint32_t) r);
            if (!a.refused[i]) {
                const int32_t pos = a.kv_len[i] - (int32_t) (row_end[i] - r);
                slot = v.slot_of(a.table[(int64_t) i * a.width + (pos >> v.shift)], pos);
            }
        }
        a.slot[r] = slot;
    }
}

// Many rows, after k_cache_plan without them: a row a thread. The pages that each sequence takes and where in the ring follow from
// kv_len, row_start and refused; the first row of a page writes the table's entry.
__global__ __launch_bounds__(256) void k_cache_rows(cache_plan_args a) {
    __shared__ uint32_t need_end[CACHE_MAX_SEQ], wsum[4];
    const plan_view v(a);
    const int tid = (int) threadIdx.x, lane = tid & 63, wv = tid >> 6, per = (a.n_seq + 255) / 256, i0 = min(tid * per, a.n_seq), i1 = min(i0 + per, a.n_seq);
    auto held_of = [&](int i, int32_t & have) {      // pages that an admitted sequence held before
        have = a.kv_len[i] - (a.row_start[i + 1] - a.row_start[i]);
        return (have + a.page_size - 1) >> v.shift;
    };
    uint32_t mine = 0;
    for (int i = i0; i < i1; i++) {
        int32_t have;
        if (!a.refused[i]) mine += (uint32_t) (((a.kv_len[i] + a.page_size - 1) >> v.shift) - held_of(i, have));
        need_end[i] = mine;
    }
    uint32_t before = wave_scan(mine);
    if (lane == 63) wsum[wv] = before;
    __syncthreads();
    before -= mine;
    for (int w = 0; w < wv; w++) before += wsum[w];
    for (int i = i0; i < i1; i++) need_end[i] += before;
    __syncthreads();
    const uint32_t taken = wsum[0] + wsum[1] + wsum[2] + wsum[3];
    const int32_t head = ring_at(a.free_out[0], (uint32_t) v.np - taken, v.np);      // where it was before them
    const int64_t r = (int64_t) blockIdx.x * 256 + tid;
    if (r >= a.n_rows) return;
    const uint32_t * end = (const uint32_t *) a.row_start + 1;
    const int i = cache_find(end, a.n_seq, (uint32_t) r);
    int64_t slot = -1;
    if (i < a.n_seq && !a.refused[i]) {
        int32_t have;
        const int32_t held = held_of(i, have), pos = a.kv_len[i] - (int32_t) (end[i] - r), j = pos >> v.shift;
        const int32_t page = v.page_of(i, pos, held, head, i ? need_end[i - 1] : 0u);
        if (j >= held && (pos & (a.page_size - 1)) == 0) a.table[(int64_t) i * a.width + j] = page;
        slot = v.slot_of(page, pos);
    }
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
    return hipLaunchKernel((const void *) k_cache_rows, dim3((unsigned) ((a.n_rows + 255) / 256)), dim3(256), p, 0, s);
}
