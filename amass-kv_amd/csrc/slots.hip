// Block tables and slot maps of a step's new tokens for gfx950 (amass_extend) and the way
// back of finished requests' blocks (amass_release).
//
// A step moves a few KB (12 bytes per token, 8 per new page), so it is bound by its launch
// and its dependent memory rounds: lengths, then the token's table entry or free-list entry,
// then its stores.  One launch does it: every workgroup ranks all requests' new pages
// itself (a block scan over the lengths, which the L2 holds) and finds its tokens' requests
// by bisection in LDS, and a token of a new page computes its block from its rank, so
// nothing waits for the table that the launch writes.  64 requests of one token 2.8 us, 24
// prompts of 34 thousand tokens (0.4 MB) 3.9 us; with four tokens per thread, in turn or side by
// side, these are 2.8 and 6.6, and 4.2 and 6.2: rounds are what costs, not workgroups.
#include "../../include/amass_chunk.h"
#include "common.h"

namespace amass {

constexpr int SL_THREADS = 256;
constexpr int SL_WAVES = SL_THREADS / WAVE;
constexpr int REL_THREADS = 1024;

// exclusive prefix of v over the workgroup's threads; the sum in `total`
template <int WAVES>
__device__ __forceinline__ int block_excl_scan(int v, int* red, int& total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int x = wave_incl_scan(v);
    __syncthreads();
    if (lane == 63) red[w] = x;
    __syncthreads();
    int base = 0, tot = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        const int t = red[i];
        base += i < w ? t : 0;
        tot += t;
    }
    total = tot;
    return base + x - v;
}

__device__ __forceinline__ int pages_of(int len, int sh) {
    return len > 0 ? ((len - 1) >> sh) + 1 : 0;
}

// grid (chunks of SL_THREADS tokens), dynamic LDS: query_start (R+1), lengths (R), new pages
// of the requests before (R).
__global__ __launch_bounds__(SL_THREADS) void extend_kernel(const amass_extend_args a, int sh) {
    extern __shared__ int lds[];
    __shared__ int red[SL_WAVES], top_s;
    int* qs = lds;
    int* len = qs + a.n_req + 1;
    int* before = len + a.n_req;
    const int tid = threadIdx.x;
    if (tid == 0) top_s = min(max(a.top[0], 0), a.capacity);
    for (int r = tid; r <= a.n_req; r += SL_THREADS)
        qs[r] = min(max(a.query_start[r], 0), a.n_tokens);
    for (int r = tid; r < a.n_req; r += SL_THREADS) len[r] = max(a.seq_lens[r], 0);
    int fresh = 0;                       // new pages of the step
    for (int r0 = 0; r0 < a.n_req; r0 += SL_THREADS) {
        __syncthreads();
        const int r = r0 + tid;
        int n = 0;
        if (r < a.n_req) {
            const int q = qs[r + 1] - qs[r];
            if (q > 0)
                n = max(min(pages_of(len[r], sh), a.max_pages) - pages_of(len[r] - q, sh), 0);
        }
        int tot;
        const int ex = block_excl_scan<SL_WAVES>(n, red, tot);
        if (r < a.n_req) before[r] = fresh + ex;
        fresh += tot;
    }
    __syncthreads();
    const int top = top_s;
    // every workgroup reads top[0] before its arrival; the last one may overwrite it (below: the
    // arrival's answer is not waited for here)
    int arrived = blockIdx.x == 0 ? (int)gridDim.x - 1 : 0;
    const bool count = a.top_out == a.top && gridDim.x > 1;
    if (count && tid == 0) arrived = atomicAdd(&a.top[1], 1);
    const int t = blockIdx.x * SL_THREADS + tid;
    // the last request that starts at or before the token
    int r = 0;
    for (int step = a.n_req > 1 ? 1 << (31 - __clz(a.n_req - 1)) : 0; step > 0; step >>= 1)
        if (r + step < a.n_req && qs[r + step] <= t) r += step;
    int pos = -1, blk = -1;
    if (a.n_req > 0 && t >= qs[r] && t < qs[r + 1]) {
        const int start = len[r] - (qs[r + 1] - qs[r]);
        pos = max(start + (t - qs[r]), -1);
        const int p = pos >> sh;
        if (pos >= 0 && p < a.max_pages) {
            int32_t* entry = a.block_table + (int64_t)r * a.bt_st + p;
            const int k = p - pages_of(start, sh), at = top - 1 - (before[r] + k);
            if (k < 0) blk = *entry;
            else if (at >= 0 && at < a.capacity) blk = a.free_list[at];
            if (blk >= a.nb) blk = -1;
            if (k >= 0 && (pos & ((1 << sh) - 1)) == 0) *entry = max(blk, -1);    // its first token
        }
    }
    if (t < a.n_tokens) {
        a.positions[t] = pos;
        a.slots[t] = blk < 0 ? -1 : ((int64_t)blk << sh) + (pos & ((1 << sh) - 1));
    }
    if (tid == 0 && arrived == (int)gridDim.x - 1) {
        if (count) atomicExch(&a.top[1], 0);
        a.top_out[0] = max(top - fresh, 0);
        a.top_out[2] = max(fresh - top, 0);
    }
}

// One workgroup: the pages of the finished requests in order, REL_THREADS at a time.
// Dynamic LDS: pages of the requests before (R+1).
__global__ __launch_bounds__(REL_THREADS) void release_kernel(const amass_release_args a, int sh) {
    extern __shared__ int before[];
    __shared__ int red[REL_THREADS / WAVE];
    const int tid = threadIdx.x;
    int total = 0;
    for (int r0 = 0; r0 < a.n_req; r0 += REL_THREADS) {
        const int r = r0 + tid;
        int n = 0, tot;
        if (r < a.n_req && a.done[r]) n = min(pages_of(a.seq_lens[r], sh), a.max_pages);
        const int ex = block_excl_scan<REL_THREADS / WAVE>(n, red, tot);
        if (r < a.n_req) before[r] = total + ex;
        total += tot;
    }
    if (tid == 0) before[a.n_req] = total;
    __syncthreads();
    const int top = min(max(a.top[0], 0), a.capacity);
    int back = 0;                        // blocks that went back
    for (int i0 = 0; i0 < total; i0 += REL_THREADS) {
        const int i = i0 + tid;
        int32_t* entry = nullptr;
        int blk = -1, tot;
        if (i < total) {
            int lo = 0, hi = a.n_req;    // before[lo] <= i < before[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (before[mid] <= i) lo = mid;
                else hi = mid;
            }
            entry = a.block_table + (int64_t)lo * a.bt_st + (i - before[lo]);
            blk = *entry;
        }
        const bool good = blk >= 0 && blk < a.nb;
        const int at = top + back + block_excl_scan<REL_THREADS / WAVE>(good ? 1 : 0, red, tot);
        if (good && at < a.capacity) a.free_list[at] = blk;
        if (entry) *entry = -1;
        back += tot;
    }
    __syncthreads();
    if (tid == 0) {
        a.top[0] = min(top + back, a.capacity);
        a.top[2] = max(top + back - a.capacity, 0);
    }
}

static int log2_of(int page) {
    int sh = 0;
    while ((1 << sh) < page && sh < 30) ++sh;
    return sh;
}
static bool bad_page(int page) { return page < 1 || (page & (page - 1)) != 0; }

}  // namespace amass

using namespace amass;

extern "C" int amass_extend(const amass_extend_args* a, void* stream) {
    if (!a || !a->top || !a->top_out || !a->query_start || (a->capacity > 0 && !a->free_list) ||
        (a->n_req > 0 && (!a->block_table || !a->seq_lens)) ||
        (a->n_tokens > 0 && (!a->slots || !a->positions)))
        return AMASS_ERR_NULL;
    if (a->n_req < 0 || a->n_tokens < 0 || a->max_pages < 1 || a->nb < 1 || a->capacity < 0 ||
        bad_page(a->page))
        return AMASS_ERR_GEOMETRY;
    if (a->n_req > AMASS_MAX_STEP_REQS) return AMASS_ERR_CAPACITY;
    // a step without tokens or requests still writes top_out and its rows' -1
    const int chunks = a->n_tokens > 0 ? (a->n_tokens - 1) / SL_THREADS + 1 : 1;
    hipLaunchKernelGGL(extend_kernel, dim3(chunks), dim3(SL_THREADS),
                       sizeof(int) * (3 * a->n_req + 1), (hipStream_t)stream, *a,
                       log2_of(a->page));
    return check_launch();
}

extern "C" int amass_release(const amass_release_args* a, void* stream) {
    if (!a || !a->top || (a->capacity > 0 && !a->free_list) ||
        (a->n_req > 0 && (!a->block_table || !a->seq_lens || !a->done)))
        return AMASS_ERR_NULL;
    if (a->n_req < 0 || a->max_pages < 1 || a->nb < 1 || a->capacity < 0 || bad_page(a->page))
        return AMASS_ERR_GEOMETRY;
    if (a->n_req > AMASS_MAX_STEP_REQS) return AMASS_ERR_CAPACITY;
    hipLaunchKernelGGL(release_kernel, dim3(1), dim3(REL_THREADS), sizeof(int) * (a->n_req + 1),
                       (hipStream_t)stream, *a, log2_of(a->page));
    return check_launch();
}
