// Block tables and slot maps of one serving step, from the requests' lengths, without a host round trip.
//
// Request b holds cached[b] tokens and brings fresh[b] new ones; a page holds P tokens. With
//   lens = cached + fresh,  q_start = exclusive sum of fresh,  have = ceil(cached / P),  need = ceil(lens / P) - have,
// the pages free[head], free[head + 1], ... are entered into columns have[b] .. have[b] + need[b] - 1 of the requests'
// table rows in request order, and new token i of request b gets position cached[b] + i and slot
// page * P + position % P. The free list itself is only read: the new head is an output.
//
// One launch. Every CTA scans all the lengths for itself (B values, at most 8192: one load a thread and two warp scans
// a 512 requests) and then takes its share of the tokens and of the new pages, each finding its request by a binary
// search of the sums in shared memory; no CTA waits for another. A token whose page is new reads its id from the free
// list, never from the table entry that another CTA may still be writing. Lengths are brought into range where they are
// read (plan_length), and the sums stop at 2^31 - 1, so that no column or position wraps around, whatever the lengths
// hold. What bounds it is latency: the launch, one dependent load of the lengths, the scan, the search and one dependent
// page load. Measured, GPU time of a call among others: 64 requests of one token each 3.5
// us, 200 of up to 512 each 3.9 us.
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "lq_host.h"
#include "lq_ptx.cuh"
#include "lq_status.cuh"

namespace lq {

constexpr int PLAN_THREADS = 512;
constexpr int PLAN_MAX_B = 8192;  // requests: two int arrays of them fit in 64 KB + 8 of shared memory

struct PlanArgs {
    const int32_t* cached;
    const int32_t* fresh;
    int32_t* table;
    const int32_t* free_pages;
    const int32_t* head;
    int32_t* lens;
    int32_t* q_start;
    int32_t* positions;
    int32_t* slots;
    int32_t* head_out;
    int B, width, nfree, page, tokens;
};

constexpr int PLAN_FAR = 0x7fffffff - 65536;  // a request's tokens at most: a page more is still below 2^31

// Request b's cached tokens and new ones (negative: none); those beyond PLAN_FAR in all are left out.
__device__ __forceinline__ void plan_length(const PlanArgs& a, int b, int* cached, int* fresh) {
    const int c = a.cached[b], t = a.fresh[b];
    *cached = min(max(c, 0), PLAN_FAR);
    *fresh = min(max(t, 0), PLAN_FAR - *cached);
    if (c > *cached || t > *fresh) record_status(LQ_DEV_BOUNDS);
}
// a + b of numbers from 0 on, at most 2^31 - 1.
__device__ __forceinline__ int plan_add(int a, int b) { return int(min(unsigned(a) + unsigned(b), 0x7fffffffu)); }

// The last i in [0, n) with a[i] <= x (a ascending, a[0] <= x).
__device__ __forceinline__ int plan_find(const int32_t* a, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(PLAN_THREADS) page_plan_kernel(const PlanArgs a) {
    extern __shared__ int32_t plan_smem[];
    int32_t* tok = plan_smem;            // B + 1 exclusive sums of the new tokens
    int32_t* pag = plan_smem + a.B + 1;  // B + 1 exclusive sums of the new pages
    __shared__ int32_t wt[PLAN_THREADS / 32], wp[PLAN_THREADS / 32];
    grid_dep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int head = *a.head;
    int base_t = 0, base_p = 0;
    for (int b0 = 0; b0 < a.B; b0 += PLAN_THREADS) {
        const int b = b0 + threadIdx.x;
        int t = 0, p = 0;
        if (b < a.B) {
            int c;
            plan_length(a, b, &c, &t);
            p = (c + t + a.page - 1) / a.page - (c + a.page - 1) / a.page;
            if (blockIdx.x == 0) a.lens[b] = c + t;
        }
        int st = t, sp = p;  // inclusive sums within the warp
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int ut = __shfl_up_sync(0xffffffffu, st, d), up = __shfl_up_sync(0xffffffffu, sp, d);
            if (lane >= d) st = plan_add(st, ut), sp = plan_add(sp, up);
        }
        if (lane == 31) wt[warp] = st, wp[warp] = sp;
        __syncthreads();
        int at = base_t, ap = base_p;
        for (int w = 0; w < PLAN_THREADS / 32; ++w) {
            if (w < warp) at = plan_add(at, wt[w]), ap = plan_add(ap, wp[w]);
            base_t = plan_add(base_t, wt[w]);
            base_p = plan_add(base_p, wp[w]);
        }
        st = __shfl_up_sync(0xffffffffu, st, 1), sp = __shfl_up_sync(0xffffffffu, sp, 1);  // exclusive
        if (lane == 0) st = sp = 0;
        if (b < a.B) {
            tok[b] = plan_add(at, st);
            pag[b] = plan_add(ap, sp);
            if (blockIdx.x == 0) a.q_start[b] = tok[b];
        }
        __syncthreads();  // the sums are in place, and wt / wp free for the next round
    }
    grid_dep_launch();
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        a.q_start[a.B] = base_t;
        *a.head_out = head < 0 ? head : plan_add(head, base_p);
        if (base_t > a.tokens || head < 0 || (long long)head + base_p > a.nfree) record_status(LQ_DEV_BOUNDS);
    }
    const unsigned step = gridDim.x * PLAN_THREADS, first = blockIdx.x * PLAN_THREADS + threadIdx.x;
    for (unsigned j = first; j < unsigned(base_p); j += step) {  // the new pages
        const int b = plan_find(pag, a.B, int(j));
        const int col = (min(max(a.cached[b], 0), PLAN_FAR) + a.page - 1) / a.page + int(j) - pag[b];
        const long long f = (long long)head + j;
        if (col >= a.width) {  // on to the next request's
            record_status(LQ_DEV_BOUNDS);
            j += ((b + 1 < a.B ? pag[b + 1] : base_p) - 1 - j) / step * step;
        } else {
            a.table[size_t(b) * a.width + col] = f >= 0 && f < a.nfree ? a.free_pages[f] : -1;
        }
    }
    for (unsigned i = first; i < unsigned(a.tokens); i += step) {  // the new tokens (past the last one: position 0, no slot)
        int pos = 0, slot = -1;
        if (i < unsigned(base_t)) {
            const int b = plan_find(tok, a.B, int(i));
            const int c = min(max(a.cached[b], 0), PLAN_FAR);
            pos = c + (int(i) - tok[b]);
            const int col = pos / a.page, have = (c + a.page - 1) / a.page;
            int id = -1;
            if (col < a.width) {
                if (col < have) {
                    id = a.table[size_t(b) * a.width + col];
                } else {
                    const long long f = (long long)head + pag[b] + (col - have);
                    if (f >= 0 && f < a.nfree) id = a.free_pages[f];
                }
            }
            const int off = pos - col * a.page;
            if (id >= 0 && id <= (0x7fffffff - off) / a.page)  // (an id whose slots are beyond 31 bits is none)
                slot = id * a.page + off;
            else
                record_status(LQ_DEV_BOUNDS);
        }
        a.positions[i] = pos;
        a.slots[i] = slot;
    }
}

bool page_plan_shape_ok(int B, int width, int nfree, int page, int tokens) {
    return B >= 1 && B <= PLAN_MAX_B && width >= 1 && nfree >= 0 && page >= 8 && page % 8 == 0 && page <= 65536 &&
           tokens >= 0;
}

int page_plan_run(const int32_t* cached, const int32_t* fresh, int B, int32_t* table, int width,
                  const int32_t* free_pages, int nfree, const int32_t* head, int page, int tokens, int32_t* lens,
                  int32_t* q_start, int32_t* positions, int32_t* slots, int32_t* head_out, cudaStream_t st) {
    const PlanArgs a = {cached, fresh, table, free_pages, head, lens, q_start, positions, slots, head_out,
                        B, width, nfree, page, tokens};
    // Shared memory beyond the default limit, the static arrays among it: allowed once a device, up to the largest batch, so
    // that a call depends on none before or beside it.
    const size_t smem = size_t(2 * B + 2) * sizeof(int32_t);
    static std::atomic<uint32_t> set{0};
    const uint32_t bit = 1u << (device_info().device & 31);
    if (smem > 32 * 1024 && !(set.load(std::memory_order_relaxed) & bit)) {
        if (cudaFuncSetAttribute(page_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 int((2 * PLAN_MAX_B + 2) * sizeof(int32_t))) != cudaSuccess)
            return LQ_E_CUDA;
        set.fetch_or(bit, std::memory_order_relaxed);
    }
    // one CTA a 512 tokens, at most one a SM (each further CTA scans the lengths again)
    const int ctas = max(1, min((tokens + PLAN_THREADS - 1) / PLAN_THREADS, device_info().sm_count));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(PLAN_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, page_plan_kernel, a) == cudaSuccess ? LQ_OK : LQ_E_CUDA;
}

}  // namespace lq
