// What the two attention kernels over the paged 4-bit cache share (kv4_attend.cu: few rows a request; kv4_prefill.cu:
// many): arguments, a request's place in the step, and the joining of parts.
#pragma once

#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "kv4.cuh"
#include "lq_host.h"
#include "lq_ptx.cuh"
#include "lq_status.cuh"

namespace lq {

constexpr float KV4_LOG2E = 1.4426950408889634f;
constexpr uint32_t KV4_NONE = 0xffffffffu;  // no page

struct Kv4AttArgs {
    Kv4Pool pool;
    const uint16_t* q;
    const int32_t* q_start;  // may be null: query b is request b's
    const int32_t* table;
    const int32_t* lens;
    const float* sinks;
    uint16_t* out;
    float* part_ml;    // (CTA, 2, rows) x {m, l}, base 2
    float* part_o;     // (CTA, 2, rows) x D
    int32_t* records;  // (CTA) x 8: the item that the start of a CTA's share divides
    uint8_t* dense;    // (request, kv head, dense_steps) x {keys, values} of a step as fp16 tiles (kv4_prefill's dense form)
    int8_t* dense_keys;  // powers of two of the keys' values and of the keys, where those of a step differ widely
    int2* dense_meta;  // their keys' and values' powers of two, and the runs of 8 keys without a page
    int dense_steps;
    float scale_log2;
    int N, B, H, G, width, window, max_q;
    int split_rows;  // requests of more rows are kv4_prefill's
};

// A sink's logit in base 2, finite at its upper end so that differences from it stay numbers. (A NaN stays one.)
__device__ __forceinline__ float kv4_sink(const float* sinks, int head) {
    const float s = sinks ? sinks[head] * KV4_LOG2E : -INFINITY;
    return s > 3.4028234e38f ? 3.4028234e38f : s;
}
__device__ __forceinline__ float kv4_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}

// A request's place in the step: its queries' first row, their number, its keys and the 128-key steps that they span.
struct Kv4Req {
    int first, fresh, len, s_lo, s_hi;
    __device__ __forceinline__ int steps() const { return s_hi - s_lo; }
};

// Rows that request b names, within the queries.
__device__ __forceinline__ void kv4_rows_of(const Kv4AttArgs& a, int b, int* from, int* to) {
    *from = min(max(a.q_start[b], 0), a.N);
    *to = max(min(a.q_start[b + 1], a.N), *from);
}

// first, fresh and len only. Of more than max_q queries (or of ones beyond the query rows) the first are kept, where they
// stand: len then ends with the last that is kept.
__device__ __forceinline__ Kv4Req kv4_new(const Kv4AttArgs& a, int b) {
    Kv4Req r;
    r.first = b;
    r.fresh = b < a.N ? 1 : 0;
    r.len = max(a.lens[b], 0);
    if (a.q_start) {
        int to;
        kv4_rows_of(a, b, &r.first, &to);
        r.fresh = min(to - r.first, a.max_q);
        const int named = max(max(a.q_start[b + 1], 0) - r.first, 0);
        if (named > r.fresh) {
            record_status(LQ_DEV_BOUNDS);
            r.len -= named - r.fresh;
        }
    }
    return r;
}

// Rows that no request's queries are: before the first, past the last, and beyond a request's max_q. They are 0 (the CTAs
// share them).
__device__ __forceinline__ void kv4_zero_rest(const Kv4AttArgs& a, int D) {
    if (!a.q_start) return;
    const long long row = (long long)a.H * D / 8;  // 16-byte pieces a token
    const long long tid = (long long)blockIdx.x * blockDim.x + threadIdx.x, threads = (long long)gridDim.x * blockDim.x;
    auto zero = [&](int from, int to, long long first, long long step) {
        for (long long i = from * row + first; i < to * row; i += step) reinterpret_cast<uint4*>(a.out)[i] = make_uint4(0, 0, 0, 0);
    };
    zero(0, min(max(a.q_start[0], 0), a.N), tid, threads);
    zero(max(min(a.q_start[a.B], a.N), 0), a.N, tid, threads);
    const int lane = threadIdx.x & 31;
    for (long long b0 = tid & ~31LL; b0 < a.B; b0 += threads) {  // a warp 32 requests
        int from = 0, to = 0;
        if (b0 + lane < a.B) kv4_rows_of(a, int(b0) + lane, &from, &to);
        for (uint32_t more = __ballot_sync(0xffffffffu, to - from > a.max_q); more; more &= more - 1)
            zero(__shfl_sync(0xffffffffu, from, __ffs(more) - 1) + a.max_q, __shfl_sync(0xffffffffu, to, __ffs(more) - 1), lane, 32);
    }
}

// The CTA that the x-th of S steps falls to: CTA i of n has steps i S / n .. (i + 1) S / n - 1.
__device__ __forceinline__ int kv4_owner(long long x, long long S, int n) { return int(((x + 1) * n - 1) / S); }

// A row's softmax parts (m, l, O; base 2) with its sink: T(O / L), 0 where nothing was seen.
template <typename T>
__device__ __forceinline__ uint16_t kv4_finish(float m, float l, float o, float sink) {
    const float M = fmaxf(m, sink);
    if (M == -INFINITY) return F16Traits<T>::from_f32(l != l ? l : 0.0f);
    const float f = kv4_ex2(m - M), L = l * f + kv4_ex2(sink - M);
    return F16Traits<T>::from_f32(L == 0.0f ? 0.0f : o * f / L);
}

// The parts of row j that CTAs c0 .. c1 hold (R rows a part; c0's is its second, the others' their first), joined by W
// warps (this one: `warp`): each sums every W-th part, four at a time, a lane 4 dimensions, and the first adds them up in
// order. sum, sml: W x D / 4 and W of shared memory (W = 1: unused).
template <typename T, int D, int W>
__device__ __forceinline__ void kv4_join_row(const Kv4AttArgs& a, int R, int j, int c0, int c1, int warp, float sink, uint16_t* out,
                                             float4 (*sum)[D / 4], float4* sml) {
    constexpr int V = (D + 127) / 128;  // float4s a lane (D = 64: half the lanes)
    const int lane = threadIdx.x & 31;
    const bool in = lane * 4 < D;
    auto part = [&](int cta) { return ((size_t)cta * 2 + (cta == c0 ? 1 : 0)) * R + j; };
    float M = -INFINITY;
    for (int p = c0 + lane; p <= c1; p += 32) M = fmaxf(M, a.part_ml[2 * part(p)]);
#pragma unroll
    for (int d = 16; d; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
    float4 O[V];
    float L = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) O[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int p0 = c0 + warp; p0 <= c1; p0 += 4 * W) {
        float2 ml[4];
        float4 o[4][V];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int p = p0 + k * W;
            ml[k] = make_float2(-INFINITY, 0.0f);
#pragma unroll
            for (int v = 0; v < V; ++v) o[k][v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (p <= c1) {
                const size_t at = part(p);
                ml[k] = *reinterpret_cast<const float2*>(a.part_ml + 2 * at);
                if (in) {
#pragma unroll
                    for (int v = 0; v < V; ++v) o[k][v] = *reinterpret_cast<const float4*>(a.part_o + at * D + v * 128 + lane * 4);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float f = ml[k].x == -INFINITY ? 0.0f : kv4_ex2(ml[k].x - M);
            L += ml[k].y == 0.0f ? 0.0f : ml[k].y * (ml[k].x == -INFINITY ? 1.0f : f);  // (l without an m is a NaN's)
            if (f == 0.0f) continue;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                O[v].x = fmaf(o[k][v].x, f, O[v].x), O[v].y = fmaf(o[k][v].y, f, O[v].y);
                O[v].z = fmaf(o[k][v].z, f, O[v].z), O[v].w = fmaf(o[k][v].w, f, O[v].w);
            }
        }
    }
    if constexpr (W > 1) {
        if (in) {
#pragma unroll
            for (int v = 0; v < V; ++v) sum[warp][v * 32 + lane] = O[v];
        }
        if (lane == 0) sml[warp].x = L;
        __syncthreads();
        if (warp) return;
#pragma unroll
        for (int w = 1; w < W; ++w) {
            L += sml[w].x;
            if (in) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float4 x = sum[w][v * 32 + lane];
                    O[v].x += x.x, O[v].y += x.y, O[v].z += x.z, O[v].w += x.w;
                }
            }
        }
    }
    if (!in) return;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const uint32_t lo = kv4_finish<T>(M, L, O[v].x, sink) | uint32_t(kv4_finish<T>(M, L, O[v].y, sink)) << 16;
        const uint32_t hi = kv4_finish<T>(M, L, O[v].z, sink) | uint32_t(kv4_finish<T>(M, L, O[v].w, sink)) << 16;
        *reinterpret_cast<uint2*>(out + v * 128 + lane * 4) = make_uint2(lo, hi);
    }
}

// The shared-memory limit is an attribute of the function on a device: set at the kernel's first launch on each (`set`
// has a bit a device), not at every launch, where it costs about as much as a small launch itself.
template <typename K, typename A>
static int kv4_launch(K kern, std::atomic<uint32_t>& set, dim3 grid, dim3 block, size_t smem, cudaStream_t st, const A& a,
                      int cluster = 1) {
    if (smem > 48 * 1024) {
        const uint32_t bit = 1u << (device_info().device & 31);
        if (!(set.load(std::memory_order_relaxed) & bit)) {
            if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) != cudaSuccess)
                return LQ_E_CUDA;
            set.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, a) == cudaSuccess ? LQ_OK : LQ_E_CUDA;
}

}  // namespace lq
