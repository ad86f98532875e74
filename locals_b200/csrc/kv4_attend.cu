// Attention of queries over a paged 4-bit cache (layout: kv4.cuh).
//
// Query i of request b stands at position lens[b] - new[b] + i and sees the keys from max(0, position - window + 1)
// (window 0: from 0) to its own: out = sum_j e^(s_j - m) v_j / (sum_j e^(s_j - m) + e^(sink - m)), s_j = scale q . k_j,
// and 0 where nothing is seen.
//
// One CTA a (query, head); each of its warps takes every fourth key with a running maximum and sum of its own, a lane
// holding D / 32 dimensions; the warps are joined in shared memory.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "kv4.cuh"
#include "lq_host.h"
#include "lq_ptx.cuh"
#include "lq_status.cuh"

namespace lq {

constexpr int KV4_NW = 4;
constexpr float KV4_LOG2E = 1.4426950408889634f;

// A sink's logit in base 2, finite at its upper end so that differences from it stay numbers.
__device__ __forceinline__ float kv4_sink(const float* sinks, int head) {
    return sinks ? fminf(sinks[head] * KV4_LOG2E, 3.4028234e38f) : -INFINITY;
}

struct Kv4AttArgs {
    Kv4Pool pool;
    const uint16_t* q;
    const int32_t* q_start;  // may be null: query b is request b's
    const int32_t* table;
    const int32_t* lens;
    const float* sinks;
    uint16_t* out;
    float scale_log2;
    int N, B, H, width, window;
};

template <typename T, int D>
__global__ void __launch_bounds__(KV4_NW * 32) kv4_attend_kernel(const Kv4AttArgs a) {
    constexpr int E = D / 32;  // dimensions a lane
    __shared__ float sm[KV4_NW], sl[KV4_NW], so[KV4_NW][D];
    grid_dep_wait();
    const int n = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint16_t* out = a.out + ((size_t)n * a.H + h) * D;
    int b = n, pos = 0, len = 0;
    bool real = n < a.B;
    if (a.q_start) {
        int lo = 0, hi = a.B;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.q_start[mid] <= n)
                lo = mid;
            else
                hi = mid;
        }
        b = lo;
        real = n < a.q_start[a.B];
    }
    if (real) {
        len = a.lens[b];
        if ((long long)len > (long long)a.width * a.pool.page) {
            record_status(LQ_DEV_BOUNDS);
            len = a.width * a.pool.page;
        }
        pos = a.q_start ? len - (a.q_start[b + 1] - n) : len - 1;
    }
    const int hi = real ? pos + 1 : 0, lo = a.window ? max(0, hi - a.window) : 0;
    const int G = a.H / a.pool.KVH, kvh = h / G;
    float q[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        q[e] = F16Traits<T>::to_f32(a.q[((size_t)n * a.H + h) * D + lane * E + e]) * a.scale_log2;
        o[e] = 0.0f;
    }
    for (int j = lo + warp; j < hi; j += KV4_NW) {
        const int id = a.table[(size_t)b * a.width + j / a.pool.page];
        if (unsigned(id) >= unsigned(a.pool.pages)) {
            record_status(LQ_DEV_BOUNDS);
            continue;
        }
        const size_t row = kv4_row(a.pool, id, kvh, j % a.pool.page);
        const size_t g = row * (D / 64) + lane * E / 64;
        const uint32_t kw = a.pool.kq[row * (D / 8) + lane * E / 8] >> (4 * (lane * E % 8));
        const uint32_t vw = a.pool.vq[row * (D / 8) + lane * E / 8] >> (4 * (lane * E % 8));
        const float ks = F16Traits<T>::to_f32(a.pool.ks[g]), kb = F16Traits<T>::to_f32(a.pool.kb[g]);
        const float vs = F16Traits<T>::to_f32(a.pool.vs[g]), vb = F16Traits<T>::to_f32(a.pool.vb[g]);
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) s = fmaf(q[e], fmaf(ks, float((kw >> (4 * e)) & 15u), kb), s);
#pragma unroll
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        const float mn = fmaxf(m, s);
        const float c = mn == -INFINITY ? 1.0f : exp2f(m - mn), p = mn == -INFINITY ? 0.0f : exp2f(s - mn);
        l = l * c + p;
        m = mn;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(p, fmaf(vs, float((vw >> (4 * e)) & 15u), vb), o[e] * c);
    }
    if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
    for (int e = 0; e < E; ++e) so[warp][lane * E + e] = o[e];
    __syncthreads();
    const float sink = kv4_sink(a.sinks, h);
    float M = sink;
#pragma unroll
    for (int w = 0; w < KV4_NW; ++w) M = fmaxf(M, sm[w]);
    for (int d = threadIdx.x; d < D; d += KV4_NW * 32) {
        float L = sink == -INFINITY || !real ? 0.0f : exp2f(sink - M), O = 0.0f;
#pragma unroll
        for (int w = 0; w < KV4_NW; ++w) {
            const float f = sm[w] == -INFINITY ? 0.0f : exp2f(sm[w] - M);
            L += sl[w] * f;
            O += so[w][d] * f;
        }
        out[d] = F16Traits<T>::from_f32(L > 0.0f ? O / L : (L == L ? 0.0f : L));
    }
}

bool kv4_attend_shape_ok(int N, int B, int max_q, int H, int KVH, int width, int window) {
    return N >= 0 && B >= 1 && max_q >= 1 && H >= 1 && H % KVH == 0 && H <= 65535 && width >= 1 && window >= 0;
}

size_t kv4_attend_workspace_bytes(int N, int B, int max_q, int H, int KVH, int D) { return 0; }

template <typename T, int D>
static int kv4_attend_d(const Kv4AttArgs& a, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.N, a.H);
    cfg.blockDim = dim3(KV4_NW * 32);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv4_attend_kernel<T, D>, a) == cudaSuccess ? LQ_OK : LQ_E_CUDA;
}

template <typename T>
static int kv4_attend_t(const Kv4AttArgs& a, int D, cudaStream_t st) {
    return D == 64 ? kv4_attend_d<T, 64>(a, st) : D == 128 ? kv4_attend_d<T, 128>(a, st) : kv4_attend_d<T, 256>(a, st);
}

int kv4_attend_run(const Kv4Pool& pool, const void* q, int N, const int32_t* q_start, int max_q, const int32_t* table,
                   int width, const int32_t* lens, int B, const float* sinks, float scale, int window, int H, int D,
                   int dtype, void* workspace, size_t workspace_bytes, void* out, cudaStream_t st) {
    if (N == 0) return LQ_OK;
    Kv4AttArgs a = {};
    a.pool = pool;
    a.q = static_cast<const uint16_t*>(q);
    a.q_start = q_start;
    a.table = table;
    a.lens = lens;
    a.sinks = sinks;
    a.out = static_cast<uint16_t*>(out);
    a.scale_log2 = scale * KV4_LOG2E;
    a.N = N;
    a.B = B;
    a.H = H;
    a.width = width;
    a.window = window;
    return dtype == LQ_BF16 ? kv4_attend_t<__nv_bfloat16>(a, D, st) : kv4_attend_t<__half>(a, D, st);
}

}  // namespace lq
