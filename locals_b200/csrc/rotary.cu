// Rotary positions with several axes on queries and keys (the arithmetic is rotary.cuh's).
//
// A work item is one unit (rot_rows) of R rows of one token, all of them queries or all keys. Items are numbered unit
// fastest, so a warp's accesses run along rows. The vectors are the widest that the sizes, strides and addresses allow,
// 16 bytes where they allow it. cos and sin of a CTA's tokens are staged in shared memory once for all their rows, whatever
// the axes' order. HBM-bound: 4 bytes a value, and the table rows (32-bit values, from L2 after their first use).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "lq_host.h"
#include "rotary.cuh"

namespace lq {

constexpr int ROT_THREADS = 256;

struct RotaryArgs {
    RotArgs r;
    const uint16_t* q;
    uint16_t* qo;
    const uint16_t* k;
    uint16_t* ko;
    long long q_row, k_row;  // values from one token's rows to the next's (inputs; outputs are contiguous)
    int H, KVH;
    unsigned units, q_groups, groups, items;  // units a row, groups of R rows of q and of q and k a token
    int staged;                               // floats of cos (and of sin) in shared memory
};

template <typename T, int V, int R, bool PAIRS2>
__global__ void __launch_bounds__(ROT_THREADS) rotary_kernel(const RotaryArgs a) {
    extern __shared__ __align__(16) float rot_smem[];
    grid_dep_wait();
    const unsigned first = blockIdx.x * ROT_THREADS, item = first + threadIdx.x;
    const unsigned per = a.units * a.groups;  // items a token
    const int n0 = int(first / per), count = int(min(first + ROT_THREADS, a.items) - 1) / int(per) - n0 + 1;
    const int half = a.r.rot >> 1;
    float* sn = rot_smem + a.staged;
    rot_stage(a.r, n0, count, rot_smem, sn);
    if (item >= a.items) return;
    const unsigned n = item / per, rest = item - n * per;
    const int g = int(rest / a.units), unit = int(rest - unsigned(g) * a.units);
    const bool isq = unsigned(g) < a.q_groups;
    const int row = (isq ? g : g - int(a.q_groups)) * R, D = a.r.D, at = (int(n) - n0) * half;
    const uint16_t* src = isq ? a.q + (long long)n * a.q_row : a.k + (long long)n * a.k_row;
    uint16_t* dst = isq ? a.qo + (long long)n * a.H * D : a.ko + (long long)n * a.KVH * D;
    rot_rows<T, V, R, PAIRS2>(a.r, src + row * D, dst + row * D, (isq ? a.H : a.KVH) - row, unit, rot_smem + at, sn + at);
}

template <typename T, int V, int R, bool PAIRS2>
static int rotary_launch(RotaryArgs a, cudaStream_t st) {
    a.q_groups = unsigned(a.H + R - 1) / R;
    a.groups = a.q_groups + unsigned(a.KVH + R - 1) / R;
    const unsigned long long items = (unsigned long long)a.r.N * a.groups * a.units;
    if (items >= 0x7fffff00ull) return LQ_E_SHAPE;
    a.items = unsigned(items);
    const int per = int(a.units * a.groups);  // a CTA's items lie in at most this many tokens
    a.staged = ((ROT_THREADS + per - 2) / per + 1) * (a.r.rot / 2);
    a.staged = (a.staged + 3) / 4 * 4;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned((items + ROT_THREADS - 1) / ROT_THREADS));
    cfg.blockDim = dim3(ROT_THREADS);
    cfg.dynamicSmemBytes = size_t(a.staged) * 2 * sizeof(float);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, rotary_kernel<T, V, R, PAIRS2>, a) == cudaSuccess ? LQ_OK : LQ_E_CUDA;
}

template <typename T, int V>
static int rotary_v(RotaryArgs a, cudaStream_t st) {
    // Four rows a thread once every SM has work for a few CTAs: one read of cos and sin then serves four rows.
    const long long items1 = (long long)a.r.N * (a.H + a.KVH) * a.units;
    const bool many = items1 >= 4LL * device_info().sm_count * 4 * ROT_THREADS;
    if (a.r.interleaved) {
        if constexpr (V >= 2)
            return many ? rotary_launch<T, V, 4, true>(a, st) : rotary_launch<T, V, 1, true>(a, st);
        else
            return LQ_E_ALIGN;
    }
    return many ? rotary_launch<T, V, 4, false>(a, st) : rotary_launch<T, V, 1, false>(a, st);
}

bool rotary_shape_ok(int N, int H, int KVH, int D, int rot, int max_pos, int naxes) {
    return N >= 0 && H >= 0 && KVH >= 0 && H + KVH >= 1 && D >= 2 && D <= 1024 && rot >= 2 && rot % 2 == 0 &&
           rot <= D && max_pos >= 1 && naxes >= 1;
}

int rotary_run(const void* q, long long q_row, void* q_out, int H, const void* k, long long k_row, void* k_out,
               int KVH, int N, int D, int rot, const int32_t* positions, const float* cos, const float* sin,
               int max_pos, const int32_t* axes, int naxes, int interleaved, int dtype, cudaStream_t st) {
    if (N == 0) return LQ_OK;
    RotaryArgs a = {};
    a.r = {positions, cos, sin, axes, N, D, rot, max_pos, naxes, interleaved};
    a.q = static_cast<const uint16_t*>(q);
    a.qo = static_cast<uint16_t*>(q_out);
    a.k = static_cast<const uint16_t*>(k);
    a.ko = static_cast<uint16_t*>(k_out);
    a.q_row = q_row;
    a.k_row = k_row;
    a.H = H;
    a.KVH = KVH;
    // the widest vector that divides every offset: rows, pairs' halves, strides and addresses
    const int half = rot / 2;
    unsigned long long all = (unsigned long long)D | 8ull;
    all |= interleaved ? (unsigned long long)rot : (unsigned long long)half;
    if (H) all |= (unsigned long long)q_row | (reinterpret_cast<uintptr_t>(q) >> 1) | (reinterpret_cast<uintptr_t>(q_out) >> 1);
    if (KVH) all |= (unsigned long long)k_row | (reinterpret_cast<uintptr_t>(k) >> 1) | (reinterpret_cast<uintptr_t>(k_out) >> 1);
    const int V = int(all & (~all + 1));
    a.units = unsigned((interleaved ? D : half + (D - rot)) / V);
    const bool bf = dtype == LQ_BF16;
    switch (V) {
        case 8: return bf ? rotary_v<__nv_bfloat16, 8>(a, st) : rotary_v<__half, 8>(a, st);
        case 4: return bf ? rotary_v<__nv_bfloat16, 4>(a, st) : rotary_v<__half, 4>(a, st);
        case 2: return bf ? rotary_v<__nv_bfloat16, 2>(a, st) : rotary_v<__half, 2>(a, st);
        default: return bf ? rotary_v<__nv_bfloat16, 1>(a, st) : rotary_v<__half, 1>(a, st);
    }
}

}  // namespace lq
