// Writing and reading back the paged 4-bit cache (layout: kv4.cuh).
//
// append: a step's queries and keys rotated (rotary.cuh), keys and values quantized to 4 bits and stored in their slots,
// in one launch. The rotated keys are quantized from their 32-bit values, never rounded in between. Quantization is the
// MLX affine algorithm of quant.cu, a group of 64 in the registers of 8 lanes (8 values each): minimum and maximum by
// three shuffles each, scale and bias as there from exact 32-bit operations, codes from the 32-bit scale and bias, both
// then rounded to the activation dtype. A lane's 8 codes are one word. A token whose slot is negative is padding and
// stores nothing; a slot outside the pool is recorded and stores nothing.
// CTAs [0, q_blocks) rotate queries, the others write the cache. HBM-bound: q 4 bytes a value, k and v 2 bytes read and
// 0.5625 written.
//
// read: the values that the cache holds at given slots (zeros for a negative slot), T(scale * code + bias).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kv4.cuh"
#include "lq_host.h"
#include "rotary.cuh"

namespace lq {

constexpr int ST_THREADS = 256;

struct StoreArgs {
    RotArgs r;
    Kv4Pool pool;
    const uint16_t* q;
    uint16_t* qo;
    const uint16_t* k;
    const uint16_t* v;
    const int32_t* slots;
    long long q_row, k_row, v_row;
    int H, q_blocks;
};

// cos and sin for the 8 dimensions d0 .. d0 + 7 of token n (rotated: d0 < rot): c, s of each dimension's pair.
__device__ __forceinline__ void st_cos_sin(const RotArgs& r, int n, int d0, float (&c)[8], float (&s)[8]) {
    if (r.interleaved) {
        float c4[4], s4[4];
        rot_cos_sin<4>(r, n, d0 >> 1, c4, s4);
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = c4[i >> 1], s[i] = s4[i >> 1];
    } else {
        const int half = r.rot >> 1;
        rot_cos_sin<8>(r, n, d0 < half ? d0 : d0 - half, c, s);
    }
}

// x (8 dimensions from d0 of a row whose lanes are this warp's 8-dimension pieces) rotated in 32 bits. Every lane of
// the warp takes part; `live` lanes hold a row.
template <typename T>
__device__ __forceinline__ void st_rotate(const RotArgs& r, const RotVec<T, 8>& w, int n, int d0, bool live,
                                          float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = w.get(i);
    if (!r.positions) return;
    float c[8], s[8];
    const bool turned = live && d0 < r.rot;
    if (turned) st_cos_sin(r, n, d0, c, s);
    if (r.interleaved) {
        if (turned) {
#pragma unroll
            for (int i = 0; i < 8; i += 2) rot_pair(x[i], x[i + 1], c[i], s[i]);
        }
        return;
    }
    // halves: the partner's 8 dimensions sit rot / 16 lanes away
    const int half = r.rot >> 1, lane = threadIdx.x & 31;
    const bool first = d0 < half;
    const int from = turned ? (first ? lane + (half >> 3) : lane - (half >> 3)) : lane;
    float y[8];
    const uint32_t* p = reinterpret_cast<const uint32_t*>(w.h);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t u = __shfl_sync(0xffffffffu, p[i], from);
        y[2 * i] = F16Traits<T>::to_f32(u & 0xffffu);
        y[2 * i + 1] = F16Traits<T>::to_f32(u >> 16);
    }
    if (turned) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (first)
                rot_pair(x[i], y[i], c[i], s[i]);
            else
                rot_pair(y[i], x[i], c[i], s[i]);
        }
    }
}

// 8 values of a group of 64 held by 8 neighbouring lanes -> the lane's word of codes, and the group's scale and bias.
__device__ __forceinline__ uint32_t st_quantize(const float (&x)[8], float* scale_out, float* bias_out) {
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) lo = fminf(lo, x[i]), hi = fmaxf(hi, x[i]);
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
    }
    const bool neg = fabsf(lo) > fabsf(hi);
    float scale = fmaxf(__fdiv_rn(hi - lo, 15.0f), 1e-7f);
    scale = neg ? scale : -scale;
    const float edge = neg ? lo : hi;
    const float q0 = rintf(__fdiv_rn(edge, scale));
    float bias = 0.0f;
    if (q0 != 0.0f) {
        scale = __fdiv_rn(edge, q0);
        bias = edge;
    }
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float q = fminf(fmaxf(rintf(__fdiv_rn(x[i] - bias, scale)), 0.0f), 15.0f);
        word |= uint32_t(q) << (4 * i);
    }
    *scale_out = scale;
    *bias_out = bias;
    return word;
}

template <typename T, int D>
__global__ void __launch_bounds__(ST_THREADS) kv4_append_kernel(const StoreArgs a) {
    constexpr int L = D / 8;  // lanes a row
    grid_dep_wait();
    const int sub = threadIdx.x % L, d0 = sub * 8;
    if (int(blockIdx.x) < a.q_blocks) {
        const long long row = (long long)blockIdx.x * (ST_THREADS / L) + threadIdx.x / L;
        const bool live = row < (long long)a.r.N * a.H;
        const int n = live ? int(row / a.H) : 0, h = live ? int(row % a.H) : 0;
        RotVec<T, 8> w = {};
        if (live) w.load(a.q + n * a.q_row + (long long)h * D + d0);
        float x[8];
        st_rotate<T>(a.r, w, n, d0, live, x);
        if (live) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w.set(i, x[i]);
            w.store(a.qo + row * D + d0);
        }
        return;
    }
    const int KVH = a.pool.KVH;
    const long long row = (long long)(blockIdx.x - a.q_blocks) * (ST_THREADS / L) + threadIdx.x / L;
    const bool live = row < (long long)a.r.N * KVH;
    const int n = live ? int(row / KVH) : 0, h = live ? int(row % KVH) : 0;
    RotVec<T, 8> wk = {}, wv = {};
    int slot = -1;
    if (live) {
        slot = a.slots[n];
        wk.load(a.k + n * a.k_row + (long long)h * D + d0);
        wv.load(a.v + n * a.v_row + (long long)h * D + d0);
    }
    float x[8], ks, kb, vs, vb;
    st_rotate<T>(a.r, wk, n, d0, live, x);
    const uint32_t kw = st_quantize(x, &ks, &kb);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = wv.get(i);
    const uint32_t vw = st_quantize(x, &vs, &vb);
    if (slot < 0) return;
    const int id = slot / a.pool.page;
    if (id >= a.pool.pages) {
        record_status(LQ_DEV_BOUNDS);
        return;
    }
    const size_t at = kv4_row(a.pool, id, h, slot - id * a.pool.page);
    a.pool.kq[at * L + sub] = kw;
    a.pool.vq[at * L + sub] = vw;
    if (sub % 8 == 0) {
        const size_t g = at * (D / 64) + sub / 8;
        a.pool.ks[g] = F16Traits<T>::from_f32(ks);
        a.pool.kb[g] = F16Traits<T>::from_f32(kb);
        a.pool.vs[g] = F16Traits<T>::from_f32(vs);
        a.pool.vb[g] = F16Traits<T>::from_f32(vb);
    }
}

struct ReadArgs {
    Kv4Pool pool;
    const int32_t* slots;
    uint16_t* ko;
    uint16_t* vo;
    int N;
};

template <typename T, int D>
__global__ void __launch_bounds__(ST_THREADS) kv4_read_kernel(const ReadArgs a) {
    constexpr int L = D / 8;
    grid_dep_wait();
    const int sub = threadIdx.x % L, KVH = a.pool.KVH;
    const long long row = (long long)blockIdx.x * (ST_THREADS / L) + threadIdx.x / L;
    if (row >= (long long)a.N * KVH) return;
    const int n = int(row / KVH), h = int(row % KVH);
    const int slot = a.slots[n];
    RotVec<T, 8> k = {}, v = {};
    const int id = slot < 0 ? -1 : slot / a.pool.page;
    if (id >= a.pool.pages) record_status(LQ_DEV_BOUNDS);
    if (id >= 0 && id < a.pool.pages) {
        const size_t at = kv4_row(a.pool, id, h, slot - id * a.pool.page);
        const size_t g = at * (D / 64) + sub / 8;
        const uint32_t kw = a.pool.kq[at * L + sub], vw = a.pool.vq[at * L + sub];
        const float ks = F16Traits<T>::to_f32(a.pool.ks[g]), kb = F16Traits<T>::to_f32(a.pool.kb[g]);
        const float vs = F16Traits<T>::to_f32(a.pool.vs[g]), vb = F16Traits<T>::to_f32(a.pool.vb[g]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            k.set(i, fmaf(ks, float((kw >> (4 * i)) & 15u), kb));
            v.set(i, fmaf(vs, float((vw >> (4 * i)) & 15u), vb));
        }
    }
    k.store(a.ko + row * D + sub * 8);
    v.store(a.vo + row * D + sub * 8);
}

// ---- host ----------------------------------------------------------------------------------------

template <typename K, typename A>
static int st_launch(K kern, long long blocks, cudaStream_t st, const A& a) {
    if (blocks > 0x7fffffffLL) return LQ_E_SHAPE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(blocks));
    cfg.blockDim = dim3(ST_THREADS);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, a) == cudaSuccess ? LQ_OK : LQ_E_CUDA;
}

template <typename T, int D>
static int append_d(StoreArgs& a, cudaStream_t st) {
    const int per = ST_THREADS / (D / 8);  // rows a CTA
    const long long qb = ((long long)a.r.N * a.H + per - 1) / per;
    const long long kvb = ((long long)a.r.N * a.pool.KVH + per - 1) / per;
    if (qb + kvb > 0x7fffffffLL) return LQ_E_SHAPE;
    a.q_blocks = int(qb);
    return st_launch(kv4_append_kernel<T, D>, qb + kvb, st, a);
}

template <typename T>
static int append_t(StoreArgs& a, cudaStream_t st) {
    return a.r.D == 64 ? append_d<T, 64>(a, st) : a.r.D == 128 ? append_d<T, 128>(a, st) : append_d<T, 256>(a, st);
}

bool kv4_pool_ok(const Kv4Pool& p, int D) {
    return p.pages >= 1 && p.KVH >= 1 && p.page >= 8 && p.page % 8 == 0 && p.page <= 65536 &&
           (D == 64 || D == 128 || D == 256) && (unsigned long long)p.pages * p.KVH <= 0xffffffffull / p.page &&
           (unsigned long long)p.pages * p.page <= 0x7fffffffull;
}

int kv4_append_run(const RotArgs& r, const Kv4Pool& pool, const void* q, long long q_row, void* q_out, int H,
                   const void* k, long long k_row, const void* v, long long v_row, const int32_t* slots, int dtype,
                   cudaStream_t st) {
    if (r.N == 0) return LQ_OK;
    StoreArgs a = {};
    a.r = r;
    a.pool = pool;
    a.q = static_cast<const uint16_t*>(q);
    a.qo = static_cast<uint16_t*>(q_out);
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.slots = slots;
    a.q_row = q_row;
    a.k_row = k_row;
    a.v_row = v_row;
    a.H = H;
    return dtype == LQ_BF16 ? append_t<__nv_bfloat16>(a, st) : append_t<__half>(a, st);
}

template <typename T>
static int read_t(const ReadArgs& a, int D, cudaStream_t st) {
    const int per = ST_THREADS / (D / 8);
    const long long blocks = ((long long)a.N * a.pool.KVH + per - 1) / per;
    return D == 64    ? st_launch(kv4_read_kernel<T, 64>, blocks, st, a)
           : D == 128 ? st_launch(kv4_read_kernel<T, 128>, blocks, st, a)
                      : st_launch(kv4_read_kernel<T, 256>, blocks, st, a);
}

int kv4_read_run(const Kv4Pool& pool, int D, const int32_t* slots, int N, void* k_out, void* v_out, int dtype,
                 cudaStream_t st) {
    if (N == 0) return LQ_OK;
    const ReadArgs a = {pool, slots, static_cast<uint16_t*>(k_out), static_cast<uint16_t*>(v_out), N};
    return dtype == LQ_BF16 ? read_t<__nv_bfloat16>(a, D, st) : read_t<__half>(a, D, st);
}

}  // namespace lq
