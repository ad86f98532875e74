// Writing and reading back the paged 4-bit cache (layout: kv4.cuh).
//
// append: a step's queries and keys rotated (rotary.cuh), keys and values quantized to 4 bits and stored in their slots,
// in one launch. The rotated keys are quantized from their 32-bit values, never rounded in between. Quantization is the
// MLX affine algorithm of quant.cu, a group of 64 in the registers of 8 lanes (8 values each): minimum and maximum by
// three shuffles each, scale and bias as there from exact 32-bit operations, codes from the 32-bit scale and bias, both
// then rounded to the activation dtype. A lane's 8 codes are one word. A token whose slot is negative is padding and
// stores nothing; a slot outside the pool is recorded and stores nothing.
// CTAs [0, q_blocks) rotate queries (rot_rows), the others write the cache, a lane 8 values of a row. HBM-bound: q 4 bytes a value, k and v 2 bytes read and
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
    int H;
    unsigned q_blocks, q_items, units, q_groups;  // query part: units a row, groups of rows a token
    unsigned kv_items, kv_groups;                 // cache part: (token, group of kv heads)
};

// cos and sin for the 8 dimensions d0 .. d0 + 7 of token n (rotated: d0 < rot): c, s of each dimension's pair.
template <bool PAIRS2>
__device__ __forceinline__ void st_cos_sin(const RotArgs& r, int n, int d0, float (&c)[8], float (&s)[8]) {
    if (PAIRS2) {
        float c4[4], s4[4];
        rot_cos_sin<4>(r, n, d0 >> 1, c4, s4);
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = c4[i >> 1], s[i] = s4[i >> 1];
    } else {
        const int half = r.rot >> 1;
        rot_cos_sin<8>(r, n, d0 < half ? d0 : d0 - half, c, s);
    }
}

// x: the 8 dimensions from d0 of a row whose lanes are this warp's 8-dimension pieces, rotated in 32 bits where `turned`.
// Every lane of the warp takes part.
template <typename T, bool PAIRS2>
__device__ __forceinline__ void st_rotate(const RotArgs& r, const RotVec<T, 8>& w, int d0, bool turned, const float (&c)[8],
                                          const float (&s)[8], float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = w.get(i);
    if (r.rot == 0) return;
    if (PAIRS2) {
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

// RQ query rows a thread, RK kv heads a thread (one read of cos and sin for all of them).
template <typename T, int D, int RQ, int RK, bool PAIRS2>
__global__ void __launch_bounds__(ST_THREADS) kv4_append_kernel(const StoreArgs a) {
    constexpr int L = D / 8;  // lanes a row
    grid_dep_wait();
    if (blockIdx.x < a.q_blocks) {
        const unsigned item = blockIdx.x * ST_THREADS + threadIdx.x;
        if (item >= a.q_items) return;
        const unsigned rest = item / a.units, n = rest / a.q_groups;
        const int unit = int(item - rest * a.units), row = int(rest - n * a.q_groups) * RQ;
        rot_rows<T, 8, RQ, PAIRS2>(a.r, a.q + (long long)n * a.q_row + row * D, a.qo + ((long long)n * a.H + row) * D,
                                   a.H - row, int(n), unit);
        return;
    }
    const int KVH = a.pool.KVH, sub = threadIdx.x % L, d0 = sub * 8;
    const unsigned item = (blockIdx.x - a.q_blocks) * (ST_THREADS / L) + threadIdx.x / L;
    const bool live = item < a.kv_items;
    const unsigned n = live ? item / a.kv_groups : 0;
    const int h0 = live ? int(item - n * a.kv_groups) * RK : 0;
    RotVec<T, 8> wk[RK], wv[RK];
    const int slot = live ? a.slots[n] : -1;
#pragma unroll
    for (int i = 0; i < RK; ++i) {
        wk[i] = wv[i] = RotVec<T, 8>{};
        if (live && h0 + i < KVH) {
            wk[i].load(a.k + (long long)n * a.k_row + (h0 + i) * D + d0);
            wv[i].load(a.v + (long long)n * a.v_row + (h0 + i) * D + d0);
        }
    }
    const bool turned = live && d0 < a.r.rot;
    float c[8], s[8];
    if (turned) st_cos_sin<PAIRS2>(a.r, int(n), d0, c, s);
    const int id = slot < 0 ? -1 : slot / a.pool.page;
    if (id >= a.pool.pages) record_status(LQ_DEV_BOUNDS);
    const bool kept = id >= 0 && id < a.pool.pages;
    const size_t at = kept ? kv4_row(a.pool, id, h0, slot - id * a.pool.page) : 0;
#pragma unroll
    for (int i = 0; i < RK; ++i) {
        float x[8], ks, kb, vs, vb;
        st_rotate<T, PAIRS2>(a.r, wk[i], d0, turned, c, s, x);
        const uint32_t kw = st_quantize(x, &ks, &kb);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = wv[i].get(e);
        const uint32_t vw = st_quantize(x, &vs, &vb);
        if (!kept || h0 + i >= KVH) continue;
        const size_t row = at + size_t(i) * a.pool.page;
        a.pool.kq[row * L + sub] = kw;
        a.pool.vq[row * L + sub] = vw;
        if (sub % 8 == 0) {
            const size_t g = row * (D / 64) + sub / 8;
            a.pool.ks[g] = F16Traits<T>::from_f32(ks);
            a.pool.kb[g] = F16Traits<T>::from_f32(kb);
            a.pool.vs[g] = F16Traits<T>::from_f32(vs);
            a.pool.vb[g] = F16Traits<T>::from_f32(vb);
        }
    }
}

struct ReadArgs {
    Kv4Pool pool;
    const int32_t* slots;
    uint16_t* ko;
    uint16_t* vo;
    unsigned items;  // (token, kv head)
};

template <typename T, int D>
__global__ void __launch_bounds__(ST_THREADS) kv4_read_kernel(const ReadArgs a) {
    constexpr int L = D / 8;
    grid_dep_wait();
    const int sub = threadIdx.x % L, KVH = a.pool.KVH;
    const unsigned item = blockIdx.x * (ST_THREADS / L) + threadIdx.x / L;
    if (item >= a.items) return;
    const unsigned n = item / unsigned(KVH);
    const int h = int(item - n * KVH);
    const size_t row = item;
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

template <typename T, int D, int RQ, int RK, bool PAIRS2>
static int append_r(StoreArgs& a, cudaStream_t st) {
    const int per = ST_THREADS / (D / 8);  // rows a CTA
    a.q_groups = unsigned(a.H + RQ - 1) / RQ;
    a.kv_groups = unsigned(a.pool.KVH + RK - 1) / RK;
    a.units = unsigned(PAIRS2 ? D : D - a.r.rot / 2) / 8;
    const unsigned long long qi = (unsigned long long)a.r.N * a.q_groups * a.units;
    const unsigned long long ki = (unsigned long long)a.r.N * a.kv_groups;
    if (qi >= 0xffffff00ull || ki * (D / 8) >= 0xffffff00ull) return LQ_E_SHAPE;
    a.q_items = unsigned(qi);
    a.kv_items = unsigned(ki);
    a.q_blocks = unsigned((qi + ST_THREADS - 1) / ST_THREADS);
    return st_launch(kv4_append_kernel<T, D, RQ, RK, PAIRS2>, (long long)a.q_blocks + (ki + per - 1) / per, st, a);
}

template <typename T, int D>
static int append_d(StoreArgs& a, cudaStream_t st) {
    // Several rows a thread (one read of cos and sin for all) once one row a thread would be several waves of CTAs.
    const bool many = (long long)a.r.N * (a.H + 2 * a.pool.KVH) * (D / 8) >= 4LL * device_info().sm_count * 8 * ST_THREADS;
    if (a.r.interleaved) return many ? append_r<T, D, 4, 2, true>(a, st) : append_r<T, D, 1, 1, true>(a, st);
    return many ? append_r<T, D, 4, 2, false>(a, st) : append_r<T, D, 1, 1, false>(a, st);
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
    const long long blocks = ((long long)a.items + per - 1) / per;
    return D == 64    ? st_launch(kv4_read_kernel<T, 64>, blocks, st, a)
           : D == 128 ? st_launch(kv4_read_kernel<T, 128>, blocks, st, a)
                      : st_launch(kv4_read_kernel<T, 256>, blocks, st, a);
}

int kv4_read_run(const Kv4Pool& pool, int D, const int32_t* slots, int N, void* k_out, void* v_out, int dtype,
                 cudaStream_t st) {
    if (N == 0) return LQ_OK;
    if ((unsigned long long)N * pool.KVH * (D / 8) >= 0xffffff00ull) return LQ_E_SHAPE;
    const ReadArgs a = {pool, slots, static_cast<uint16_t*>(k_out), static_cast<uint16_t*>(v_out), unsigned(N) * pool.KVH};
    return dtype == LQ_BF16 ? read_t<__nv_bfloat16>(a, D, st) : read_t<__half>(a, D, st);
}

}  // namespace lq
