// Writing and reading back the paged 4-bit cache (layout: kv4.cuh).
//
// append: a step's queries and keys rotated (rotary.cuh), keys and values quantized to 4 bits and stored in their slots,
// in one launch. The rotated keys are quantized from their 32-bit values, never rounded in between. Quantization is the
// MLX affine algorithm of quant.cu, a group of 64 in the registers of 8 lanes (8 values each), the groups of two
// heads' keys and values together; scale and bias as there from exact 32-bit operations, codes from the 32-bit scale and
// bias, both then rounded to the activation dtype. A lane's 8 codes are one word. A token whose slot is negative is
// padding and stores nothing; a slot outside the pool is recorded and stores nothing. Some CTAs rotate queries (rot_rows),
// the others write the cache, a lane 8 values of a row. HBM-bound by its bytes (q 4 bytes a value, k and v 2 bytes read and
// 0.5625 written), but the quantization's instructions take longer: 8,191 tokens of 32 + 8 heads of 128 on 3 axes in 42.5 us,
// 2.7 instructions a clock and SM (read of the same: 12.8 us; both together 4.16 TB/s).
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
    int staged;                                   // floats of cos (and of sin) in shared memory
};

// x: the 8 dimensions from d0 of a row whose lanes are this warp's 8-dimension pieces, rotated in 32 bits where `turned`.
// Every lane of the warp takes part.
template <typename T, bool PAIRS2>
__device__ __forceinline__ void st_rotate(const RotArgs& r, const RotVec<T, 8>& w, int d0, bool turned, const float (&c)[8],
                                          const float (&s)[8], float (&x)[8]) {
    w.get(x);
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
    RotVec<T, 8> other;
#pragma unroll
    for (int i = 0; i < 4; ++i) other.w[i] = __shfl_sync(0xffffffffu, w.w[i], from);
    float y[8];
    other.get(y);
    if (turned) {  // a c - b s in the first half, b c + a s in the second
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] = __fadd_rn(__fmul_rn(x[i], c[i]), __fmul_rn(y[i], first ? -s[i] : s[i]));
    }
}

// The scale and bias of a group from its least and largest value, and the scale's reciprocal.
__device__ __forceinline__ void st_scale(float lo, float hi, float* scale_out, float* bias_out, float* inv) {
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
    *scale_out = scale;
    *bias_out = bias;
    *inv = __frcp_rn(scale);
}

// 8 values -> their word of codes round((x - bias) / scale), the division in 32 bits. A product with the reciprocal is
// within 2^-18 of the quotient, so its rounding is the quotient's wherever it lies further than that from a half; only
// there (a few in ten thousand) is the division itself done.
__device__ __forceinline__ uint32_t st_codes(const float (&x)[8], float scale, float bias, float inv) {
    const float magic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to a whole number
    uint32_t word = 0, near = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float t = fminf(fmaxf((x[i] - bias) * inv, 0.0f), 15.0f), u = t + magic;
        if (fabsf(t - (u - magic)) > 0.5f - 1.52587890625e-5f) near |= 1u << i;
        word |= (__float_as_uint(u) & 15u) << (4 * i);
    }
    while (near) {
        const int i = __ffs(near) - 1;
        near &= near - 1;
        float v = x[0];  // x[i] without an indexed register
#pragma unroll
        for (int k = 1; k < 8; ++k) v = k == i ? x[k] : v;
        const float q = fminf(fmaxf(rintf(__fdiv_rn(v - bias, scale)), 0.0f), 15.0f);
        word = (word & ~(15u << (4 * i))) | (uint32_t(q) << (4 * i));
    }
    return word;
}

// Q (2 or 4) groups of 64, 8 values of each in each of 8 neighbouring lanes -> the lane's words of codes. The groups'
// extremes are reduced together, each step of the butterfly leaving a lane half of them, so that lane l ends with one
// group, own(l), whose scale and bias it alone works out (and returns) and the others take from it.
template <int Q>
__device__ __forceinline__ int st_own(int lane) {
    return Q == 4 ? 2 * (lane & 1) + ((lane >> 1) & 1) : lane & 1;
}
template <int Q>
__device__ __forceinline__ void st_quantize(const float (&x)[Q][8], uint32_t (&words)[Q], float* scale_out, float* bias_out) {
    const int lane = threadIdx.x & 31;
    float lo[Q], hi[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        lo[q] = hi[q] = x[q][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) lo[q] = fminf(lo[q], x[q][i]), hi[q] = fmaxf(hi[q], x[q][i]);
    }
#pragma unroll
    for (int n = Q / 2, d = 1; n >= 1; n /= 2, d *= 2) {  // keep the upper or the lower n of 2 n groups
        const bool up = lane & d;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float gl = __shfl_xor_sync(0xffffffffu, up ? lo[i] : lo[n + i], d);
            const float gh = __shfl_xor_sync(0xffffffffu, up ? hi[i] : hi[n + i], d);
            lo[i] = fminf(up ? lo[n + i] : lo[i], gl);
            hi[i] = fmaxf(up ? hi[n + i] : hi[i], gh);
        }
    }
#pragma unroll
    for (int d = Q; d < 8; d <<= 1) {
        lo[0] = fminf(lo[0], __shfl_xor_sync(0xffffffffu, lo[0], d));
        hi[0] = fmaxf(hi[0], __shfl_xor_sync(0xffffffffu, hi[0], d));
    }
    float scale, bias, inv;
    st_scale(lo[0], hi[0], &scale, &bias, &inv);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int from = (lane & ~7) | (Q == 4 ? (q >> 1) | ((q & 1) << 1) : q);
        words[q] = st_codes(x[q], __shfl_sync(0xffffffffu, scale, from), __shfl_sync(0xffffffffu, bias, from),
                            __shfl_sync(0xffffffffu, inv, from));
    }
    *scale_out = scale;
    *bias_out = bias;
}

// RQ query rows a thread, RK kv heads a thread (one read of cos and sin for all of them).
template <typename T, int D, int RQ, int RK, bool PAIRS2>
__global__ void __launch_bounds__(ST_THREADS) kv4_append_kernel(const StoreArgs a) {
    constexpr int L = D / 8;  // lanes a row
    extern __shared__ __align__(16) float st_smem[];
    grid_dep_wait();
    const int half = a.r.rot >> 1;
    float* sn = st_smem + a.staged;
    // query and cache CTAs in turn, as long as there are both: the ones wait for memory, the others compute
    const unsigned kv_blocks = gridDim.x - a.q_blocks, both = 2 * min(a.q_blocks, kv_blocks), b = blockIdx.x;
    const bool is_q = b < both ? b & 1 : a.q_blocks > kv_blocks;
    const unsigned blk = b < both ? b / 2 : b - both / 2;
    if (is_q) {
        const unsigned first = blk * ST_THREADS, item = first + threadIdx.x, per = a.units * a.q_groups;
        const int n0 = int(first / per);
        if (half) rot_stage(a.r, n0, int((min(first + ST_THREADS, a.q_items) - 1) / per) - n0 + 1, st_smem, sn);
        if (item >= a.q_items) return;
        const unsigned n = item / per, rest = item - n * per;
        const int g = int(rest / a.units), unit = int(rest - unsigned(g) * a.units), row = g * RQ;
        const int at = (int(n) - n0) * half;
        rot_rows<T, 8, RQ, PAIRS2>(a.r, a.q + (long long)n * a.q_row + row * D, a.qo + ((long long)n * a.H + row) * D,
                                   a.H - row, unit, st_smem + at, sn + at);
        return;
    }
    const int KVH = a.pool.KVH, sub = threadIdx.x % L, d0 = sub * 8;
    const unsigned first = blk * (ST_THREADS / L), item = first + threadIdx.x / L;
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
    if (half) {
        const int n0 = int(first / a.kv_groups);
        rot_stage(a.r, n0, int((min(first + ST_THREADS / L, a.kv_items) - 1) / a.kv_groups) - n0 + 1, st_smem, sn);
    }
    const bool turned = live && d0 < a.r.rot;
    float c[8], s[8];  // of the dimensions' pairs
    if (turned) {
        const int at = (int(n) - int(first / a.kv_groups)) * half;
        if constexpr (PAIRS2) {
            float c4[4], s4[4];
            rot_staged(st_smem + at + d0 / 2, c4);
            rot_staged(sn + at + d0 / 2, s4);
#pragma unroll
            for (int i = 0; i < 8; ++i) c[i] = c4[i >> 1], s[i] = s4[i >> 1];
        } else {
            rot_staged(st_smem + at + (d0 < half ? d0 : d0 - half), c);
            rot_staged(sn + at + (d0 < half ? d0 : d0 - half), s);
        }
    }
    const int id = slot < 0 ? -1 : slot / a.pool.page;
    if (id >= a.pool.pages) record_status(LQ_DEV_BOUNDS);
    const bool kept = id >= 0 && id < a.pool.pages;
    const size_t at = kept ? kv4_row(a.pool, id, h0, slot - id * a.pool.page) : 0;
    float x[2 * RK][8], scale, bias;  // group 2 i: keys of head i, 2 i + 1: its values
    uint32_t words[2 * RK];
#pragma unroll
    for (int i = 0; i < RK; ++i) {
        st_rotate<T, PAIRS2>(a.r, wk[i], d0, turned, c, s, x[2 * i]);
        wv[i].get(x[2 * i + 1]);
    }
    st_quantize<2 * RK>(x, words, &scale, &bias);
    if (!kept) return;
#pragma unroll
    for (int i = 0; i < RK; ++i) {
        if (h0 + i >= KVH) continue;
        const size_t row = at + size_t(i) * a.pool.page;
        a.pool.kq[row * L + sub] = words[2 * i];
        a.pool.vq[row * L + sub] = words[2 * i + 1];
    }
    const int own = st_own<2 * RK>(threadIdx.x & 31), mine = sub & 7;
    if (mine < 2 * RK && h0 + own / 2 < KVH) {
        const size_t g = (at + size_t(own / 2) * a.pool.page) * (D / 64) + sub / 8;
        (own & 1 ? a.pool.vs : a.pool.ks)[g] = F16Traits<T>::from_f32(scale);
        (own & 1 ? a.pool.vb : a.pool.kb)[g] = F16Traits<T>::from_f32(bias);
    }
}

struct ReadArgs {
    Kv4Pool pool;
    const int32_t* slots;
    uint16_t* ko;
    uint16_t* vo;
    unsigned items;  // (token, kv head)
};

// Code i of a word: as the last bits of 2^23 + code, which a subtraction takes (a conversion runs at a quarter of its rate).
__device__ __forceinline__ float st_code(uint32_t w, int i) {
    return __uint_as_float(0x4b000000u | ((w >> (4 * i)) & 15u)) - 8388608.0f;
}

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
        float x[8], y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = fmaf(ks, st_code(kw, i), kb);
            y[i] = fmaf(vs, st_code(vw, i), vb);
        }
        k.set(x);
        v.set(y);
    }
    k.store(a.ko + row * D + sub * 8);
    v.store(a.vo + row * D + sub * 8);
}

// ---- host ----------------------------------------------------------------------------------------

template <typename K, typename A>
static int st_launch(K kern, long long blocks, cudaStream_t st, const A& a, size_t smem = 0) {
    if (blocks > 0x7fffffffLL) return LQ_E_SHAPE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(blocks));
    cfg.blockDim = dim3(ST_THREADS);
    cfg.dynamicSmemBytes = smem;
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
    // tokens that a CTA's items can lie in, of either part
    const int qp = int(a.units * a.q_groups), kp = int(a.kv_groups);
    const int qt = qp ? (ST_THREADS + qp - 2) / qp + 1 : 0, kt = (per + kp - 2) / kp + 1;
    a.staged = (qt > kt ? qt : kt) * (a.r.rot / 2);
    return st_launch(kv4_append_kernel<T, D, RQ, RK, PAIRS2>, (long long)a.q_blocks + (ki + per - 1) / per, st, a,
                     size_t(a.staged) * 2 * sizeof(float));
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
