// Microscaled 4-bit floating point: the format, and the PTX of its block-scaled tensor-core products.
//
// A value is 4 bits (e2m1: sign, 2 exponent bits, 1 mantissa bit; 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), eight
// to a 32-bit word, lowest bits first; rows are filled with zero codes to a multiple of 128 values. Groups along a row share a
// scale byte: "mxfp4" 32 values and 2^(b - 127) (255: not a number), "nvfp4" 16 values and an e4m3 number (127: not a
// number). Scale bytes lie in tiles of 128 rows x 4 groups, 512 bytes, the order in which tcgen05.cp.32x128b takes them to
// tensor memory: byte 16 (r % 32) + 4 (r / 32) + g % 4 of tile (r / 128, g / 4); the tiles of 128 rows follow one another
// along the groups.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/lq.h"
#include "lq_ptx.cuh"

namespace lq {

constexpr int FP4_PAD = 128;  // values a row is filled to a multiple of

__host__ __device__ constexpr int fp4_padded(int K) { return (K + FP4_PAD - 1) / FP4_PAD * FP4_PAD; }
__host__ __device__ constexpr int fp4_group(int mode) { return mode == LQ_MXFP4 ? 32 : 16; }
// 512-byte scale tiles along a row of K values
__host__ __device__ constexpr int fp4_ktiles(int K, int mode) { return fp4_padded(K) / (4 * fp4_group(mode)); }

__host__ __device__ constexpr int fp4_tile_byte(int row, int group) {
    return 16 * (row % 32) + 4 * (row / 32) + group % 4;
}

// Eight floats to a word of e2m1 codes (nearest, ties to even, saturating), the first in the lowest bits.
__device__ __forceinline__ uint32_t codes8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// Two e4m3 bytes to fp16 (exact).
__device__ __forceinline__ float2 e4m3x2_to_f32(uint32_t v) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(v)));
    return __half22float2(*reinterpret_cast<__half2*>(&h));
}

// What a scale byte stands for.
__device__ __forceinline__ float fp4_scale_value(uint32_t b, int mode) {
    if (mode == LQ_MXFP4)  // 2^(b - 127): the exponent field, but for 0 (2^-127 is no normal number) and 255 (not a number)
        return b == 0 ? __uint_as_float(0x00400000u) : b == 255 ? __uint_as_float(0x7FC00000u) : __uint_as_float(b << 23);
    return e4m3x2_to_f32(b).x;
}

// Values [k0, k0 + 8) of a row of K 16-bit values, zeros beyond it; `vec`: the row starts on a 16-byte boundary.
template <typename T16>
__device__ __forceinline__ uint4 load8_16(const T16* row, int k0, int K, bool vec) {
    if (vec && k0 + 8 <= K) return *reinterpret_cast<const uint4*>(row + k0);
    uint32_t w[4] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (k0 + i < K) w[i >> 1] |= uint32_t(reinterpret_cast<const uint16_t*>(row)[k0 + i]) << (16 * (i & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The largest magnitude of 8 values (a number that is none, if one is).
template <typename T2>
__device__ __forceinline__ float amax8_16(const uint4& x) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    T2 m = __habs2(*reinterpret_cast<const T2*>(&w[0]));
#pragma unroll
    for (int i = 1; i < 4; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const T2*>(&w[i])));
    float lo, hi, top;
    if constexpr (std::is_same<T2, __half2>::value) {
        lo = __low2float(m);
        hi = __high2float(m);
    } else {
        const uint32_t b = *reinterpret_cast<uint32_t*>(&m);
        lo = __uint_as_float(b << 16);
        hi = __uint_as_float(b & 0xFFFF0000u);
    }
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(top) : "f"(lo), "f"(hi));
    return top;
}

// The largest magnitude of a and b; not a number if one of them is none.
__device__ __forceinline__ float amax_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Values [k0, k0 + 8) of a row of K, zeros beyond it, as they lie in memory; `vec`: the row starts on a 16-byte boundary.
template <typename T>
struct Eight {
    uint4 q;
    __device__ __forceinline__ void load(const T* row, int k0, int K, bool vec) { q = load8_16(row, k0, K, vec); }
    __device__ __forceinline__ void zero() { q = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ float amax() const {
        return amax8_16<typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type>(q);
    }
    __device__ __forceinline__ void times(float f, float (&v)[8]) const {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = F16Traits<T>::to_f32(w[i] & 0xFFFFu) * f;
            v[2 * i + 1] = F16Traits<T>::to_f32(w[i] >> 16) * f;
        }
    }
};
template <>
struct Eight<float> {
    float x[8];
    __device__ __forceinline__ void load(const float* row, int k0, int K, bool vec) {
        if (vec && k0 + 8 <= K) {
            *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(row + k0);
            *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(row + k0 + 4);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = k0 + i < K ? row[k0 + i] : 0.f;
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 0.f;
    }
    __device__ __forceinline__ float amax() const {
        float m = fabsf(x[0]);
#pragma unroll
        for (int i = 1; i < 8; ++i) m = amax_nan(m, fabsf(x[i]));
        return m;
    }
    __device__ __forceinline__ void times(float f, float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = x[i] * f;
    }
};

// One lane of a whole warp, chosen in a way that the compiler knows to be uniform: tcgen05 and TMA instructions take their
// operands from uniform registers, and behind `lane == 0` each operand is moved there one by one (70 cycles a tcgen05.cp and
// 55 to 70 a small MMA; 20 and 45 behind this).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "elect.sync _|q, 0xFFFFFFFF;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(p));
    return p != 0;
}

// ---- pairs of CTAs ----

// Tiled loads to this CTA's shared memory; `bar` is an address of the cluster's window, in a pair the lower rank's barrier.
template <int CG>
__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1, uint64_t policy) {
    if constexpr (CG == 1)
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
            " [%0], [%1, {%3, %4}], [%2], %5;" ::"r"(dst),
            "l"(m), "r"(bar), "r"(c0), "r"(c1), "l"(policy)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
            " [%0], [%1, {%3, %4}], [%2], %5;" ::"r"(dst),
            "l"(m), "r"(bar), "r"(c0), "r"(c1), "l"(policy)
            : "memory");
}

template <int CG>
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1, int c2, uint64_t policy) {
    if constexpr (CG == 1)
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
            " [%0], [%1, {%3, %4, %5}], [%2], %6;" ::"r"(dst),
            "l"(m), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "l"(policy)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
            " [%0], [%1, {%3, %4, %5}], [%2], %6;" ::"r"(dst),
            "l"(m), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "l"(policy)
            : "memory");
}

// Arrive on the barrier at this offset of another CTA of the cluster.
__device__ __forceinline__ void mbar_arrive_peer(uint64_t* bar, uint32_t rank) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(map_peer(smem_u32(bar), rank)) : "memory");
}

// mbar_wait for a barrier that another CTA of the cluster arrives on.
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity) {
    for (uint32_t i = 0; i < LQ_SPIN_LIMIT; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
        if (ok) return true;
    }
    record_status(LQ_DEV_TIMEOUT);
    return false;
}

template <int CG>
__device__ __forceinline__ bool mbar_wait_cg(uint64_t* bar, uint32_t parity) {
    return CG == 1 ? mbar_wait(bar, parity) : mbar_wait_cluster(bar, parity);
}

// ---- block-scaled tcgen05; CG: CTAs that work on a tile (1, or a pair whose lower rank issues for both) ----

template <int CG>
__device__ __forceinline__ void tc_alloc(uint32_t* dst_smem, uint32_t ncols) {
    if constexpr (CG == 1) {
        tmem_alloc(dst_smem, ncols);
        tmem_relinquish();
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst_smem)), "r"(ncols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}

template <int CG>
__device__ __forceinline__ void tc_dealloc(uint32_t taddr, uint32_t ncols) {
    if constexpr (CG == 1)
        tmem_dealloc(taddr, ncols);
    else
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

// Arrive on `bar` (of both CTAs of a pair) once every tcgen05 operation issued so far has completed.
template <int CG>
__device__ __forceinline__ void tc_commit_all(uint64_t* bar) {
    if constexpr (CG == 1)
        tc_commit(bar);
    else
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
            "h"(uint16_t(3))
            : "memory");
}

// One scale tile (512 bytes of shared memory, rows of 16 bytes) to 4 columns of tensor memory, in all four lane quarters (of
// a pair: in each CTA from its own shared memory).
template <int CG>
__device__ __forceinline__ void tc_copy_scales(uint32_t taddr, uint64_t desc) {
    if constexpr (CG == 1)
        asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
    else
        asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// Shared-memory descriptor of unswizzled 8-row x 16-byte core matrices that follow one another (128 bytes apart).
__device__ __forceinline__ uint64_t umma_desc_scales(uint32_t smem_addr) {
    return uint64_t((smem_addr >> 4) & 0x3FFFu) | (uint64_t(128 >> 4) << 16) | (uint64_t(128 >> 4) << 32) |
           (uint64_t(1) << 46);
}

// The forms of a block-scaled MMA: both operands mxfp4 or both nvfp4 (K = 64 a MMA), or e2m1 (in bytes) by e4m3 (K = 32).
enum { FP4_MX = 0, FP4_NV = 1, FP4_SPLIT = 2 };

// Instruction descriptor: A e2m1, B e2m1 or e4m3, both K-major, M x N tile, the byte of each 32-bit scale word that
// the MMA starts at in bits 4-5 (B) and 29-30 (A), the scales' type in bit 23 (1: powers of two).
template <int KIND>
__host__ __device__ constexpr uint32_t fp4_idesc(int M, int N) {
    return (uint32_t(KIND == FP4_SPLIT ? 5 : 1) << 7) | (uint32_t(KIND == FP4_SPLIT ? 0 : 1) << 10) |
           (uint32_t(N >> 3) << 17) | (uint32_t(KIND == FP4_NV ? 0 : 1) << 23) | (uint32_t(M >> 4) << 24);
}
__host__ __device__ constexpr uint32_t fp4_idesc_byte(int id) { return (uint32_t(id) << 4) | (uint32_t(id) << 29); }

#define LQ_FP4_MMA(CG_, FORM_)                                                                                         \
    asm volatile(                                                                                                       \
        "{\n\t.reg .pred p;\n\t"                                                                                        \
        "setp.ne.b32 p, %6, 0;\n\t"                                                                                     \
        "tcgen05.mma.cta_group::" CG_ ".kind::" FORM_ " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d_tmem),            \
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)                                         \
        : "memory")

template <int KIND, int CG>
__device__ __forceinline__ void tc_mma_fp4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sa,
                                           uint32_t sb, uint32_t accumulate) {
    if constexpr (KIND == FP4_MX && CG == 1) LQ_FP4_MMA("1", "mxf4.block_scale.scale_vec::2X");
    if constexpr (KIND == FP4_MX && CG == 2) LQ_FP4_MMA("2", "mxf4.block_scale.scale_vec::2X");
    if constexpr (KIND == FP4_NV && CG == 1) LQ_FP4_MMA("1", "mxf4nvf4.block_scale.scale_vec::4X");
    if constexpr (KIND == FP4_NV && CG == 2) LQ_FP4_MMA("2", "mxf4nvf4.block_scale.scale_vec::4X");
    if constexpr (KIND == FP4_SPLIT && CG == 1) LQ_FP4_MMA("1", "mxf8f6f4.block_scale.scale_vec::1X");
    if constexpr (KIND == FP4_SPLIT && CG == 2) LQ_FP4_MMA("2", "mxf8f6f4.block_scale.scale_vec::1X");
}
#undef LQ_FP4_MMA

}  // namespace lq
