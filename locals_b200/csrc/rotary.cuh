// Rotary positions, shared by the rotation of queries and keys (rotary.cu) and by the cache write (kv4_store.cu).
//
// Pair j of a head's rot / 2 pairs of dimensions, (a, b) -> (a c - b s, b c + a s) with c, s = cos, sin of the token's
// position on axis axes[j] times the pair's frequency, read from tables of 32-bit values (rows: positions). Pairs are
// (j, j + rot / 2) or, interleaved, (2 j, 2 j + 1); dimensions from rot on are copied. The products and their
// difference or sum are rounded separately in 32 bits (no fused multiply-add), so that a rotation rounds as the formula
// written out in 32-bit operations does, and once more when the result is stored.
#pragma once

#include <stdint.h>

#include <type_traits>

#include "lq_ptx.cuh"
#include "lq_status.cuh"

namespace lq {

struct RotArgs {
    const int32_t* positions;  // (naxes, N); null: nothing is rotated
    const float* cos;          // (max_pos, rot / 2)
    const float* sin;
    const int32_t* axes;  // (rot / 2) axis of each pair; null: every pair on axis 0
    int N, D, rot, max_pos, naxes, interleaved;
};

// A CTA's tokens n0 .. n0 + count - 1: cos and sin of each pair into shared memory (count x rot / 2 floats each), one
// table read a thread and pair whatever the axes' order, for all the rows that the CTA then rotates. An axis or position
// outside the tables is recorded and moved to the nearest.
__device__ __forceinline__ void rot_stage(const RotArgs& r, int n0, int count, float* c, float* s) {
    const int half = r.rot >> 1;
    for (int i = threadIdx.x; i < count * half; i += blockDim.x) {
        const int t = i / half, j = i - t * half;
        int axis = r.axes ? r.axes[j] : 0;
        if (unsigned(axis) >= unsigned(r.naxes)) {
            record_status(LQ_DEV_BOUNDS);
            axis = 0;
        }
        int p = r.positions[size_t(axis) * r.N + n0 + t];
        if (unsigned(p) >= unsigned(r.max_pos)) {
            record_status(LQ_DEV_BOUNDS);
            p = p < 0 ? 0 : r.max_pos - 1;
        }
        c[i] = r.cos[size_t(p) * half + j];
        s[i] = r.sin[size_t(p) * half + j];
    }
    __syncthreads();
}

// P (2, 4, 8: from a multiple of 4 P bytes, or 1) staged values.
template <int P>
__device__ __forceinline__ void rot_staged(const float* from, float (&x)[P]) {
    if constexpr (P % 4 == 0) {
#pragma unroll
        for (int i = 0; i < P; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(from + i);
            x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < P; ++i) x[i] = from[i];
    }
}

__device__ __forceinline__ void rot_pair(float& a, float& b, float c, float s) {
    const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
    b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
    a = x;
}

// V values of T (V = 1, 2, 4, 8) as one load or store, converted in pairs.
template <typename T, int V>
struct RotVec {
    uint32_t w[(V + 1) / 2];
    __device__ __forceinline__ void load(const uint16_t* p) {
        if constexpr (V == 8) {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else if constexpr (V == 4) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            w[0] = v.x, w[1] = v.y;
        } else if constexpr (V == 2) {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        } else {
            w[0] = *p;
        }
    }
    __device__ __forceinline__ void store(uint16_t* p) const {
        if constexpr (V == 8)
            *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        else if constexpr (V == 4)
            *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        else if constexpr (V == 2)
            *reinterpret_cast<uint32_t*>(p) = w[0];
        else
            *p = uint16_t(w[0]);
    }
    __device__ __forceinline__ void get(float (&x)[V]) const {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if constexpr (std::is_same<T, __nv_bfloat16>::value)  // bf16: the upper half of a float
                x[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
            else
                x[i] = F16Traits<T>::to_f32(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu);
        }
    }
    __device__ __forceinline__ void set(const float (&x)[V]) {
        if constexpr (V == 1) {
            w[0] = F16Traits<T>::from_f32(x[0]);
        } else {
#pragma unroll
            for (int i = 0; i < V; i += 2) w[i / 2] = F16Traits<T>::pack2(x[i + 1], x[i]);
        }
    }
};

// Unit u of up to R rows of a token (src, dst: the first row; rows lie D values apart): V values and, where pairs are
// halves, the V of their partners half a rotation further; or, past the rotated dimensions, V values copied. The rows'
// loads are issued together; cs, sn: the token's staged cos and sin, read once for the rows.
template <typename T, int V, int R, bool PAIRS2>
__device__ __forceinline__ void rot_rows(const RotArgs& r, const uint16_t* src, uint16_t* dst, int rows, int u,
                                         const float* cs, const float* sn) {
    const int half = r.rot >> 1;
    int at;
    bool turned;
    if (PAIRS2) {
        at = u * V;
        turned = at < r.rot;
    } else {
        turned = u * V < half;
        at = turned ? u * V : r.rot + (u * V - half);
    }
    src += at;
    dst += at;
    RotVec<T, V> lo[R], hi[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (i >= rows) continue;
        lo[i].load(src + i * r.D);
        if (!PAIRS2 && turned) hi[i].load(src + i * r.D + half);
    }
    if (turned) {
        constexpr int P = PAIRS2 ? V / 2 : V;
        float c[P], s[P];
        rot_staged(cs + (PAIRS2 ? at / 2 : at), c);
        rot_staged(sn + (PAIRS2 ? at / 2 : at), s);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (i >= rows) continue;
            float x[V];
            lo[i].get(x);
            if constexpr (PAIRS2) {
#pragma unroll
                for (int j = 0; j < P; ++j) rot_pair(x[2 * j], x[2 * j + 1], c[j], s[j]);
            } else {
                float y[V];
                hi[i].get(y);
#pragma unroll
                for (int j = 0; j < P; ++j) rot_pair(x[j], y[j], c[j], s[j]);
                hi[i].set(y);
            }
            lo[i].set(x);
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (i >= rows) continue;
        lo[i].store(dst + i * r.D);
        if (!PAIRS2 && turned) hi[i].store(dst + i * r.D + half);
    }
}

}  // namespace lq
