// Rotary positions, shared by the rotation of queries and keys (rotary.cu) and by the cache write (kv4_store.cu).
//
// Pair j of a head's rot / 2 pairs of dimensions, (a, b) -> (a c - b s, b c + a s) with c, s = cos, sin of the token's
// position on axis axes[j] times the pair's frequency, read from tables of 32-bit values (rows: positions). Pairs are
// (j, j + rot / 2) or, interleaved, (2 j, 2 j + 1); dimensions from rot on are copied. The products and their
// difference or sum are rounded separately in 32 bits (no fused multiply-add), so that a rotation rounds as the formula
// written out in 32-bit operations does, and once more when the result is stored.
#pragma once

#include <stdint.h>

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

// The table row of token n on axis `axis`. An axis or position outside the tables is recorded and moved to the nearest.
__device__ __forceinline__ const float* rot_row(const RotArgs& r, const float* table, int n, int axis) {
    if (unsigned(axis) >= unsigned(r.naxes)) {
        record_status(LQ_DEV_BOUNDS);
        axis = 0;
    }
    int p = r.positions[size_t(axis) * r.N + n];
    if (unsigned(p) >= unsigned(r.max_pos)) {
        record_status(LQ_DEV_BOUNDS);
        p = p < 0 ? 0 : r.max_pos - 1;
    }
    return table + size_t(p) * (r.rot >> 1);
}

// cos and sin of pairs j0 .. j0 + P - 1 of token n.
template <int P>
__device__ __forceinline__ void rot_cos_sin(const RotArgs& r, int n, int j0, float (&c)[P], float (&s)[P]) {
    const bool wide = P % 4 == 0 && ((r.rot >> 1) & 3) == 0 && (j0 & 3) == 0 &&
                      ((reinterpret_cast<uintptr_t>(r.cos) | reinterpret_cast<uintptr_t>(r.sin)) & 15) == 0;
    bool one = true;  // every pair on the same axis
    int axis = 0;
    if (r.axes) {
        axis = r.axes[j0];
#pragma unroll
        for (int i = 1; i < P; ++i) one = one && r.axes[j0 + i] == axis;
    }
    if (one) {
        const float *rc = rot_row(r, r.cos, n, axis) + j0, *rs = r.sin + (rc - r.cos);
        if (wide) {
            if constexpr (P % 4 == 0) {
#pragma unroll
                for (int i = 0; i < P; i += 4) {
                    const float4 u = *reinterpret_cast<const float4*>(rc + i);
                    const float4 v = *reinterpret_cast<const float4*>(rs + i);
                    c[i] = u.x, c[i + 1] = u.y, c[i + 2] = u.z, c[i + 3] = u.w;
                    s[i] = v.x, s[i + 1] = v.y, s[i + 2] = v.z, s[i + 3] = v.w;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < P; ++i) c[i] = rc[i], s[i] = rs[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const float* rc = rot_row(r, r.cos, n, r.axes[j0 + i]) + j0 + i;
            c[i] = *rc;
            s[i] = r.sin[rc - r.cos];
        }
    }
}

__device__ __forceinline__ void rot_pair(float& a, float& b, float c, float s) {
    const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
    b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
    a = x;
}

// V values of T (V = 1, 2, 4, 8) as one load or store.
template <typename T, int V>
struct RotVec {
    alignas(2 * V) uint16_t h[V];
    __device__ __forceinline__ void load(const uint16_t* p) {
        if constexpr (V == 8)
            *reinterpret_cast<uint4*>(h) = *reinterpret_cast<const uint4*>(p);
        else if constexpr (V == 4)
            *reinterpret_cast<uint2*>(h) = *reinterpret_cast<const uint2*>(p);
        else if constexpr (V == 2)
            *reinterpret_cast<uint32_t*>(h) = *reinterpret_cast<const uint32_t*>(p);
        else
            h[0] = *p;
    }
    __device__ __forceinline__ void store(uint16_t* p) const {
        if constexpr (V == 8)
            *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
        else if constexpr (V == 4)
            *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(h);
        else if constexpr (V == 2)
            *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(h);
        else
            *p = h[0];
    }
    __device__ __forceinline__ float get(int i) const { return F16Traits<T>::to_f32(h[i]); }
    __device__ __forceinline__ void set(int i, float v) { h[i] = F16Traits<T>::from_f32(v); }
};

// Unit u of up to R rows of token n (src, dst: the first row; rows lie D values apart): V values and, where pairs are
// halves, the V of their partners half a rotation further; or, past the rotated dimensions, V values copied. The
// token's cos and sin are read once, the rows' loads are issued together.
template <typename T, int V, int R, bool PAIRS2>
__device__ __forceinline__ void rot_rows(const RotArgs& r, const uint16_t* src, uint16_t* dst, int rows, int n, int u) {
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
        rot_cos_sin<P>(r, n, PAIRS2 ? at / 2 : at, c, s);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (i >= rows) continue;
#pragma unroll
            for (int j = 0; j < P; ++j) {
                const int ja = PAIRS2 ? 2 * j : j, jb = PAIRS2 ? 2 * j + 1 : j;
                RotVec<T, V>& other = PAIRS2 ? lo[i] : hi[i];
                float x = lo[i].get(ja), y = other.get(jb);
                rot_pair(x, y, c[j], s[j]);
                lo[i].set(ja, x);
                other.set(jb, y);
            }
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
