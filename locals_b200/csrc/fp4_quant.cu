// Microscaled 4-bit floating point in and out: quantize and dequantize.
//
// quantize: a lane takes 8 values (one word of codes) at a time, a group is 4 (mxfp4) or 2 (nvfp4) threads, its largest magnitude
// found with shuffles. mxfp4: scale 2^(floor(log2 amax) - 2), at least 2^-127: the exponent field of amax less 2, so that no
// logarithm is taken, and x 2^-e is exact. nvfp4: scale = the e4m3 number nearest to amax / (6 f), f the matrix' factor, and
// codes nearest to x / (scale f), both decided as in exact arithmetic: with 32-bit arithmetic where it is clear, in
// 64 bits where a value lies within its error of the middle between two codes.
#include <cuda_runtime.h>

#include "fp4.cuh"
#include "fp4_host.h"
#include "lq_host.h"

namespace lq {

// The e4m3 byte nearest to t >= 0 (ties to even), at most 448.
__device__ __forceinline__ uint32_t e4m3_of(double t) {
    if (!(t < 448.0)) return t != t ? 0x7Fu : 0x7Eu;
    int e = int((__double_as_longlong(t) >> 52) & 0x7FF) - 1023;
    e = e < -6 ? -6 : e;
    const double n = rint(t * __longlong_as_double((long long)(1023 + 3 - e) << 52));
    return uint32_t((e + 6) * 8 + int(n));
}

// The code nearest to |x| / s, decided in 64 bits (s has at most 28 bits, so that s times a middle is exact).
__device__ __noinline__ uint32_t code_exact(float x, double s) {
    const double a = fabs(double(x));
    uint32_t c = (a > 0.25 * s) + (a >= 0.75 * s) + (a > 1.25 * s) + (a >= 1.75 * s) + (a > 2.5 * s) + (a >= 3.5 * s) + (a > 5.0 * s);
    return c | (__float_as_uint(x) >> 31 << 3);
}

// A warp takes UNR times 256 values of a row, all loads first.
template <typename T, int MODE, int UNR>
__global__ void __launch_bounds__(256) fp4_quantize_kernel(const T* __restrict__ x, int64_t x_row, int rows, int K, bool vec,
                                                           const float* __restrict__ factor, uint32_t* __restrict__ codes,
                                                           uint8_t* __restrict__ tiles) {
    constexpr int LANES = MODE == LQ_MXFP4 ? 4 : 2;  // threads a group
    const int lane = threadIdx.x & 31, words = fp4_padded(K) / 8, ktiles = fp4_ktiles(K, MODE), parts = (words + 32 * UNR - 1) / (32 * UNR);
    const float f = MODE == LQ_NVFP4 && factor ? *factor : 1.f;
    const int64_t tasks = int64_t(rows) * parts;
    for (int64_t u = (int64_t(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; u < tasks; u += (int64_t(gridDim.x) * blockDim.x) >> 5) {
        const int row = int(u / parts), w0 = int(u - int64_t(row) * parts) * 32 * UNR + lane;
        const T* src = x + int64_t(row) * x_row;
        uint32_t* codes_row = codes + int64_t(row) * words;
        uint8_t* tiles_row = tiles + int64_t(row >> 7) * ktiles * 512 + fp4_tile_byte(row & 127, 0);
        Eight<T> x8[UNR];
#pragma unroll
        for (int i = 0; i < UNR; ++i)  // (beyond the row: zeros)
            x8[i].load(src, 8 * (w0 + 32 * i), K, vec);
#pragma unroll
        for (int i = 0; i < UNR; ++i) {
            const int word = w0 + 32 * i;
            if (word - lane >= words) break;  // (rows are a multiple of 16 words: half a warp may be beyond)
            float v[8], top = x8[i].amax();
#pragma unroll
            for (int d = 1; d < LANES; d *= 2) top = amax_nan(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
            uint32_t byte, w;
            if constexpr (MODE == LQ_MXFP4) {
                const uint32_t e = __float_as_uint(top) >> 23 & 0xFF;
                byte = e == 255 ? 255u : e < 2 ? 0u : e - 2;
                const float up = __uint_as_float((254u - (byte == 255 ? 127u : byte)) << 23);
                x8[i].times(up, v);
                w = codes8(v);
            } else {
                // (zeros have scale 0 whatever the factor is: that of a matrix of zeros is 0 where it is made of its largest)
                byte = top == INFINITY ? 0x7Fu : top == 0.f ? 0u : e4m3_of(double(top) / (6.0 * double(f)));
                const float s = fp4_scale_value(byte, LQ_NVFP4);
                w = 0;
                if (byte != 0 && byte != 0x7F) {
                    const double sf = double(s) * double(f);
                    const float r = __frcp_rn(float(sf));
                    float lo[8], hi[8];
                    x8[i].times(r, v);
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        lo[q] = v[q] * (1.f - 0x1p-20f);
                        hi[q] = v[q] * (1.f + 0x1p-20f);
                    }
                    w = codes8(lo);
                    // (the reciprocal of a factor near the ends of the range is no normal number: 64 bits then)
                    if (w != codes8(hi) || !(r > 0x1p-126f && r < 0x1p127f)) {
                        w = 0;
                        x8[i].times(1.f, v);
#pragma unroll
                        for (int q = 0; q < 8; ++q) w |= code_exact(v[q], sf) << (4 * q);
                    }
                }
            }
            if (word >= words) continue;
            codes_row[word] = w;
            const int g = word / LANES;
            if (word % LANES == 0) tiles_row[(g >> 2) * 512 + (g & 3)] = uint8_t(byte);
        }
    }
}

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The values of a word's eight codes (exact in fp16).
__device__ __forceinline__ void values8(uint32_t w, float (&v)[8]) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = __half22float2(*reinterpret_cast<__half2*>(&h[i]));
        v[2 * i] = p.x;
        v[2 * i + 1] = p.y;
    }
}

// A warp takes four times 256 values of a row, all loads first.
template <typename T, int MODE>
__global__ void __launch_bounds__(256) fp4_dequantize_kernel(const uint32_t* __restrict__ codes,
                                                             const uint8_t* __restrict__ tiles, int stack, int rows, int K,
                                                             const float* __restrict__ factor, T* __restrict__ out, bool vec) {
    constexpr int GROUP = MODE == LQ_MXFP4 ? 32 : 16, UNR = 4;
    const int stored = fp4_padded(K) / 8, words = (K + 7) / 8, ktiles = fp4_ktiles(K, MODE), rtiles = (rows + 127) / 128;
    const int lane = threadIdx.x & 31, parts = (words + 32 * UNR - 1) / (32 * UNR);
    const float f = factor ? *factor : 1.f;
    const int64_t tasks = int64_t(stack) * rows * parts;
    for (int64_t u = (int64_t(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; u < tasks; u += (int64_t(gridDim.x) * blockDim.x) >> 5) {
        const int64_t at = u / parts;  // row of the stack
        const int w0 = int(u - at * parts) * 32 * UNR + lane, e = int(at / rows), row = int(at - int64_t(e) * rows);
        const uint8_t* tl = tiles + (int64_t(e) * rtiles + (row >> 7)) * ktiles * 512;
        uint32_t w[UNR], byte[UNR];
#pragma unroll
        for (int i = 0; i < UNR; ++i) {
            const int word = w0 + 32 * i, g = word * 8 / GROUP;
            w[i] = byte[i] = 0;
            if (word < words) {
                w[i] = codes[at * stored + word];
                byte[i] = tl[int64_t(g >> 2) * 512 + fp4_tile_byte(row & 127, g)];
            }
        }
#pragma unroll
        for (int i = 0; i < UNR; ++i) {
            const int word = w0 + 32 * i;
            if (word - lane >= words) break;
            const float s = fp4_scale_value(byte[i], MODE);
            float a[8];
            values8(w[i], a);
            if constexpr (sizeof(T) == 4) {
                // two lanes a word, 16 bytes each, so that a store fills whole sectors (72 -> 50 us for 14336 x 4096)
                if (vec) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int from = 16 * h + lane / 2;
                        float4 q;
                        float* qp = &q.x;
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const float lo = __shfl_sync(0xFFFFFFFFu, a[c] * s * f, from), hi = __shfl_sync(0xFFFFFFFFu, a[4 + c] * s * f, from);
                            qp[c] = lane & 1 ? hi : lo;
                        }
                        const int at8 = w0 - lane + 32 * i + from;
                        if (at8 < words) *reinterpret_cast<float4*>(out + at * K + 8 * at8 + 4 * (lane & 1)) = q;
                    }
                    continue;
                }
            }
            if (word >= words) break;
            T* dst = out + at * K + 8 * word;
            alignas(16) T v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = from_f32<T>(a[q] * s * f);
            if (vec) {
#pragma unroll
                for (int q = 0; q < int(8 * sizeof(T) / 16); ++q) reinterpret_cast<uint4*>(dst)[q] = reinterpret_cast<uint4*>(v)[q];
            } else {
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (8 * word + q < K) dst[q] = v[q];
            }
        }
    }
}

// ---- host ----

// Blocks of eight warps for so many tasks of a warp.
static int spread(int64_t tasks) {
    const int64_t blocks = (tasks + 7) / 8, most = int64_t(device_info().sm_count) * 16;
    return int(blocks < most ? blocks : most);
}

template <typename T, int MODE>
static int quantize_tm(const T* x, int64_t x_row, int rows, int K, bool vec, const float* factor, uint32_t* codes, uint8_t* tiles,
                       cudaStream_t st) {
    // few rows: as many warps as there are pieces of 256 values; many: more loads a warp
    const int64_t pieces = int64_t(rows) * ((fp4_padded(K) + 255) / 256);
    constexpr int UNR = sizeof(T) == 4 ? 2 : 4;
    if (pieces < int64_t(device_info().sm_count) * 64)
        fp4_quantize_kernel<T, MODE, 1><<<spread(pieces), 256, 0, st>>>(x, x_row, rows, K, vec, factor, codes, tiles);
    else
        fp4_quantize_kernel<T, MODE, UNR><<<spread(int64_t(rows) * ((fp4_padded(K) + 256 * UNR - 1) / (256 * UNR))), 256, 0, st>>>(
            x, x_row, rows, K, vec, factor, codes, tiles);
    return cuda_status(cudaGetLastError());
}

template <typename T>
static int quantize_t(const void* x, int64_t x_row, int rows, int K, int mode, const float* factor, uint32_t* codes,
                      uint8_t* tiles, cudaStream_t st) {
    const T* xs = static_cast<const T*>(x);
    const bool vec = aligned(x, 16) && x_row * int64_t(sizeof(T)) % 16 == 0;
    return mode == LQ_MXFP4 ? quantize_tm<T, LQ_MXFP4>(xs, x_row, rows, K, vec, factor, codes, tiles, st)
                            : quantize_tm<T, LQ_NVFP4>(xs, x_row, rows, K, vec, factor, codes, tiles, st);
}

int fp4_quantize_run(const void* x, int dt, int64_t x_row, int rows, int K, int mode, const float* factor, uint32_t* codes,
                     uint8_t* tiles, cudaStream_t st) {
    if (dt == LQ_F32) return quantize_t<float>(x, x_row, rows, K, mode, factor, codes, tiles, st);
    if (dt == LQ_F16) return quantize_t<__half>(x, x_row, rows, K, mode, factor, codes, tiles, st);
    return quantize_t<__nv_bfloat16>(x, x_row, rows, K, mode, factor, codes, tiles, st);
}

template <typename T>
static int dequantize_t(const uint32_t* codes, const uint8_t* tiles, int stack, int rows, int K, int mode, const float* factor,
                        void* out, cudaStream_t st) {
    const int grid = spread(int64_t(stack) * rows * ((K + 1023) / 1024));
    T* o = static_cast<T*>(out);
    const bool vec = K % 8 == 0 && aligned(out, 16);
    if (mode == LQ_MXFP4)
        fp4_dequantize_kernel<T, LQ_MXFP4><<<grid, 256, 0, st>>>(codes, tiles, stack, rows, K, factor, o, vec);
    else
        fp4_dequantize_kernel<T, LQ_NVFP4><<<grid, 256, 0, st>>>(codes, tiles, stack, rows, K, factor, o, vec);
    return cuda_status(cudaGetLastError());
}

int fp4_dequantize_run(const uint32_t* codes, const uint8_t* tiles, int stack, int rows, int K, int mode, const float* factor,
                       int dt, void* out, cudaStream_t st) {
    if (dt == LQ_F32) return dequantize_t<float>(codes, tiles, stack, rows, K, mode, factor, out, st);
    if (dt == LQ_F16) return dequantize_t<__half>(codes, tiles, stack, rows, K, mode, factor, out, st);
    return dequantize_t<__nv_bfloat16>(codes, tiles, stack, rows, K, mode, factor, out, st);
}

}  // namespace lq
