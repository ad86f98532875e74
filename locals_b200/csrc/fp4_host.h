// Host entry points of the microscaled 4-bit kernels (fp4_quant.cu, fp4_gemm.cu), for fp4_api.cu.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace lq {

int fp4_quantize_run(const void* x, int dt, int64_t x_row, int rows, int K, int mode, const float* factor, uint32_t* codes,
                     uint8_t* tiles, cudaStream_t st);
int fp4_dequantize_run(const uint32_t* codes, const uint8_t* tiles, int stack, int rows, int K, int mode, const float* factor,
                       int dt, void* out, cudaStream_t st);
int fp4_qmm_run(const uint32_t* xc, const uint8_t* xt, const float* xf, const uint32_t* wc, const uint8_t* wt, const float* wf,
                int M, int N, int K, int mode, int glu, int dtype, void* y, cudaStream_t st);

// A product of 16-bit rows (or the 32-bit hidden rows of experts) with mxfp4 weights; segments > 0: grouped over at most that
// many segments.
struct Fp4Linear {
    const void* x;
    int64_t x_row;
    const int32_t *order, *starts, *experts, *nseg;
    int gather, src_rows, segments, max_rows, E;
    const uint32_t* wc;
    const uint8_t* wt;
    int rows, N, K, glu, x_dtype, dtype;
    void* y;
    void* ws;
    size_t ws_bytes;
};
size_t fp4_linear_workspace_bytes(int rows, int N, int K, int x_dtype, int segments, int max_rows);
int fp4_linear_run(const Fp4Linear& l, cudaStream_t st);

// moe.cu
int group_run(const uint32_t* inds, int P, int E, int32_t* order, int32_t* starts, int32_t* experts, int32_t* nseg,
              int32_t* pos, cudaStream_t st);
int combine_f32_run(const float* ys, const float* w, const int32_t* pos, const int32_t* ids, int E, void* y, int T, int k, int D, int dt,
                    cudaStream_t st);

}  // namespace lq
