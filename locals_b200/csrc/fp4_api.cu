// The C ABI of microscaled 4-bit floating point (include/lq.h): argument checks, then the kernels.
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/lq.h"
#include "fp4_host.h"
#include "lq_host.h"

using namespace lq;

extern "C" {

static int fp4_rows_ok(int64_t rows, int K, int mode) {
    if (mode != LQ_MXFP4 && mode != LQ_NVFP4) return LQ_E_UNSUPPORTED;
    if (rows < 1 || K < 1 || K > (1 << 24) || rows > (1 << 29)) return LQ_E_SHAPE;
    return LQ_OK;
}

int lq_fp4_quantize(const void* x, int dtype, int64_t x_row, int rows, int K, int mode, const float* factor,
                    uint32_t* codes, uint8_t* tiles, void* stream) {
    if (!x || !codes || !tiles) return LQ_E_ARG;
    if (dtype != LQ_F32 && !is16(dtype)) return LQ_E_ARG;
    if (mode == LQ_MXFP4 && factor) return LQ_E_ARG;
    int rc = fp4_rows_ok(rows, K, mode);
    if (rc) return rc;
    if (x_row < K && rows > 1) return LQ_E_SHAPE;
    if (!aligned(codes, 32) || !aligned(tiles, 16) || !aligned(x, dtype == LQ_F32 ? 4 : 2)) return LQ_E_ALIGN;
    rc = check_device();
    if (rc) return rc;
    return finish(fp4_quantize_run(x, dtype, x_row, rows, K, mode, factor, codes, tiles, reinterpret_cast<cudaStream_t>(stream)));
}

int lq_fp4_dequantize(const uint32_t* codes, const uint8_t* tiles, int stack, int rows, int K, int mode,
                      const float* factor, int dtype, void* out, void* stream) {
    if (!codes || !tiles || !out) return LQ_E_ARG;
    if (dtype != LQ_F32 && !is16(dtype)) return LQ_E_ARG;
    if (stack < 1) return LQ_E_SHAPE;
    int rc = fp4_rows_ok(int64_t(stack) * rows, K, mode);
    if (rc) return rc;
    if (!aligned(codes, 32) || !aligned(tiles, 16)) return LQ_E_ALIGN;
    rc = check_device();
    if (rc) return rc;
    return finish(fp4_dequantize_run(codes, tiles, stack, rows, K, mode, factor, dtype, out, reinterpret_cast<cudaStream_t>(stream)));
}

int lq_fp4_qmm(const uint32_t* x_codes, const uint8_t* x_tiles, const float* x_factor, const uint32_t* w_codes,
               const uint8_t* w_tiles, const float* w_factor, int M, int N, int K, int mode, int glu, int dtype, void* y,
               void* stream) {
    if (!x_codes || !x_tiles || !w_codes || !w_tiles || !y) return LQ_E_ARG;
    if (dtype != LQ_F32 && !is16(dtype)) return LQ_E_ARG;
    int rc = fp4_rows_ok(M, K, mode);
    if (!rc) rc = fp4_rows_ok(N, K, mode);
    if (rc) return rc;
    if (glu && N % 2) return LQ_E_SHAPE;
    if (!aligned(x_codes, 32) || !aligned(w_codes, 32) || !aligned(x_tiles, 16) || !aligned(w_tiles, 16) || !aligned(y, dtype == LQ_F32 ? 4 : 2))
        return LQ_E_ALIGN;
    rc = check_device();
    if (rc) return rc;
    return finish(fp4_qmm_run(x_codes, x_tiles, x_factor, w_codes, w_tiles, w_factor, M, N, K, mode, glu, dtype, y,
                              reinterpret_cast<cudaStream_t>(stream)));
}

size_t lq_fp4_linear_workspace(int M, int N, int K, int dtype) {
    return fp4_rows_ok(M, K, LQ_MXFP4) || fp4_rows_ok(N, K, LQ_MXFP4) || !is16(dtype) ? 0 : fp4_linear_workspace_bytes(M, N, K, dtype, 0, M);
}

int lq_fp4_linear(const void* x, int64_t x_row, const uint32_t* codes, const uint8_t* tiles, int M, int N, int K, int glu,
                  int dtype, void* y, void* workspace, size_t workspace_bytes, void* stream) {
    if (!x || !codes || !tiles || !y || !is16(dtype)) return LQ_E_ARG;
    int rc = fp4_rows_ok(M, K, LQ_MXFP4);
    if (!rc) rc = fp4_rows_ok(N, K, LQ_MXFP4);
    if (rc) return rc;
    if (glu && N % 2) return LQ_E_SHAPE;
    if (x_row < K && M > 1) return LQ_E_SHAPE;
    const size_t bytes = lq_fp4_linear_workspace(M, N, K, dtype);
    if (bytes && !workspace) return LQ_E_ARG;
    if (workspace_bytes < bytes) return LQ_E_SHAPE;
    if (!aligned(codes, 32) || !aligned(tiles, 16) || !aligned(workspace, 256) || !aligned(x, 2) || !aligned(y, 2)) return LQ_E_ALIGN;
    rc = check_device();
    if (rc) return rc;
    Fp4Linear l = {};
    l.x = x;
    l.x_row = x_row;
    l.wc = codes;
    l.wt = tiles;
    l.src_rows = M;
    l.rows = M;
    l.N = N;
    l.K = K;
    l.glu = glu;
    l.dtype = dtype;
    l.y = y;
    l.ws = workspace;
    return finish(fp4_linear_run(l, reinterpret_cast<cudaStream_t>(stream)));
}

static int fp4_segments(int P, int E) { return P < E + 1 ? P : E + 1; }

size_t lq_fp4_experts_workspace(int P, int max_rows, int E, int N, int K, int dtype) {
    if (fp4_rows_ok(P, K, LQ_MXFP4) || fp4_rows_ok(N, K, LQ_MXFP4) || !is16(dtype) || E < 1 || max_rows < 1) return 0;
    const size_t some = fp4_linear_workspace_bytes(P, N, K, dtype, fp4_segments(P, E), max_rows);
    const size_t each = P <= 1024 ? fp4_linear_workspace_bytes(P, N, K, dtype, P, max_rows) : 0;  // without segments
    return some > each ? some : each;
}

int lq_fp4_experts(const void* x, int x_rows, const int32_t* gather_order, int gather_k, const int32_t* starts,
                   const int32_t* experts, const int32_t* nseg, int P, int max_rows, int glu, const uint32_t* codes,
                   const uint8_t* tiles, void* out, int E, int N, int K, int dtype, void* workspace,
                   size_t workspace_bytes, void* stream) {
    if (!x || !experts || !codes || !tiles || !out || !is16(dtype) || !starts != !nseg) return LQ_E_ARG;
    if (gather_k < 0 || (gather_order && gather_k < 1)) return LQ_E_ARG;
    int rc = fp4_rows_ok(P, K, LQ_MXFP4);
    if (!rc && (E < 1 || max_rows < 1 || x_rows < 1 || (!gather_order && x_rows <= (P - 1) / (gather_k ? gather_k : 1)))) rc = LQ_E_SHAPE;
    if (!rc) rc = fp4_rows_ok(int64_t(E) * N, K, LQ_MXFP4);
    if (rc) return rc;
    const int segments = starts ? fp4_segments(P, E) : P;
    if ((glu && N % 2) || segments > 1024) return LQ_E_SHAPE;
    const size_t bytes = lq_fp4_experts_workspace(P, max_rows, E, N, K, dtype);
    if (bytes && !workspace) return LQ_E_ARG;
    if (workspace_bytes < bytes) return LQ_E_SHAPE;
    if (!aligned(codes, 32) || !aligned(tiles, 16) || !aligned(workspace, 256) || !aligned(x, 2) || !aligned(out, 2)) return LQ_E_ALIGN;
    rc = check_device();
    if (rc) return rc;
    Fp4Linear l = {};
    l.x = x;
    l.x_row = K;
    l.order = gather_order;
    l.gather = gather_k;
    l.src_rows = x_rows;
    l.starts = starts;
    l.experts = experts;
    l.nseg = nseg;
    l.segments = segments;
    l.max_rows = max_rows;
    l.E = E;
    l.wc = codes;
    l.wt = tiles;
    l.rows = P;
    l.N = N;
    l.K = K;
    l.glu = glu;
    l.dtype = dtype;
    l.y = out;
    l.ws = workspace;
    return finish(fp4_linear_run(l, reinterpret_cast<cudaStream_t>(stream)));
}

}  // extern "C"
