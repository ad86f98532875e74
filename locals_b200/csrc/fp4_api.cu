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
    l.x_dtype = l.dtype = dtype;
    l.y = y;
    l.ws = workspace;
    l.ws_bytes = workspace_bytes;
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
    l.x_dtype = l.dtype = dtype;
    l.y = out;
    l.ws = workspace;
    l.ws_bytes = workspace_bytes;
    return finish(fp4_linear_run(l, reinterpret_cast<cudaStream_t>(stream)));
}

// Where the parts of lq_fp4_moe's workspace lie, in bytes: hidden rows and experts' outputs in 32 bits, the grouping (from two
// tokens on), the workspace of the two products in turn.
struct MoeParts {
    size_t hidden, outputs, group, product, all;
    int segments;
};

static int fp4_moe_parts(int T, int k, int E, int D, int I, int dtype, MoeParts& m) {
    if (!is16(dtype)) return LQ_E_ARG;
    if (T < 1 || k < 1 || E < 1 || int64_t(T) * k > (1 << 29) || I > (1 << 28)) return LQ_E_SHAPE;
    const int P = T * k;
    int rc = fp4_rows_ok(int64_t(E) * 2 * I, D, LQ_MXFP4);
    if (!rc) rc = fp4_rows_ok(int64_t(E) * D, I, LQ_MXFP4);
    if (rc) return rc;
    m.segments = T > 1 && E < P ? E : P;
    if (m.segments > 1024 || (T > 1 && E > 8192)) return LQ_E_SHAPE;  // (lq_moe_group's experts)
    auto whole = [](size_t bytes) { return (bytes + 255) / 256 * 256; };
    m.hidden = 0;
    m.outputs = m.hidden + whole(size_t(P) * I * sizeof(float));
    m.group = m.outputs + whole(size_t(P) * D * sizeof(float));
    m.product = m.group + (T > 1 ? whole((2 * size_t(P) + 2 * m.segments + 2) * sizeof(int32_t)) : 0);
    // (of the very segments that the products run with: tiles, and so these bytes, go by their number)
    const size_t up = fp4_linear_workspace_bytes(P, 2 * I, D, dtype, m.segments, T);
    const size_t down = fp4_linear_workspace_bytes(P, D, I, LQ_F32, m.segments, T);
    m.all = m.product + whole(up > down ? up : down);
    return LQ_OK;
}

size_t lq_fp4_moe_workspace(int T, int k, int E, int D, int I, int dtype) {
    MoeParts m;
    return fp4_moe_parts(T, k, E, D, I, dtype, m) ? 0 : m.all;
}

int lq_fp4_moe(const void* x, const int32_t* inds, const float* weights, const uint32_t* gate_up_codes,
               const uint8_t* gate_up_tiles, const uint32_t* down_codes, const uint8_t* down_tiles, void* y, int T, int k, int E,
               int D, int I, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    if (!x || !inds || !weights || !gate_up_codes || !gate_up_tiles || !down_codes || !down_tiles || !y) return LQ_E_ARG;
    MoeParts m;
    int rc = fp4_moe_parts(T, k, E, D, I, dtype, m);
    if (rc) return rc;
    if (!workspace) return LQ_E_ARG;
    if (workspace_bytes < m.all) return LQ_E_SHAPE;
    if (!aligned(gate_up_codes, 32) || !aligned(down_codes, 32) || !aligned(gate_up_tiles, 16) || !aligned(down_tiles, 16) ||
        !aligned(workspace, 256) || !aligned(x, 2) || !aligned(y, 2) || !aligned(inds, 4) || !aligned(weights, 4))
        return LQ_E_ALIGN;
    rc = check_device();
    if (rc) return rc;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const int P = T * k;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    float *h = reinterpret_cast<float*>(ws + m.hidden), *ys = reinterpret_cast<float*>(ws + m.outputs);
    int32_t *order = nullptr, *pos = nullptr;
    Fp4Linear l = {};
    l.experts = inds;  // one token: each slot is a segment of its own
    if (T > 1) {
        order = reinterpret_cast<int32_t*>(ws + m.group);
        pos = order + P;
        int32_t *starts = pos + P, *experts = starts + m.segments + 1, *nseg = experts + m.segments;
        rc = group_run(reinterpret_cast<const uint32_t*>(inds), P, E, order, starts, experts, nseg, pos, st);
        if (rc) return finish(rc);
        l.starts = starts;
        l.experts = experts;
        l.nseg = nseg;
    }
    l.segments = m.segments;
    l.max_rows = T;
    l.E = E;
    l.rows = P;
    l.ws = ws + m.product;
    l.ws_bytes = m.all - m.product;
    l.x = x;  // gate and up: 16-bit tokens to 32-bit hidden rows
    l.x_row = D;
    l.x_dtype = dtype;
    l.order = order;
    l.gather = k;
    l.src_rows = T;
    l.wc = gate_up_codes;
    l.wt = gate_up_tiles;
    l.N = 2 * I;
    l.K = D;
    l.glu = 1;
    l.dtype = LQ_F32;
    l.y = h;
    rc = fp4_linear_run(l, st);
    if (rc) return finish(rc);
    l.x = h;  // down: 32-bit hidden rows to 32-bit outputs
    l.x_row = I;
    l.x_dtype = LQ_F32;
    l.order = nullptr;
    l.gather = 0;
    l.src_rows = P;
    l.wc = down_codes;
    l.wt = down_tiles;
    l.N = D;
    l.K = I;
    l.glu = 0;
    l.y = ys;
    rc = fp4_linear_run(l, st);
    if (rc) return finish(rc);
    return finish(combine_f32_run(ys, weights, pos, inds, E, y, T, k, D, dtype, st));
}

}  // extern "C"
