// The host side of locals_b200.fp4 (see paged_ext.cpp, which includes this): checks, outputs and workspaces, and the calls of
// liblq.so. A product of one token takes the GPU less time than these steps take in Python (17 to 22 us a call there).
#pragma once

namespace fp4 {

int mode_code(const std::string& mode) {
    if (mode == "mxfp4") return LQ_MXFP4;
    if (mode == "nvfp4") return LQ_NVFP4;
    throw py::value_error("a 4-bit format is one of mxfp4, nvfp4, not '" + mode + "'");
}

int any_dtype(at::ScalarType t) {
    if (t == at::kHalf) return LQ_F16;
    if (t == at::kBFloat16) return LQ_BF16;
    if (t == at::kFloat) return LQ_F32;
    throw py::type_error("fp16, bf16 or fp32 expected");
}

int64_t padded(int64_t K) { return (K + 127) / 128 * 128; }

const float* factor(const MaybeTensor& scale, int mode, const at::Device& dev) {
    if (!scale) return nullptr;
    need(mode == LQ_NVFP4, "only nvfp4 has a factor for the whole matrix");
    need(scale->scalar_type() == at::kFloat && scale->numel() == 1 && scale->device() == dev,
         "scale is one float32 element on the matrix' device");
    return scale->data_ptr<float>();
}

// An operand of Python's Fp4: its fields, checked against one another.
struct Operand {
    uint32_t* codes;
    uint8_t* tiles;
    const float* scale;
    int stack, rows, K, mode;
    at::Device dev;
};

Operand operand(const py::tuple& f, int64_t dims) {
    const Tensor codes = f[0].cast<Tensor>(), tiles = f[1].cast<Tensor>();
    const int mode = mode_code(f[2].cast<std::string>());
    const int64_t K = f[3].cast<int64_t>(), Kp = padded(K);
    const MaybeTensor scale = f[4].cast<MaybeTensor>();
    need(codes.is_cuda() && tiles.device() == codes.device(), "codes and tiles are CUDA tensors of one device");
    if ((codes.scalar_type() != at::kInt && codes.scalar_type() != at::kUInt32) || tiles.scalar_type() != at::kByte)
        throw py::type_error("codes are 32-bit words and tiles uint8");
    need(codes.dim() == 2 || codes.dim() == 3, "codes are a matrix (N, Kp / 8) or a stack (E, N, Kp / 8)");
    need(dims == 0 || codes.dim() == dims, dims == 2 ? "a 4-bit matrix is wanted, not a stack" : "a stack of 4-bit matrices is wanted");
    const int64_t E = codes.dim() == 3 ? codes.size(0) : 1, N = codes.size(-2);
    need(K >= 1 && codes.size(-1) == Kp / 8, "codes do not hold K values a row, filled to a multiple of 128");
    need(tiles.dim() == codes.dim() + 1 && (codes.dim() == 2 || tiles.size(0) == E) && tiles.size(-3) == (N + 127) / 128 &&
             tiles.size(-2) == Kp / (mode == LQ_MXFP4 ? 128 : 64) && tiles.size(-1) == 512,
         "tiles do not fit codes: (..., ceil(N / 128), Kp / (4 * group), 512) expected");
    need(codes.is_contiguous() && tiles.is_contiguous(), "codes and tiles are contiguous");
    return {static_cast<uint32_t*>(codes.data_ptr()), tiles.data_ptr<uint8_t>(), factor(scale, mode, codes.device()),
            narrow(E), narrow(N), narrow(K), mode, codes.device()};
}

// x (..., K) as rows, the elements from one to the next; a copy where its values are not next to one another.
int64_t as_rows(Tensor& x) {
    need(x.dim() >= 1, "a matrix of rows is wanted");
    if (x.dim() != 2) x = x.reshape({-1, x.size(-1)});
    if ((x.size(1) > 1 && x.stride(1) != 1) || (x.size(0) > 1 && x.stride(0) < x.size(1))) x = x.contiguous();
    return x.size(0) > 1 ? x.stride(0) : x.size(1);
}

std::tuple<Tensor, Tensor> quantize(Tensor x, const std::string& mode, const MaybeTensor& scale) {
    const int m = mode_code(mode), dt = any_dtype(x.scalar_type());
    need(x.is_cuda(), "locals_b200 kernels take CUDA tensors");
    const float* f = factor(scale, m, x.device());
    need(x.dim() >= 1 && x.size(-1) >= 1, "rows of no values");
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t row = x.numel() ? as_rows(x) : 0, K = x.size(-1), R = x.numel() / K, Kp = padded(K);
    Tensor codes = at::empty({R, Kp / 8}, x.options().dtype(at::kInt));
    Tensor tiles = at::empty({(R + 127) / 128, Kp / (m == LQ_MXFP4 ? 128 : 64), 512}, x.options().dtype(at::kByte));
    if (R)
        run("lq_fp4_quantize", lq_fp4_quantize(x.data_ptr(), dt, row, narrow(R), narrow(K), m, f,
                                               static_cast<uint32_t*>(codes.data_ptr()), tiles.data_ptr<uint8_t>(), stream()));
    return {codes, tiles};
}

Tensor dequantize(const py::tuple& a, at::ScalarType dtype) {
    const Operand o = operand(a, 0);
    const int dt = any_dtype(dtype);
    const c10::cuda::CUDAGuard guard(o.dev);
    std::vector<int64_t> shape = a[0].cast<Tensor>().sizes().vec();
    shape.back() = o.K;
    Tensor out = at::empty(shape, at::TensorOptions().device(o.dev).dtype(dtype));
    if (out.numel())
        run("lq_fp4_dequantize", lq_fp4_dequantize(o.codes, o.tiles, o.stack, o.rows, o.K, o.mode, o.scale, dt, out.data_ptr(), stream()));
    return out;
}

int64_t width(const Operand& w, bool glu) {
    need(!glu || w.rows % 2 == 0, "rows of w are pairs of gate and up");
    return glu ? w.rows / 2 : w.rows;
}

Tensor product(const py::tuple& x, const py::tuple& w, at::ScalarType dtype, bool glu) {
    const Operand a = operand(x, 2), b = operand(w, 2);
    need(a.mode == b.mode && a.K == b.K, "x and w differ in format or K");
    need(a.dev == b.dev, "x and w are on different devices");
    const int dt = any_dtype(dtype);
    const c10::cuda::CUDAGuard guard(b.dev);
    Tensor y = at::empty({a.rows, width(b, glu)}, at::TensorOptions().device(b.dev).dtype(dtype));
    if (y.numel())
        run("lq_fp4_qmm", lq_fp4_qmm(a.codes, a.tiles, a.scale, b.codes, b.tiles, b.scale, a.rows, b.rows, b.K, b.mode, glu, dt,
                                     y.data_ptr(), stream()));
    return y;
}

void check_16(const Tensor& x, const Operand& w) {
    if (x.scalar_type() != at::kHalf && x.scalar_type() != at::kBFloat16) throw py::type_error("activations are fp16, bf16 or Fp4");
    need(w.mode == LQ_MXFP4, "16-bit activations are multiplied with mxfp4 weights: quantize them for nvfp4 ones");
    need(x.device() == w.dev, "x and w are on different devices");
    need(x.dim() >= 1 && x.size(-1) == w.K, "x does not have w's K values a row");
}

// A workspace of so many bytes, which the call that uses it outlives.
struct Workspace {
    Tensor t;
    void* p = nullptr;
    Workspace(size_t bytes, const Tensor& x) {
        if (!bytes) return;
        t = at::empty({int64_t(bytes)}, x.options().dtype(at::kByte));
        p = t.data_ptr();
    }
};

Tensor linear(Tensor x, const py::tuple& w, bool glu) {
    const Operand b = operand(w, 2);
    check_16(x, b);
    const c10::cuda::CUDAGuard guard(b.dev);
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = width(b, glu);
    Tensor y = at::empty(shape, x.options(), at::MemoryFormat::Contiguous);
    if (y.numel()) {
        const int64_t row = as_rows(x);
        const int M = narrow(x.size(0)), dt = dtype_code(x);
        const size_t n = lq_fp4_linear_workspace(M, b.rows, b.K, dt);
        const Workspace ws(n, x);
        run("lq_fp4_linear", lq_fp4_linear(x.data_ptr(), row, b.codes, b.tiles, M, b.rows, b.K, glu, dt, y.data_ptr(), ws.p, n, stream()));
    }
    return y;
}

int32_t* ids(const Tensor& t, int64_t n, const at::Device& dev) {
    need((t.scalar_type() == at::kInt || t.scalar_type() == at::kUInt32) && t.is_contiguous() && t.device() == dev && t.numel() >= n,
         "a grouping is contiguous int32 tensors on x's device (moe.group)");
    return static_cast<int32_t*>(t.data_ptr());
}

Tensor grouped(const Tensor& xs, const Tensor& order, const Tensor& starts, const Tensor& experts, const Tensor& nseg,
               const py::tuple& w, int64_t max_rows, bool glu, int64_t gather_k) {
    const Operand b = operand(w, 3);
    check_16(xs, b);
    need(xs.dim() == 2 && xs.is_contiguous(), "xs is a contiguous matrix of rows");
    const int64_t P = order.numel(), S = std::min<int64_t>(P, starts.numel() - 1);
    const int32_t *o = ids(order, P, b.dev), *s = ids(starts, S + 1, b.dev), *e = ids(experts, S, b.dev), *n = ids(nseg, 1, b.dev);
    need(P == 0 || S >= 1, "a grouping of pairs has segments");
    need(gather_k >= 0 && (gather_k || xs.size(0) >= P), "xs has a row a pair, or gather_k says how many pairs a token has");
    const c10::cuda::CUDAGuard guard(b.dev);
    Tensor out = at::empty({P, width(b, glu)}, xs.options());
    if (out.numel()) {
        need(xs.size(0) >= 1 && max_rows >= 1, "pairs have tokens");
        const int dt = dtype_code(xs);
        const size_t bytes = lq_fp4_experts_workspace(narrow(P), narrow(max_rows), b.stack, b.rows, b.K, dt);
        const Workspace ws(bytes, xs);
        run("lq_fp4_experts", lq_fp4_experts(xs.data_ptr(), narrow(xs.size(0)), gather_k ? o : nullptr, narrow(gather_k), s, e, n,
                                             narrow(P), narrow(max_rows), glu, b.codes, b.tiles, out.data_ptr(), b.stack, b.rows, b.K,
                                             dt, ws.p, bytes, stream()));
    }
    return out;
}

// The routed experts of a step, and their weighted sum.
Tensor experts(Tensor x, Tensor inds, Tensor weights, const py::tuple& gate_up, const py::tuple& down) {
    const Operand g = operand(gate_up, 3), d = operand(down, 3);
    need(x.dim() == 2 && inds.dim() == 2 && inds.size(0) == x.size(0), "x (T, D) and inds (T, k) are wanted");
    check_16(x, g);
    need(inds.scalar_type() == at::kInt || inds.scalar_type() == at::kUInt32, "inds are int32");
    need(weights.sizes() == inds.sizes() && weights.scalar_type() == at::kFloat, "weights are float32, one an expert id");
    need(inds.device() == x.device() && weights.device() == x.device() && d.dev == x.device(), "tensors of one device are wanted");
    need(g.rows % 2 == 0 && d.stack == g.stack && d.K == g.rows / 2 && d.rows == g.K && d.mode == LQ_MXFP4,
         "gate_up (E, 2 I, D) and down (E, D, I) do not fit one another");
    const c10::cuda::CUDAGuard guard(g.dev);
    x = x.contiguous();
    inds = inds.contiguous();
    weights = weights.contiguous();
    const int T = narrow(x.size(0)), k = narrow(inds.size(1)), E = g.stack, D = g.K, I = d.K, dt = dtype_code(x);
    if (T == 0 || k == 0) return at::zeros(x.sizes(), x.options());
    Tensor y = at::empty({T, D}, x.options());
    const size_t n = lq_fp4_moe_workspace(T, k, E, D, I, dt);
    const Workspace ws(n, x);
    run("lq_fp4_moe", lq_fp4_moe(x.data_ptr(), static_cast<const int32_t*>(inds.data_ptr()), weights.data_ptr<float>(), g.codes, g.tiles,
                                 d.codes, d.tiles, y.data_ptr(), T, k, E, D, I, dt, ws.p, n, stream()));
    return y;
}

}  // namespace fp4
