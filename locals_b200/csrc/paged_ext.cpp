// The host side of locals_b200.paged, locals_b200.rotary and (fp4_ext.h) locals_b200.fp4 between Python and the C ABI (include/lq.h): argument checks,
// outputs and workspaces from the tensor library's allocator on the current stream, one call of liblq.so each. What these
// operators do at their smallest sizes takes the GPU a few microseconds, less than the checks and allocations take in
// Python (attend at one token: 19.5 us a call there).
//
// Refusals raise ValueError or TypeError before any launch; an LQ_E_* code raises locals_b200._lib.LQError.
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/lq.h"

namespace py = pybind11;
using at::Tensor;
using Triple = std::tuple<Tensor, Tensor, Tensor>;
using MaybeTensor = std::optional<Tensor>;

namespace {

void need(bool ok, const char* what) {
    if (!ok) throw py::value_error(what);
}

int dtype_code(const Tensor& t) {
    if (t.scalar_type() == at::kHalf) return LQ_F16;
    if (t.scalar_type() == at::kBFloat16) return LQ_BF16;
    throw py::type_error("fp16 or bf16 tensors expected");
}

// The current device, where the first tensor has to lie (one on the CPU is refused before a driver is asked for).
int current(const Tensor& first) {
    need(first.is_cuda(), "locals_b200 kernels take CUDA tensors of the current device");
    return c10::cuda::current_device();
}

bool here(const Tensor& t, int dev) { return t.is_cuda() && t.get_device() == dev; }

void ints(const Tensor& t, int dev) {
    need(t.scalar_type() == at::kInt && t.is_contiguous() && here(t, dev),
         "lengths, tables, page lists and slots are contiguous int32 tensors of the current GPU");
}

int narrow(int64_t v) {
    need(v >= -0x7fffffffLL && v <= 0x7fffffffLL, "a size is beyond 32 bits");
    return int(v);
}

void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

void run(const char* name, int rc) {
    if (rc == LQ_OK) return;
    py::object error = py::module_::import("locals_b200._lib").attr("LQError");
    py::object value = error(name, rc);
    PyErr_SetObject(error.ptr(), value.ptr());
    throw py::error_already_set();
}

// x (tokens, heads, D) with a token's heads contiguous (a slice of a fused projection is fine), and the elements from one
// token to the next.
int64_t rows(Tensor& x, int dev) {
    need(x.dim() == 3, "(tokens, heads, head_dim) tensors expected");
    need(here(x, dev), "locals_b200 kernels take CUDA tensors of the current device");
    const int64_t N = x.size(0), H = x.size(1), D = x.size(2);
    if (x.is_contiguous()) return H * D;
    if ((x.stride(2) != 1 && D > 1) || (x.stride(1) != D && H > 1) || (N > 1 && x.stride(0) < H * D)) {
        x = x.contiguous();
        return H * D;
    }
    return N > 1 ? x.stride(0) : H * D;
}

// x where its rows lie on `bytes`-byte boundaries, else a copy that does.
void on_boundary(Tensor& x, int64_t& row, int bytes) {
    if (reinterpret_cast<uintptr_t>(x.data_ptr()) % bytes == 0 && row * 2 % bytes == 0) return;
    x = x.clone(at::MemoryFormat::Contiguous);
    row = x.size(1) * x.size(2);
}

Tensor like(const Tensor& x) { return at::empty(x.sizes(), x.options(), at::MemoryFormat::Contiguous); }

struct Angles {
    const int32_t* positions = nullptr;
    const float *cos = nullptr, *sin = nullptr;
    const int32_t* axes = nullptr;
    int rot = 0, max_pos = 1, naxes = 1;
};

Angles angles(const Tensor& positions, const Tensor& cos, const Tensor& sin, const MaybeTensor& axes, int64_t N, int64_t D,
              int dev) {
    need(positions.scalar_type() == at::kInt && (positions.dim() == 1 || positions.dim() == 2) && positions.size(-1) == N,
         "positions: int32 (tokens,) or (axes, tokens) expected");
    need(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat && cos.dim() == 2 && cos.sizes() == sin.sizes(),
         "cos and sin: float32 (positions, rot / 2) tables expected");
    Angles a;
    a.rot = narrow(2 * cos.size(1));
    a.max_pos = narrow(cos.size(0));
    a.naxes = positions.dim() == 1 ? 1 : narrow(positions.size(0));
    need(a.rot >= 2 && a.rot <= D && a.max_pos >= 1 && a.naxes >= 1, "the rotated dimensions do not fit head_dim");
    const char* place = "positions, cos, sin and axes must be contiguous tensors on the queries' device";
    need(here(positions, dev) && positions.is_contiguous() && here(cos, dev) && cos.is_contiguous() && here(sin, dev) &&
             sin.is_contiguous(),
         place);
    if (axes) {
        need(axes->scalar_type() == at::kInt && axes->dim() == 1 && axes->size(0) == a.rot / 2, "axes: int32 (rot / 2,) expected");
        need(here(*axes, dev) && axes->is_contiguous(), place);
        a.axes = axes->data_ptr<int32_t>();
    }
    a.positions = positions.data_ptr<int32_t>();
    a.cos = cos.data_ptr<float>();
    a.sin = sin.data_ptr<float>();
    return a;
}

struct Pool {
    uint32_t *kq, *vq;
    void *ks, *kb, *vs, *vb;
    int pages, KVH, page, D;
};

Pool pool(const Triple& keys, const Triple& values, at::ScalarType dtype, int dev) {
    const auto& [kq, ks, kb] = keys;
    const auto& [vq, vs, vb] = values;
    need(kq.dim() == 4 && kq.scalar_type() == at::kInt && vq.scalar_type() == at::kInt,
         "words: int32 (pages, KVH, page_size, head_dim / 8) expected");
    need(vq.sizes() == kq.sizes() && ks.dim() == 4 && ks.size(0) == kq.size(0) && ks.size(1) == kq.size(1) &&
             ks.size(2) == kq.size(2) && ks.size(3) * 8 == kq.size(3) && kb.sizes() == ks.sizes() &&
             vs.sizes() == ks.sizes() && vb.sizes() == ks.sizes(),
         "keys and values are not 4-bit triples of one pool");
    for (const Tensor* t : {&ks, &kb, &vs, &vb})
        if (t->scalar_type() != dtype) throw py::type_error("scales and biases must have the queries' dtype");
    for (const Tensor* t : {&kq, &ks, &kb, &vq, &vs, &vb})
        need(here(*t, dev) && t->is_contiguous(), "the cache must be contiguous tensors on the queries' device, the current one");
    return {reinterpret_cast<uint32_t*>(kq.data_ptr()), reinterpret_cast<uint32_t*>(vq.data_ptr()), ks.data_ptr(), kb.data_ptr(),
            vs.data_ptr(), vb.data_ptr(), narrow(kq.size(0)), narrow(kq.size(1)), narrow(kq.size(2)), narrow(kq.size(3) * 8)};
}

std::vector<Tensor> plan(const Tensor& cached, const Tensor& fresh, const Tensor& table, const Tensor& free_pages,
                         const Tensor& head, int64_t page, int64_t tokens) {
    const int dev = current(cached);
    for (const Tensor* t : {&cached, &fresh, &table, &free_pages, &head}) ints(*t, dev);
    need(cached.dim() == 1 && cached.sizes() == fresh.sizes() && table.dim() == 2 && table.size(0) == cached.size(0),
         "plan: cached (B,), new (B,), block_table (B, width)");
    need(free_pages.dim() == 1 && head.numel() == 1, "plan: free (pages,), head (1,)");
    need(tokens >= 0, "plan: tokens must not be negative");
    const int64_t B = cached.size(0);
    Tensor buf = at::empty({B + B + 1 + 2 * tokens + 1}, cached.options());
    int32_t* p = buf.data_ptr<int32_t>();
    run("lq_page_plan",
        lq_page_plan(cached.data_ptr<int32_t>(), fresh.data_ptr<int32_t>(), narrow(B), table.data_ptr<int32_t>(),
                     narrow(table.size(1)), free_pages.data_ptr<int32_t>(), narrow(free_pages.size(0)),
                     head.data_ptr<int32_t>(), narrow(page), narrow(tokens), p, p + B, p + 2 * B + 1, p + 2 * B + 1 + tokens,
                     p + 2 * B + 1 + 2 * tokens, stream()));
    return buf.split_with_sizes({B, B + 1, tokens, tokens, 1});
}

std::tuple<Tensor, MaybeTensor> rotate(Tensor q, MaybeTensor k, const Tensor& positions, const Tensor& cos, const Tensor& sin,
                                       const MaybeTensor& axes, bool interleaved) {
    const int dev = current(q);
    int64_t q_row = rows(q, dev), k_row = 0, KVH = 0;
    const int64_t N = q.size(0), H = q.size(1), D = q.size(2);
    if (interleaved) on_boundary(q, q_row, 4);
    if (k) {
        k_row = rows(*k, dev);
        if (interleaved) on_boundary(*k, k_row, 4);
        KVH = k->size(1);
        need(k->size(0) == N && k->size(2) == D && k->scalar_type() == q.scalar_type(),
             "q and k must have the same tokens, head_dim and dtype");
    }
    const Angles a = angles(positions, cos, sin, axes, N, D, dev);
    Tensor qo = like(q);
    MaybeTensor ko;
    if (k) ko = like(*k);
    if (N)
        run("lq_rotary", lq_rotary(q.data_ptr(), q_row, qo.data_ptr(), narrow(H), k ? k->data_ptr() : nullptr, k_row,
                                   k ? ko->data_ptr() : nullptr, narrow(KVH), narrow(N), narrow(D), a.rot, a.positions, a.cos,
                                   a.sin, a.max_pos, a.axes, a.naxes, interleaved, dtype_code(q), stream()));
    return {qo, ko};
}

MaybeTensor append(MaybeTensor q, Tensor k, Tensor v, const Tensor& slots, const Triple& keys, const Triple& values,
                   const MaybeTensor& positions, const MaybeTensor& cos, const MaybeTensor& sin, const MaybeTensor& axes,
                   bool interleaved) {
    const int dev = current(k);
    int64_t k_row = rows(k, dev), v_row = rows(v, dev);
    on_boundary(k, k_row, 16);
    on_boundary(v, v_row, 16);
    const int64_t N = k.size(0), KVH = k.size(1), D = k.size(2);
    const Pool p = pool(keys, values, k.scalar_type(), dev);
    need(v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() && KVH == p.KVH && D == p.D,
         "append: k and v do not fit the cache's heads and head_dim");
    ints(slots, dev);
    need(slots.dim() == 1 && slots.size(0) == N, "append: a slot a token expected");
    int64_t q_row = 0, H = 0;
    MaybeTensor qo;
    if (q) {
        q_row = rows(*q, dev);
        on_boundary(*q, q_row, 16);
        H = q->size(1);
        need(q->size(0) == N && q->size(2) == D && q->scalar_type() == k.scalar_type(),
             "append: q and k must have the same tokens, head_dim and dtype");
        qo = like(*q);
    }
    Angles a;
    if (positions) {
        need(cos.has_value() && sin.has_value(), "append: positions without cos and sin tables");
        a = angles(*positions, *cos, *sin, axes, N, D, dev);
    }
    if (N)
        run("lq_kv4_append",
            lq_kv4_append(q ? q->data_ptr() : nullptr, q_row, q ? qo->data_ptr() : nullptr, narrow(H), k.data_ptr(), k_row,
                          v.data_ptr(), v_row, p.KVH, narrow(N), p.D, a.rot, a.positions, a.cos, a.sin, a.max_pos, a.axes,
                          a.naxes, interleaved, slots.data_ptr<int32_t>(), p.kq, p.ks, p.kb, p.vq, p.vs, p.vb, p.pages, p.page,
                          dtype_code(k), stream()));
    return qo;
}

std::tuple<Tensor, Tensor> read_slots(const Triple& keys, const Triple& values, const Tensor& slots) {
    const int dev = current(slots);
    ints(slots, dev);
    need(slots.dim() == 1, "read: slots (N,) expected");
    const Tensor& scales = std::get<1>(keys);
    const Pool p = pool(keys, values, scales.scalar_type(), dev);
    const int64_t N = slots.size(0);
    Tensor ko = at::empty({N, p.KVH, p.D}, scales.options()), vo = at::empty({N, p.KVH, p.D}, scales.options());
    if (N)
        run("lq_kv4_read", lq_kv4_read(p.kq, p.ks, p.kb, p.vq, p.vs, p.vb, p.pages, p.page, p.KVH, p.D,
                                       slots.data_ptr<int32_t>(), narrow(N), ko.data_ptr(), vo.data_ptr(), dtype_code(scales),
                                       stream()));
    return {ko, vo};
}

Tensor attend(Tensor q, const Triple& keys, const Triple& values, const Tensor& table, const Tensor& lens, double scale,
              const MaybeTensor& q_start, int64_t max_q, MaybeTensor sinks, int64_t window) {
    const int dev = current(q);
    int64_t q_row = rows(q, dev);
    const int64_t N = q.size(0), H = q.size(1), D = q.size(2);
    if (q_row != H * D) q = q.contiguous(), q_row = H * D;
    on_boundary(q, q_row, 16);
    const Pool p = pool(keys, values, q.scalar_type(), dev);
    ints(table, dev);
    ints(lens, dev);
    need(D == p.D && p.KVH > 0 && H % p.KVH == 0, "attend: the queries' heads do not fit the cache's");
    need(lens.dim() == 1 && table.dim() == 2 && table.size(0) == lens.size(0), "attend: lens (B,), block_table (B, width)");
    const int64_t B = lens.size(0);
    if (q_start) {
        ints(*q_start, dev);
        need(q_start->dim() == 1 && q_start->size(0) == B + 1, "attend: q_start (B + 1,) expected");
    } else {
        need(N == B && max_q == 1, "attend: without q_start there is one query a request");
    }
    if (sinks) {
        if (sinks->scalar_type() != at::kFloat || !here(*sinks, dev) || !sinks->is_contiguous())
            sinks = sinks->to(q.options().dtype(at::kFloat)).contiguous();
        need(sinks->dim() == 1 && sinks->size(0) == H, "attend: a sink a head expected");
    }
    Tensor out = at::empty(q.sizes(), q.options());
    if (!N) return out;
    const size_t bytes =
        lq_kv4_attend_workspace(narrow(B), narrow(max_q), narrow(H), p.KVH, p.D, narrow(table.size(1)), p.page);
    Tensor ws;
    if (bytes) ws = at::empty({int64_t(bytes / 2)}, q.options());
    run("lq_kv4_attend",
        lq_kv4_attend(q.data_ptr(), narrow(N), q_start ? q_start->data_ptr<int32_t>() : nullptr, narrow(max_q), p.kq, p.ks, p.kb,
                      p.vq, p.vs, p.vb, p.pages, p.page, table.data_ptr<int32_t>(), narrow(table.size(1)),
                      lens.data_ptr<int32_t>(), narrow(B), sinks ? sinks->data_ptr<float>() : nullptr, float(scale),
                      narrow(window), narrow(H), p.KVH, p.D, dtype_code(q), bytes ? ws.data_ptr() : nullptr, bytes,
                      out.data_ptr(), stream()));
    return out;
}

#include "fp4_ext.h"

}  // namespace

PYBIND11_MODULE(_paged_ext, m) {
    m.def("plan", &plan);
    m.def("rotate", &rotate);
    m.def("append", &append);
    m.def("read", &read_slots);
    m.def("attend", &attend);
    m.def("fp4_quantize", &fp4::quantize);
    m.def("fp4_dequantize", &fp4::dequantize);
    m.def("fp4_product", &fp4::product);
    m.def("fp4_linear", &fp4::linear);
    m.def("fp4_grouped", &fp4::grouped);
    m.def("fp4_experts", &fp4::experts);
}
