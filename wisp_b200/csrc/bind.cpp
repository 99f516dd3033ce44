// Python binding of the stateless operators: checks, outputs, device and
// stream, then the C entry point of libwisp_b200.so (include/wisp_b200.h).
//
// A decode step's operators run for two to twenty microseconds.  The same
// checks in Python, two or three torch.empty calls and a ctypes call took
// eleven to fourteen; here they take about five.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cstdint>
#include <optional>
#include <string>
#include <tuple>

#include "../../include/wisp_b200.h"

namespace py = pybind11;
using at::Tensor;
using Maybe = std::optional<Tensor>;

namespace {

[[noreturn]] void value_error(const std::string &s) { throw py::value_error(s); }
[[noreturn]] void type_error(const std::string &s) { throw py::type_error(s); }

std::string shape_of(const Tensor &t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + ")";
}
int type_code(at::ScalarType t) {
    return t == at::kBFloat16 ? WISP_BF16 : t == at::kHalf ? WISP_FP16 : t == at::kFloat ? WISP_FP32 : -1;
}
// Sizes beyond 32 bits stay too large, for the library to refuse.
int32_t to_int(int64_t v) { return (int32_t)std::clamp<int64_t>(v, INT32_MIN, INT32_MAX); }
// The library's error, raised as its Python binding raises it.
void check(int rc, const char *what) {
    if (rc == WISP_OK) return;
    const py::gil_scoped_acquire gil;
    py::module_::import("wisp_b200._lib").attr("check")(rc, what);
}
void need_cuda(const char *name, const Tensor &t) {
    if (!t.is_cuda()) value_error(std::string(name) + " must be on a CUDA device; got " + t.device().str());
}
void same_device(const char *name, const Tensor &t, const Tensor &as) {
    if (t.device() != as.device())
        value_error(std::string(name) + " is on " + t.device().str() + ", not on " + as.device().str());
}
void *stream_of(const Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
// `given`, checked, or a new tensor.
Tensor output(const char *name, const Maybe &given, at::IntArrayRef shape, const at::TensorOptions &options) {
    if (!given) return at::empty(shape, options);
    if (given->sizes() != shape || given->scalar_type() != c10::typeMetaToScalarType(options.dtype()) ||
        !given->is_contiguous() || given->device() != options.device())
        value_error(std::string(name) + " must be a contiguous tensor of the result's shape, type and device; got " +
                    shape_of(*given));
    return *given;
}
// Rows [.., cols] of one stride (a copy where the strides do not allow that).
Tensor as_rows(const Tensor &t, int64_t cols, int64_t &stride) {
    stride = cols;
    if (t.is_contiguous()) return t;
    if (t.dim() == 2 && t.stride(1) == 1 && t.stride(0) >= 0) {
        stride = t.stride(0);
        return t;
    }
    return t.contiguous();
}
bool aligned16(const Tensor &t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
const void *ptr(const Maybe &t) { return t ? t->data_ptr() : nullptr; }

std::tuple<Tensor, Tensor> mx4_quantize(Tensor x, const Maybe &codes_out, const Maybe &scales_out) {
    need_cuda("x", x);
    const int dt = type_code(x.scalar_type());
    if (dt < 0) type_error("x must be bf16, fp16 or fp32");
    if (x.dim() < 1 || x.size(-1) == 0 || x.size(-1) % 32)
        value_error("the last axis of x must be a multiple of 32; got shape " + shape_of(x));
    const int64_t cols = x.size(-1), size = x.element_size();
    auto shape = x.sizes().vec();
    int64_t stride = cols;
    if (!x.is_contiguous()) {
        if (x.dim() == 2 && x.stride(1) == 1 && x.stride(0) >= cols && x.stride(0) * size % 16 == 0)
            stride = x.stride(0);
        else
            x = x.contiguous();
    }
    if (!aligned16(x)) {
        x = x.clone(at::MemoryFormat::Contiguous);
        stride = cols;
    }
    const c10::cuda::CUDAGuard guard(x.device());
    const auto bytes = x.options().dtype(at::kByte);
    shape.back() = cols / 2;
    Tensor codes = output("out.codes", codes_out, shape, bytes);
    shape.back() = cols / 32;
    Tensor scales = output("out.scales", scales_out, shape, bytes);
    check(wisp_mx4_quantize(x.data_ptr(), dt, x.numel() / cols, cols, stride, codes.data_ptr(), scales.data_ptr(),
                            stream_of(x)),
          "mx4_quantize");
    return {codes, scales};
}

Tensor mx4_dequantize(const Tensor &codes, const Tensor &scales, at::ScalarType dtype, const Maybe &out_) {
    need_cuda("q", codes);
    const int dt = type_code(dtype);
    if (dt < 0) type_error("dtype must be bf16, fp16 or fp32");
    if (!codes.is_contiguous() || !scales.is_contiguous()) value_error("mx4_dequantize takes contiguous matrices");
    const c10::cuda::CUDAGuard guard(codes.device());
    auto shape = codes.sizes().vec();
    const int64_t cols = shape.back() *= 2;
    Tensor out = output("out", out_, shape, codes.options().dtype(dtype));
    check(wisp_mx4_dequantize(codes.data_ptr(), scales.data_ptr(), out.numel() / cols, cols, out.data_ptr(), dt,
                              stream_of(codes)),
          "mx4_dequantize");
    return out;
}

Tensor mx4_matmul(const Tensor &a, const Tensor &a_scales, const Tensor &w, const Tensor &w_scales,
                  const Maybe &offsets, const Maybe &out_) {
    need_cuda("a", a);
    if (a.dim() != 2 || (w.dim() != 2 && w.dim() != 3) || w.size(-1) != a.size(1))
        value_error("a is [M, K], w [N, K] or [G, N, K]; got codes " + shape_of(a) + " and " + shape_of(w));
    if (!a.is_contiguous() || !a_scales.is_contiguous() || !w.is_contiguous() || !w_scales.is_contiguous())
        value_error("mx4_matmul takes contiguous matrices");
    const int64_t rows = a.size(0), n = w.size(-2), groups = w.dim() == 3 ? w.size(0) : 1;
    same_device("w", w, a);
    if (offsets) {
        same_device("offsets", *offsets, a);
        if (offsets->scalar_type() != at::kInt || offsets->dim() != 1 || offsets->size(0) != groups + 1 ||
            !offsets->is_contiguous())
            value_error("offsets must be a contiguous int32 [" + std::to_string(groups + 1) + "] tensor; got " +
                        shape_of(*offsets));
    } else if (groups != 1) {
        value_error(std::to_string(groups) + " groups need offsets");
    }
    const c10::cuda::CUDAGuard guard(a.device());
    Tensor out = output("out", out_, {rows, n}, a.options().dtype(at::kBFloat16));
    check(wisp_mx4_matmul(a.data_ptr(), a_scales.data_ptr(), rows, w.data_ptr(), w_scales.data_ptr(), to_int(groups),
                          to_int(n), to_int(2 * a.size(1)), reinterpret_cast<const int32_t *>(ptr(offsets)),
                          out.data_ptr(), stream_of(a)),
          "mx4_matmul");
    return out;
}

Tensor mx4_moe(Tensor x, const Tensor &w13, const Tensor &s13, const Tensor &w2, const Tensor &s2,
               std::optional<int64_t> top_k, const Maybe &router, bool renormalize, Maybe weights, Maybe ids,
               const Maybe &expert_map, const Maybe &out_) {
    need_cuda("x", x);
    if (x.scalar_type() != at::kBFloat16) type_error("mx4_moe computes from bf16 activations");
    if (x.dim() != 2 || w13.dim() != 3 || w2.dim() != 3) value_error("x is [T, H], w13 [S, 2I, H] and w2 [S, H, I]");
    const int64_t tokens = x.size(0), hidden = x.size(1), slots = w13.size(0), inter2 = w13.size(1);
    if (2 * w13.size(2) != hidden || inter2 % 2 || w2.size(0) != slots || w2.size(1) != hidden ||
        4 * w2.size(2) != inter2)
        value_error("shapes do not match: x " + shape_of(x) + ", codes of w13 " + shape_of(w13) + " and w2 " +
                    shape_of(w2));
    if (tokens > 64)
        value_error("mx4_moe takes at most 64 tokens a call; got " + std::to_string(tokens) +
                    " (mx4_quantize and mx4_matmul serve longer ones)");
    same_device("w13", w13, x);
    same_device("w2", w2, x);
    const int64_t experts = expert_map ? expert_map->numel() : slots;
    if (expert_map) {
        same_device("expert_map", *expert_map, x);
        if (expert_map->scalar_type() != at::kInt || !expert_map->is_contiguous())
            type_error("expert_map must be a contiguous int32 tensor");
    }
    if (router) {
        same_device("router", *router, x);
        if (ids || weights || !top_k) value_error("give either router and top_k, or topk_weights and topk_ids");
        if (router->scalar_type() != at::kBFloat16 || router->dim() != 2 || router->size(0) != experts ||
            router->size(1) != hidden || !router->is_contiguous())
            value_error("router must be a contiguous bf16 [" + std::to_string(experts) + ", " + std::to_string(hidden) +
                        "] tensor; got " + shape_of(*router));
    } else {
        if (!ids || !weights) value_error("give either router and top_k, or topk_weights and topk_ids");
        same_device("topk_ids", *ids, x);
        same_device("topk_weights", *weights, x);
        if (ids->scalar_type() != at::kInt && ids->scalar_type() != at::kLong)
            type_error("topk_ids must be int32 or int64");
        if (ids->dim() != 2 || ids->size(0) != tokens || weights->sizes() != ids->sizes())
            value_error("topk_ids and topk_weights are [T, k]");
        if (top_k && *top_k != ids->size(1))
            value_error("top_k is " + std::to_string(*top_k) + ", topk_ids " + shape_of(*ids));
        top_k = ids->size(1);
    }
    const c10::cuda::CUDAGuard guard(x.device());
    if (ids) {
        ids = ids->contiguous();
        weights = weights->to(at::kFloat).contiguous();
    }
    if (x.stride(1) != 1 || (tokens > 1 && (x.stride(0) < hidden || x.stride(0) % 8)) || !aligned16(x))
        x = x.clone(at::MemoryFormat::Contiguous);
    int64_t strides[4] = {w13.stride(0), s13.stride(0), w2.stride(0), s2.stride(0)};
    const bool packed = w13.is_contiguous() && s13.is_contiguous() && w2.is_contiguous() && s2.is_contiguous();
    Tensor out = output("out", out_, {tokens, hidden}, x.options());
    int64_t need = 0;
    check(wisp_mx4_moe_workspace(to_int(tokens), to_int(experts), to_int(*top_k), to_int(hidden),
                                 to_int(inter2 / 2), &need),
          "mx4_moe");
    Tensor ws = at::empty({need}, x.options().dtype(at::kByte));
    check(wisp_mx4_moe(x.data_ptr(), x.stride(0), ptr(router), ptr(ids), ids && ids->scalar_type() == at::kLong,
                       reinterpret_cast<const float *>(ptr(weights)), reinterpret_cast<const int32_t *>(ptr(expert_map)),
                       w13.data_ptr(), s13.data_ptr(), w2.data_ptr(), s2.data_ptr(), packed ? nullptr : strides,
                       to_int(slots), to_int(tokens), to_int(experts), to_int(*top_k), to_int(hidden),
                       to_int(inter2 / 2), renormalize, ws.data_ptr(), need, out.data_ptr(), stream_of(x)),
          "mx4_moe");
    return out;
}

void mx4_synchronize(int64_t device) {
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
    check(wisp_mx4_sync(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream()), "mx4_synchronize");
}

std::tuple<Tensor, Tensor> block_norm(const Tensor &y, const Tensor &residual, const Tensor &weight, const Maybe &post,
                                      Maybe gate, double scale, double eps, const Maybe &out_, const Maybe &res_out_) {
    need_cuda("y", y);
    const int dt = type_code(y.scalar_type()), rdt = type_code(residual.scalar_type()),
              wdt = type_code(weight.scalar_type());
    if (dt < 0) type_error("y must be bf16, fp16 or fp32");
    if ((rdt != dt && rdt != WISP_FP32) || (wdt != dt && wdt != WISP_FP32))
        type_error("residual and weight must have y's type or be fp32");
    if (y.dim() < 1 || residual.sizes() != y.sizes())
        value_error("residual must have y's shape " + shape_of(y) + "; got " + shape_of(residual));
    const int64_t cols = y.size(-1);
    if (weight.dim() != 1 || weight.size(0) != cols || !weight.is_contiguous())
        value_error("weight must be contiguous [" + std::to_string(cols) + "]; got " + shape_of(weight));
    same_device("residual", residual, y);
    same_device("weight", weight, y);
    if (post) {
        same_device("post_weight", *post, y);
        if (post->sizes() != weight.sizes() || !post->is_contiguous() || post->scalar_type() != weight.scalar_type())
            value_error("post_weight must be contiguous [" + std::to_string(cols) + "] of weight's type");
    }
    const c10::cuda::CUDAGuard guard(y.device());
    int kind = WISP_GATE_NONE;
    int64_t gate_stride = 0, y_stride = 0, res_stride = 0;
    if (gate) {
        same_device("gate", *gate, y);
        if (gate->scalar_type() != y.scalar_type()) type_error("gate must have y's type");
        if (gate->dim() == 1 && gate->size(0) == cols) {
            kind = WISP_GATE_CHANNEL;
            gate = gate->contiguous();
        } else if (gate->dim() == y.dim() && gate->size(-1) == 1 &&
                   gate->sizes().slice(0, gate->dim() - 1) == y.sizes().slice(0, y.dim() - 1)) {
            kind = WISP_GATE_TOKEN;
            if (gate->dim() == 2 && gate->stride(0) >= 0) {
                gate_stride = gate->stride(0);
            } else {
                gate = gate->contiguous();
                gate_stride = 1;
            }
        } else if (gate->sizes() == y.sizes()) {
            kind = WISP_GATE_FULL;
            gate = as_rows(*gate, cols, gate_stride);
        } else {
            value_error("gate must be [" + std::to_string(cols) + "], [..., 1] or [..., " + std::to_string(cols) +
                        "]; got " + shape_of(*gate));
        }
    }
    const Tensor yr = as_rows(y, cols, y_stride), rr = as_rows(residual, cols, res_stride);
    Tensor out = output("out", out_, y.sizes(), y.options());
    Tensor res_out = output("residual_out", res_out_, y.sizes(), residual.options());
    check(wisp_block_norm(yr.data_ptr(), y_stride, rr.data_ptr(), res_stride, weight.data_ptr(), ptr(post), ptr(gate), kind,
                          gate_stride, dt, rdt, wdt, cols ? out.numel() / cols : 0, to_int(cols), (float)scale,
                          (float)eps, out.data_ptr(), res_out.data_ptr(), stream_of(y)),
          "block_norm");
    return {out, res_out};
}

}  // namespace

// Without the interpreter's lock, as torch's own calls: a launch waits where the
// stream's queue is full, and what it waits for may need another Python thread.
PYBIND11_MODULE(_wisp_bind, m) {
    const auto unlocked = py::call_guard<py::gil_scoped_release>();
    m.def("mx4_quantize", &mx4_quantize, unlocked);
    m.def("mx4_dequantize", &mx4_dequantize, unlocked);
    m.def("mx4_matmul", &mx4_matmul, unlocked);
    m.def("mx4_moe", &mx4_moe, unlocked);
    m.def("mx4_synchronize", &mx4_synchronize, unlocked);
    m.def("block_norm", &block_norm, unlocked);
}
