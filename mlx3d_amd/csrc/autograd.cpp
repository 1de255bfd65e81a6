// autograd.cpp -- the field layers' nodes of torch's autograd graph: what allocates
// their tensors, calls the gsx entry points and hands gradients on.
//
// A node that is written in Python costs a small step more than its kernels: autograd
// runs the backward pass on a thread of its own, where every Python object is another
// core's.  Forward and gradient, us, nodes in Python and here (a node in Python that does
// nothing takes 36 to 42): dropout of 64 x 64 on a residual 88 / 52, layer norm of 23 751
// x 27 with three gradients 116 / 67, embedding of 20 tokens 96 / 52; forward alone 11, 12
// and 11 / 6, 7 and 6.
//
// Arguments are checked by the Python functions in front of these.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <atomic>
#include <limits>
#include <optional>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "gsx.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

namespace {

std::atomic<bool> timed{false};  // whether a StageTimer is active

// mlx3d_amd.profiling.stage(label), while a timer is active.
class Stage {
  public:
    explicit Stage(const char* label) {
        if (!timed.load(std::memory_order_relaxed)) return;
        py::gil_scoped_acquire gil;
        stage_ = new py::object(py::module_::import("mlx3d_amd.profiling").attr("stage")(label));
        stage_->attr("__enter__")();
    }
    ~Stage() {
        if (!stage_) return;
        py::gil_scoped_acquire gil;
        try {
            stage_->attr("__exit__")(py::none(), py::none(), py::none());
        } catch (py::error_already_set& e) {
            e.discard_as_unraisable("mlx3d_amd.profiling.stage");
        }
        delete stage_;
    }
    Stage(const Stage&) = delete;

  private:
    py::object* stage_ = nullptr;
};

// A status below zero; mlx3d_amd._lib.GsxError in Python.
struct Failure : std::runtime_error {
    using std::runtime_error::runtime_error;
};
// mlx3d_amd._lib.GsxError; never let go: the interpreter may have ended before statics do.
const py::object* gsx_error = nullptr;

int64_t check(int64_t status, const char* what) {
    if (status < 0)
        throw Failure(std::string(what) + " failed: " + gsx_strerror((int)status) + " (status " +
                      std::to_string(status) + ")");
    return status;
}

// t's last dimension as the entry points take it.  What 32 bits do not hold is refused here,
// as the entry points refuse what is too large, and before anything is copied or divided.
int width_of(const Tensor& t, const char* what) {
    const int64_t width = t.size(-1);
    if (width > std::numeric_limits<int32_t>::max()) check(GSX_ERR_TOO_LARGE, what);
    return (int)width;
}

int dtype_of(const Tensor& t) {
    return t.scalar_type() == at::kFloat      ? GSX_F32
           : t.scalar_type() == at::kBFloat16 ? GSX_BF16
                                              : GSX_F16;
}
// The current stream of t's device, which is the current one where a Launch lives.
struct Launch {
    explicit Launch(const Tensor& t, const char* label)
        : guard(t.device()),
          stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()),
          stage(label) {}
    c10::DeviceGuard guard;
    void* stream;
    Stage stage;
};

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* ptr(const OptTensor& t) { return t ? ptr(*t) : nullptr; }
OptTensor contiguous(const OptTensor& t) { return t ? OptTensor(t->contiguous()) : t; }
Tensor contiguous_like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }
Tensor scratch(int64_t n, const Tensor& t) { return at::empty({n}, t.options().dtype(at::kByte)); }

// t (..., C) as (rows, C) with its row stride in elements; copied only if its last
// dimension is strided or its leading ones do not fold into one.
std::pair<Tensor, int64_t> rows_of(const Tensor& t) {
    const int64_t width = t.size(-1);
    if (t.is_contiguous()) return {t, width};
    Tensor r = t.reshape({-1, width});
    if ((r.size(0) > 1 && r.stride(0) < width) || (width > 1 && r.stride(1) != 1))
        r = r.contiguous();
    return {r, r.size(0) > 1 ? r.stride(0) : width};
}

// Hands a gradient on that was formed from `source`, too; differentiating it raises.
struct NoSecondDerivative : Function<NoSecondDerivative> {
    static Tensor forward(AutogradContext* ctx, const std::string& what, const Tensor& grad,
                          const Tensor&) {
        ctx->saved_data["what"] = what;
        return grad.view_as(grad);
    }
    static variable_list backward(AutogradContext* ctx, const variable_list&) {
        TORCH_CHECK(false, ctx->saved_data["what"].toStringRef(),
                    " has no second derivatives (once_differentiable).");
        return {};
    }
};

// A backward pass's gradients; with create_graph they depend on what they were formed
// from, and raise when they are differentiated.
variable_list once(const char* what, variable_list grads, const variable_list& incoming,
                   const variable_list& saved) {
    if (!at::GradMode::is_enabled()) return grads;
    for (Tensor& g : grads)
        for (const auto* from : {&incoming, &saved})
            for (const Tensor& t : *from)
                if (g.defined() && t.defined() && t.requires_grad())
                    g = NoSecondDerivative::apply(std::string(what), g, t);
    return grads;
}

// A node whose gradient is Op::gradient.  The engine, which calls backward, hands a Python
// error on as it is, and makes a RuntimeError of any other exception.
template <class Op>
struct Layer : Function<Op> {
    static variable_list backward(AutogradContext* ctx, const variable_list& incoming) {
        try {
            return Op::gradient(ctx, incoming);
        } catch (const Failure& e) {
            py::gil_scoped_acquire gil;
            PyErr_SetString(gsx_error->ptr(), e.what());
            python_error raised;
            raised.persist();
            throw raised;
        }
    }
};

// ---- embedding ----

struct Embedding : Layer<Embedding> {
    static Tensor forward(AutogradContext* ctx, const Tensor& indices, const Tensor& table,
                          double scale) {
        const int width = width_of(table, "gsx_embed_fwd");
        const Tensor held = indices.contiguous();
        const auto [rows, stride] = rows_of(table);
        std::vector<int64_t> shape = held.sizes().vec();
        shape.push_back(width);
        Tensor y = at::empty(shape, table.options());
        {
            const Launch on(table, "embed_fwd");
            check(gsx_embed_fwd(dtype_of(table), held.numel(), table.size(0), width, ptr(held),
                                held.scalar_type() == at::kLong, ptr(rows), stride, (float)scale,
                                ptr(y), on.stream),
                  "gsx_embed_fwd");
        }
        ctx->save_for_backward({indices});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["rows"] = table.size(0);
        return y;
    }
    static variable_list gradient(AutogradContext* ctx, const variable_list& incoming) {
        const variable_list saved = ctx->get_saved_variables();
        Tensor g_table;
        {
            const at::NoGradGuard no_grad;
            const Tensor& g_y = incoming[0];
            const int dtype = dtype_of(g_y), width = width_of(g_y, "gsx_embed_bwd");
            const Tensor held = saved[0].contiguous();
            const auto [g_rows, stride] = rows_of(g_y);
            const int64_t rows = ctx->saved_data["rows"].toInt(), count = held.numel();
            g_table = at::empty({rows, width}, g_y.options());
            const int64_t n = check(gsx_embed_bwd_workspace_bytes(dtype, count, rows, width),
                                    "gsx_embed_bwd_workspace_bytes");
            const Tensor ws = scratch(n, g_y);
            const Launch on(g_y, "embed_bwd");
            check(gsx_embed_bwd(dtype, count, rows, width, ptr(held),
                                held.scalar_type() == at::kLong, ptr(g_rows), stride,
                                (float)ctx->saved_data["scale"].toDouble(), ptr(g_table), ptr(ws),
                                n, on.stream),
                  "gsx_embed_bwd");
        }
        return once("embedding", {Tensor(), g_table, Tensor()}, incoming, saved);
    }
};

// ---- layer norm ----

struct LayerNorm : Layer<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight,
                          const OptTensor& bias, double eps) {
        const int width = width_of(x, "gsx_layer_norm_fwd");
        const auto [rows, stride] = rows_of(x);
        const OptTensor w = contiguous(weight), b = contiguous(bias);
        Tensor y = contiguous_like(x);
        {
            const Launch on(x, "layer_norm_fwd");
            check(gsx_layer_norm_fwd(dtype_of(x), x.numel() / width, width, ptr(rows), stride,
                                     ptr(w), ptr(b), (float)eps, ptr(y), on.stream),
                  "gsx_layer_norm_fwd");
        }
        ctx->save_for_backward({x, weight ? *weight : Tensor()});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["bias"] = bias.has_value();
        return y;
    }
    static variable_list gradient(AutogradContext* ctx, const variable_list& incoming) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &g_y = incoming[0];
        // inputs that are tensors are counted, absent ones are not
        const bool has_w = weight.defined(), has_b = ctx->saved_data["bias"].toBool();
        const bool need_w = has_w && ctx->needs_input_grad(1);
        const bool need_b = has_b && ctx->needs_input_grad(1 + has_w);
        Tensor g_x, g_w, g_b;
        {
            const at::NoGradGuard no_grad;
            const int dtype = dtype_of(x), width = width_of(x, "gsx_layer_norm_bwd");
            const auto [rows, stride] = rows_of(x);
            const auto [g_rows, g_stride] = rows_of(g_y);
            const Tensor w = has_w ? weight.contiguous() : weight;
            const int64_t count = x.numel() / width;
            if (ctx->needs_input_grad(0)) g_x = contiguous_like(x);
            if (need_w) g_w = at::empty({width}, x.options());
            if (need_b) g_b = at::empty({width}, x.options());
            Tensor ws;
            int64_t n = 0;
            if (need_w || need_b) {
                n = check(gsx_layer_norm_bwd_workspace_bytes(dtype, count, width),
                          "gsx_layer_norm_bwd_workspace_bytes");
                ws = scratch(n, x);
            }
            const Launch on(x, "layer_norm_bwd");
            check(gsx_layer_norm_bwd(dtype, count, width, ptr(rows), stride, ptr(w), ptr(g_rows),
                                     g_stride, (float)ctx->saved_data["eps"].toDouble(), ptr(g_x),
                                     ptr(g_w), ptr(g_b), ptr(ws), n, on.stream),
                  "gsx_layer_norm_bwd");
        }
        return once("layer_norm", {g_x, g_w, g_b, Tensor()}, incoming, saved);
    }
};

// ---- dropout ----

Tensor drop(const Tensor& x, const OptTensor& residual, double p, int64_t seed, int64_t offset,
            const Tensor& at_device) {
    const Tensor held = x.contiguous();
    const OptTensor base = contiguous(residual);
    Tensor y = contiguous_like(x);
    const Launch on(x, "dropout");
    check(gsx_dropout(dtype_of(x), held.numel(), p, (uint64_t)seed, offset,
                      (const int64_t*)ptr(at_device), ptr(held), ptr(base), ptr(y), on.stream),
          "gsx_dropout");
    return y;
}

struct Dropout : Layer<Dropout> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& residual,
                          double p, int64_t seed, int64_t offset, const OptTensor& at_device) {
        const Tensor at = at_device ? *at_device : Tensor();
        // saved, so that a counter that moves on before the gradient is noticed
        ctx->save_for_backward({at});
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["offset"] = offset;
        ctx->saved_data["residual"] = residual.has_value();
        return drop(x, residual, p, seed, offset, at);
    }
    static variable_list gradient(AutogradContext* ctx, const variable_list& incoming) {
        const variable_list saved = ctx->get_saved_variables();
        Tensor g_x, g_residual;
        {
            const at::NoGradGuard no_grad;
            if (ctx->needs_input_grad(0))
                g_x = drop(incoming[0], std::nullopt, ctx->saved_data["p"].toDouble(),
                           ctx->saved_data["seed"].toInt(), ctx->saved_data["offset"].toInt(),
                           saved[0]);
        }
        if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1))
            g_residual = incoming[0];
        return once("dropout", {g_x, g_residual, Tensor(), Tensor(), Tensor(), Tensor()}, incoming,
                    saved);
    }
};

}  // namespace

PYBIND11_MODULE(_autograd, m) {
    gsx_error = new py::object(py::module_::import("mlx3d_amd._lib").attr("GsxError"));
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Failure& e) {
            PyErr_SetString(gsx_error->ptr(), e.what());
        }
    });
    using Release = py::call_guard<py::gil_scoped_release>;
    m.def("set_timed", [](bool on) { timed = on; });
    m.def(
        "embedding",
        [](const Tensor& indices, const Tensor& table, double scale) {
            return Embedding::apply(indices, table, scale);
        },
        Release());
    m.def(
        "layer_norm",
        [](const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
            return LayerNorm::apply(x, weight, bias, eps);
        },
        Release());
    m.def(
        "dropout",
        [](const Tensor& x, const OptTensor& residual, double p, uint64_t seed, int64_t offset,
           const OptTensor& at_device) {
            return Dropout::apply(x, residual, p, (int64_t)seed, offset, at_device);
        },
        Release());
}
