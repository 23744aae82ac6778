// haste_amd._host.layer_norm: the argument checks, outputs and autograd node of ops.layer_norm.
// Made here and not in Python because a small norm's kernels take 4 to 20 us: a Python
// autograd Function took 60 to 130 us for forward and backward, whose thread then waits for the
// interpreter.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "host_rows.hpp"

namespace haste_host {
namespace {

void check(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias,
           const at::Tensor& residual) {
    check_not_traced("layer_norm");
    check_no_tangent("layer_norm", {&x, &weight, &bias, &residual});
    check_device(x, "x");
    TORCH_CHECK(dtype_code(x.scalar_type()) >= 0, "unsupported dtype ", x.scalar_type());
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1,
                "layer_norm: x must have a last axis to normalise (got ", x.sizes(), ")");
    for (const auto& [t, name] : {std::pair<const at::Tensor&, const char*>(weight, "weight"),
                                  std::pair<const at::Tensor&, const char*>(bias, "bias")}) {
        if (!t.defined()) continue;
        check_device(t, name);
        TORCH_CHECK(t.dim() == 1 && t.size(0) == x.size(-1), "layer_norm: ", name, " must be [",
                    x.size(-1), "] (got ", t.sizes(), ")");
        TORCH_CHECK(t.scalar_type() == weight.scalar_type() &&
                        (t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat),
                    "layer_norm: weight and bias must both be of x's dtype (", x.scalar_type(),
                    ") or float32 (got ", name, " ", t.scalar_type(), ")");
        TORCH_CHECK(t.device() == x.device(), "layer_norm: ", name, " is on ", t.device(), ", x on ",
                    x.device());
    }
    if (residual.defined()) {
        check_device(residual, "residual");
        TORCH_CHECK(residual.scalar_type() == x.scalar_type() && residual.device() == x.device(),
                    "layer_norm: residual must be ", x.scalar_type(), " on ", x.device(), " (got ",
                    residual.scalar_type(), " on ", residual.device(), ")");
    }
}

struct Forward {
    at::Tensor y, h, rows, weight, stats;
};
Forward forward(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias, double eps,
                const at::Tensor& residual, bool with_stats) {
    const int64_t D = x.size(-1);
    const Rows r = rows_of(x, D);
    Forward f;
    const auto options = at::TensorOptions().dtype(x.scalar_type()).device(x.device());
    f.weight = weight.is_neg() ? weight.resolve_neg().contiguous() : weight.contiguous();
    at::Tensor b;
    if (bias.defined()) b = bias.is_neg() ? bias.resolve_neg().contiguous() : bias.contiguous();
    f.y = at::empty(x.sizes(), options);
    Rows s;
    if (residual.defined()) {
        s = rows_of(residual, D);
        f.h = at::empty(x.sizes(), options);
    }
    const int64_t N = r.t.size(0);
    if (with_stats) f.stats = at::empty({N, 2}, options.dtype(at::kFloat));
    f.rows = f.h.defined() ? f.h : r.t;
    call(haste_layer_norm(ptr(r.t), r.ld, ptr(s.t), s.ld, ptr(f.weight), ptr(b), out_ptr(f.y),
                          out_ptr(f.h), static_cast<float*>(out_ptr(f.stats)), N, D, eps,
                          dtype_code(x.scalar_type()), dtype_code(weight.scalar_type()),
                          stream_of(x)));
    return f;
}

enum { kX = 1, kWeight = 2, kBias = 4, kResidual = 8 };

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x,
                                 const at::Tensor& weight,
                                 const std::optional<at::Tensor>& bias_arg, double eps,
                                 const std::optional<at::Tensor>& residual_arg) {
        const at::Tensor bias = bias_arg.value_or(at::Tensor()),
                         residual = residual_arg.value_or(at::Tensor());
        Forward f = haste_host::forward(x, weight, bias, eps, residual, true);
        ctx->save_for_backward({f.rows, f.weight, f.stats});
        ctx->set_materialize_grads(false);
        auto need = [](const at::Tensor& t, int bit) {
            return t.defined() && t.requires_grad() ? bit : 0;
        };
        ctx->saved_data["need"] = (int64_t)(need(x, kX) | need(weight, kWeight) |
                                            need(bias, kBias) | need(residual, kResidual));
        ctx->saved_data["shape"] = x.sizes().vec();
        if (!f.h.defined()) return {f.y};
        return {f.y, f.h};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_gradients("layer_norm", grads);
        at::Tensor dy = grads[0], dh = grads.size() > 1 ? grads[1] : at::Tensor();
        const int64_t need = ctx->saved_data["need"].toInt();
        const variable_list saved = ctx->get_saved_variables();
        variable_list out(5);
        at::Tensor dx, dw, db;
        {
            const at::AutoGradMode off(false);
            if (!dy.defined()) {  // only the sum's gradient: it passes through
                dx = dh;
            } else {
                const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
                const int64_t D = shape.back();
                const at::Tensor &weight = saved[1], &stats = saved[2];
                const Rows h = rows_of(saved[0], D), g = rows_of(dy, D);
                Rows s;
                if (dh.defined()) s = rows_of(dh, D);
                const int64_t N = h.t.size(0);
                const auto options =
                    at::TensorOptions().dtype(h.t.scalar_type()).device(h.t.device());
                if (need & (kX | kResidual)) dx = at::empty(shape, options);
                if (need & kWeight) dw = at::empty({D}, options.dtype(weight.scalar_type()));
                if (need & kBias) db = at::empty({D}, options.dtype(weight.scalar_type()));
                at::Tensor ws;
                int64_t size = 0;
                if (dw.defined() || db.defined()) {
                    size = haste_layer_norm_bwd_workspace_size(N, D);
                    ws = at::empty({size}, options.dtype(at::kByte));
                }
                call(haste_layer_norm_bwd(ptr(g.t), g.ld, ptr(s.t), s.ld, ptr(h.t), h.ld,
                                          ptr(weight), static_cast<const float*>(ptr(stats)),
                                          out_ptr(dx), out_ptr(dw), out_ptr(db), out_ptr(ws), size, N,
                                          D, dtype_code(h.t.scalar_type()),
                                          dtype_code(weight.scalar_type()), stream_of(h.t)));
            }
        }
        if (need & kX) out[0] = dx;
        if (need & kWeight) out[1] = dw;
        if (need & kBias) out[2] = db;
        if (need & kResidual) out[4] = dx;
        once_differentiable("layer_norm", out);
        return out;
    }
};

}  // namespace

PyObject* layer_norm(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(count == 5, "layer_norm: x, weight, bias, eps and residual are expected");
    const at::Tensor x = tensor_arg(args[0], "x", false);
    const at::Tensor weight = tensor_arg(args[1], "weight", false);
    const at::Tensor bias = tensor_arg(args[2], "bias", true);
    const double eps = PyFloat_AsDouble(args[3]);
    if (PyErr_Occurred()) return nullptr;
    at::Tensor residual = tensor_arg(args[4], "residual", true);
    at::Tensor y, h;
    {
        pybind11::gil_scoped_release no_gil;
        check(x, weight, bias, residual);
        const c10::DeviceGuard guard(x.device());
        if (residual.defined() && residual.sizes() != x.sizes())
            residual = residual.expand(x.sizes());
        auto grad = [](const at::Tensor& t) { return t.defined() && t.requires_grad(); };
        if (at::GradMode::is_enabled() &&
            (grad(x) || grad(weight) || grad(bias) || grad(residual))) {
            const variable_list out = LayerNorm::apply(x, weight, std::optional<at::Tensor>(bias), eps,
                                                       std::optional<at::Tensor>(residual));
            y = out[0];
            if (out.size() > 1) h = out[1];
        } else {
            Forward f = forward(x, weight, bias, eps, residual, false);
            y = f.y;
            h = f.h;
        }
    }
    return h.defined() ? pair_of(y, h) : THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

}  // namespace haste_host
