// haste_amd._host.embedding: the argument checks, outputs and autograd node of ops.embedding.
#include "host_rows.hpp"

namespace haste_host {
namespace {

int token_bits(const at::Tensor& t) { return t.scalar_type() == at::kLong ? 64 : 32; }

at::Tensor forward(const at::Tensor& tokens, const at::Tensor& weight, double scale) {
    const int64_t V = weight.size(0), D = weight.size(1);
    const Rows w = rows_of(weight, D);
    std::vector<int64_t> shape = tokens.sizes().vec();
    shape.push_back(D);
    at::Tensor y =
        at::empty(shape, at::TensorOptions().dtype(weight.scalar_type()).device(weight.device()));
    call(haste_embedding(ptr(tokens), token_bits(tokens), ptr(w.t), w.ld, out_ptr(y), tokens.numel(), V,
                         D, scale, dtype_code(weight.scalar_type()), stream_of(weight)));
    return y;
}

struct Embedding : torch::autograd::Function<Embedding> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& tokens, const at::Tensor& weight,
                              double scale, int64_t padding) {
        ctx->save_for_backward({tokens});
        ctx->set_materialize_grads(false);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["padding"] = padding;
        ctx->saved_data["rows"] = weight.size(0);
        return haste_host::forward(tokens, weight, scale);
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(4);
        if (!grads[0].defined()) return out;
        check_gradients("embedding", grads);
        const at::Tensor tokens = ctx->get_saved_variables()[0];
        {
            const at::AutoGradMode off(false);
            const int64_t V = ctx->saved_data["rows"].toInt(), D = grads[0].size(-1),
                          N = tokens.numel();
            const Rows dy = rows_of(grads[0], D);
            const auto options =
                at::TensorOptions().dtype(dy.t.scalar_type()).device(dy.t.device());
            out[1] = at::empty({V, D}, options);
            const int64_t size = haste_embedding_bwd_workspace_size(N, V, D);
            const at::Tensor ws = at::empty({size}, options.dtype(at::kByte));
            call(haste_embedding_bwd(ptr(tokens), token_bits(tokens), ptr(dy.t), dy.ld, out_ptr(out[1]),
                                     N, V, D, ctx->saved_data["scale"].toDouble(),
                                     ctx->saved_data["padding"].toInt(),
                                     dtype_code(dy.t.scalar_type()), out_ptr(ws), size,
                                     stream_of(dy.t)));
        }
        once_differentiable("embedding", out);
        return out;
    }
};

}  // namespace

PyObject* embedding(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(count == 4, "embedding: tokens, weight, scale and padding_idx are expected");
    at::Tensor tokens = tensor_arg(args[0], "tokens", false);
    const at::Tensor weight = tensor_arg(args[1], "weight", false);
    const double scale = PyFloat_AsDouble(args[2]);
    if (PyErr_Occurred()) return nullptr;
    int64_t padding = -1;
    if (args[3] != Py_None) {
        padding = PyLong_AsLongLong(args[3]);
        if (PyErr_Occurred()) return nullptr;
    }
    at::Tensor y;
    {
        pybind11::gil_scoped_release no_gil;
        check_not_traced("embedding");
        check_no_tangent("embedding", {&weight});
        check_device(weight, "weight");
        check_device(tokens, "tokens");
        TORCH_CHECK(tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt,
                    "embedding: tokens must be int64 or int32 (got ", tokens.scalar_type(), ")");
        TORCH_CHECK(tokens.device() == weight.device(), "embedding: tokens are on ", tokens.device(),
                    ", weight on ", weight.device());
        TORCH_CHECK(dtype_code(weight.scalar_type()) >= 0, "unsupported dtype ", weight.scalar_type());
        TORCH_CHECK(weight.dim() == 2 && weight.numel() > 0,
                    "embedding: weight must be [V, D] with V and D > 0 (got ", weight.sizes(), ")");
        if (args[3] != Py_None) {
            const int64_t V = weight.size(0);
            TORCH_CHECK(padding >= -V && padding < V, "embedding: padding_idx must be within the ", V,
                        " rows of weight (got ", padding, ")");
            if (padding < 0) padding += V;
        }
        const c10::DeviceGuard guard(weight.device());
        tokens = dense(tokens);
        y = at::GradMode::is_enabled() && weight.requires_grad()
                ? Embedding::apply(tokens, weight, scale, padding)
                : forward(tokens, weight, scale);
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

}  // namespace haste_host
