// haste_amd._host.gated_mlp: the argument checks, outputs and autograd node of ops.gated_mlp.
#include "host_rows.hpp"

namespace haste_host {
namespace {

struct Weights {
    Rows gate, up, down;
    int64_t H, D, O;
    int code;
};
// Rows that the kernels take: no row for all, no pitch past 2^22.
Rows matrix_of(const at::Tensor& t, int64_t cols) {
    Rows r = rows_of(t, cols);
    if (r.ld == 0 || r.ld > (1 << 22)) r = rows_of(r.t.contiguous(), cols);
    return r;
}
Weights weights_of(const at::Tensor& gate, const at::Tensor& up, const at::Tensor& down) {
    const int64_t H = gate.size(0), D = gate.size(1), O = down.size(0);
    return Weights{matrix_of(gate, D), matrix_of(up, D),
                   matrix_of(down, H), H,
                   D,                  O,
                   dtype_code(gate.scalar_type())};
}

// Whether the kernels take all of these rows where they lie (16-bit: on 16 bytes, both projections at one
// pitch).
bool aligned(const Weights& w, std::initializer_list<const Rows*> rows) {
    if (w.gate.ld != w.up.ld) return false;
    for (const Rows* r : rows)
        if (reinterpret_cast<uintptr_t>(ptr(r->t)) % 16 != 0 || r->ld % 8 != 0 || r->t.size(1) % 8 != 0)
            return false;
    return true;
}

at::Tensor workspace(int64_t N, const Weights& w, bool backward, bool is_aligned,
                     const at::TensorOptions& options, int64_t* size) {
    *size = haste_gated_mlp_workspace_size(N, w.D, w.H, w.O, w.code, backward, is_aligned);
    TORCH_CHECK(*size >= 0, haste_last_error());
    return *size ? at::empty({*size}, options.dtype(at::kByte)) : at::Tensor();
}

struct Forward {
    at::Tensor y, kept, h;
};
Forward forward(const at::Tensor& x, const at::Tensor& gate, const at::Tensor& up,
                const at::Tensor& down, int act, bool keep) {
    const Weights w = weights_of(gate, up, down);
    const Rows r = matrix_of(x, w.D);
    const int64_t N = r.t.size(0), ld = (w.H + 15) / 16 * 16;
    const auto options = at::TensorOptions().dtype(x.scalar_type()).device(x.device());
    Forward f;
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = w.O;
    f.y = at::empty(shape, options);
    // (fp32: three bf16 parts)
    const bool wide = x.scalar_type() == at::kFloat;
    f.h = at::empty({wide ? 3 * N : N, ld}, wide ? options.dtype(at::kBFloat16) : options);
    if (keep) {
        const int64_t bytes = haste_gated_mlp_kept_size(N, w.H, w.code);
        TORCH_CHECK(bytes >= 0, haste_last_error());
        f.kept = at::empty({bytes}, options.dtype(at::kByte));
    }
    int64_t size;
    const at::Tensor ws =
        workspace(N, w, false, aligned(w, {&r, &w.gate, &w.up, &w.down}), options, &size);
    call(haste_gated_mlp(ptr(r.t), r.ld, ptr(w.gate.t), w.gate.ld, ptr(w.up.t), w.up.ld, ptr(w.down.t),
                         w.down.ld, out_ptr(f.y), out_ptr(f.kept), out_ptr(f.h), N,
                         w.D, w.H, w.O, act, w.code, out_ptr(ws), size, stream_of(x)));
    return f;
}

enum { kX, kGate, kUp, kDown };  // the node's inputs

struct GatedMlp : torch::autograd::Function<GatedMlp> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& gate,
                              const at::Tensor& up, const at::Tensor& down, int64_t act) {
        Forward f = haste_host::forward(x, gate, up, down, (int)act, true);
        ctx->save_for_backward({x, gate, up, down, f.kept, f.h});
        ctx->set_materialize_grads(false);
        return f.y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(5);
        if (!grads[0].defined()) return out;
        check_gradients("gated_mlp", grads);
        // (what the engine wants now: autograd.grad may ask for fewer than require one)
        const bool need_x = ctx->needs_input_grad(kX), need_gate = ctx->needs_input_grad(kGate),
                   need_up = ctx->needs_input_grad(kUp), need_down = ctx->needs_input_grad(kDown);
        const variable_list saved = ctx->get_saved_variables();
        {
            const at::AutoGradMode off(false);
            const Weights w = weights_of(saved[1], saved[2], saved[3]);
            const Rows x = matrix_of(saved[0], w.D), dy = matrix_of(grads[0], w.O);
            const int64_t N = x.t.size(0);
            const auto options =
                at::TensorOptions().dtype(x.t.scalar_type()).device(x.t.device());
            at::Tensor dx, dg, du, dd;
            if (need_x) dx = at::empty(saved[0].sizes(), options);
            if (need_gate || need_up) {
                dg = at::empty({w.H, w.D}, options);
                du = at::empty({w.H, w.D}, options);
            }
            if (need_down) dd = at::empty({w.O, w.H}, options);
            int64_t size;
            const at::Tensor ws =
                workspace(N, w, true, aligned(w, {&x, &dy, &w.gate, &w.up, &w.down}), options, &size);
            call(haste_gated_mlp_bwd(ptr(x.t), x.ld, ptr(w.gate.t), w.gate.ld, ptr(w.up.t), w.up.ld,
                                     ptr(w.down.t), w.down.ld, ptr(dy.t), dy.ld, ptr(saved[4]),
                                     ptr(saved[5]), out_ptr(dx), out_ptr(dg),
                                     out_ptr(du), out_ptr(dd), N, w.D, w.H, w.O, w.code, out_ptr(ws),
                                     size, stream_of(x.t)));
            out[0] = dx;
            if (need_gate) out[1] = dg;
            if (need_up) out[2] = du;
            out[3] = dd;
        }
        once_differentiable("gated_mlp", out);
        return out;
    }
};

void check(const at::Tensor& x, const at::Tensor& gate, const at::Tensor& up, const at::Tensor& down) {
    check_not_traced("gated_mlp");
    check_no_tangent("gated_mlp", {&x, &gate, &up, &down});
    check_device(x, "x");
    TORCH_CHECK(dtype_code(x.scalar_type()) >= 0, "unsupported dtype ", x.scalar_type());
    TORCH_CHECK(x.dim() >= 1, "gated_mlp: x must have a last axis");
    for (const auto& [t, name] : {std::pair<const at::Tensor&, const char*>(gate, "w_gate"),
                                  std::pair<const at::Tensor&, const char*>(up, "w_up"),
                                  std::pair<const at::Tensor&, const char*>(down, "w_down")}) {
        check_device(t, name);
        TORCH_CHECK(t.scalar_type() == x.scalar_type() && t.device() == x.device(), "gated_mlp: ", name,
                    " must be ", x.scalar_type(), " on ", x.device(), " (got ", t.scalar_type(), " on ",
                    t.device(), ")");
        TORCH_CHECK(t.dim() == 2 && t.numel() > 0, "gated_mlp: ", name,
                    " must be a matrix that is not empty (got ", t.sizes(), ")");
    }
    TORCH_CHECK(gate.sizes() == up.sizes(), "gated_mlp: w_gate and w_up must be of one shape (got ",
                gate.sizes(), " and ", up.sizes(), ")");
    TORCH_CHECK(x.size(-1) == gate.size(1), "gated_mlp: x has ", x.size(-1), " features, w_gate takes ",
                gate.size(1));
    TORCH_CHECK(down.size(1) == gate.size(0), "gated_mlp: w_down takes ", down.size(1),
                " features, w_gate gives ", gate.size(0));
}

}  // namespace

PyObject* gated_mlp(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(count == 5, "gated_mlp: x, w_gate, w_up, w_down and activation are expected");
    const at::Tensor x = tensor_arg(args[0], "x", false);
    const at::Tensor gate = tensor_arg(args[1], "w_gate", false);
    const at::Tensor up = tensor_arg(args[2], "w_up", false);
    const at::Tensor down = tensor_arg(args[3], "w_down", false);
    const int64_t act = PyLong_AsLongLong(args[4]);
    if (PyErr_Occurred()) return nullptr;
    at::Tensor y;
    {
        pybind11::gil_scoped_release no_gil;
        check(x, gate, up, down);
        const c10::DeviceGuard guard(x.device());
        const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || gate.requires_grad() ||
                                                         up.requires_grad() || down.requires_grad());
        y = grad ? GatedMlp::apply(x, gate, up, down, act)
                 : forward(x, gate, up, down, (int)act, false).y;
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

}  // namespace haste_host
