// haste_amd._host.label_log_probs: the argument checks, outputs and autograd node of
// ops.label_log_probs.
#include "host_rows.hpp"

namespace haste_host {
namespace {

int label_bits(const at::Tensor& t) { return t.defined() && t.scalar_type() == at::kInt ? 32 : 64; }

struct Forward {
    at::Tensor stats, log_probs, entropy, top, top_labels;
};
Forward forward(const at::Tensor& logits, const at::Tensor& labels, int64_t top, bool with_stats) {
    const int64_t O = logits.size(-1), L = labels.defined() ? labels.size(-1) : 0;
    const Rows z = rows_of(logits, O);
    const int64_t B = z.t.size(0);
    const auto options = at::TensorOptions().dtype(at::kFloat).device(logits.device());
    std::vector<int64_t> shape = logits.sizes().vec();
    shape.pop_back();
    Forward f;
    f.entropy = at::empty(shape, options);
    if (with_stats) f.stats = at::empty({B, 2}, options);
    if (labels.defined()) f.log_probs = at::empty(labels.sizes(), options);
    if (top > 0) {
        shape.push_back(top);
        f.top = at::empty(shape, options);
        f.top_labels = at::empty(shape, options.dtype(at::kLong));
    }
    const int64_t size = haste_label_log_probs_workspace_size(B, O, (int32_t)top);
    TORCH_CHECK(size >= 0, "label_log_probs: logits too large (", logits.sizes(), ")");
    const at::Tensor ws = size ? at::empty({size}, options.dtype(at::kByte)) : at::Tensor();
    call(haste_label_log_probs(
        ptr(z.t), z.ld, ptr(labels), label_bits(labels), L, static_cast<float*>(out_ptr(f.stats)),
        static_cast<float*>(out_ptr(f.log_probs)), static_cast<float*>(out_ptr(f.entropy)),
        static_cast<float*>(out_ptr(f.top)), static_cast<int64_t*>(out_ptr(f.top_labels)), B, O,
        (int32_t)top, dtype_code(logits.scalar_type()), out_ptr(ws), size, stream_of(logits)));
    return f;
}

struct LabelLogProbs : torch::autograd::Function<LabelLogProbs> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& logits,
                                 const std::optional<at::Tensor>& labels_arg, int64_t top) {
        const at::Tensor labels = labels_arg.value_or(at::Tensor());
        Forward f = haste_host::forward(logits, labels, top, true);
        ctx->save_for_backward({logits, labels, f.stats, f.entropy});
        ctx->set_materialize_grads(false);
        variable_list out{f.entropy};
        if (labels.defined()) out.push_back(f.log_probs);
        if (top > 0) {
            ctx->mark_non_differentiable({f.top, f.top_labels});
            out.push_back(f.top);
            out.push_back(f.top_labels);
        }
        ctx->saved_data["labels"] = labels.defined();
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(3);
        check_gradients("label_log_probs", grads);
        const bool given = ctx->saved_data["labels"].toBool();
        const at::Tensor dent = dense(grads[0]), dlp = given ? dense(grads[1]) : at::Tensor();
        if (!dent.defined() && !dlp.defined()) return out;
        const variable_list saved = ctx->get_saved_variables();
        {
            const at::AutoGradMode off(false);
            const at::Tensor &logits = saved[0], &labels = saved[1];
            const int64_t O = logits.size(-1);
            const Rows z = rows_of(logits, O);
            // rows on 128-byte lines, like the logits that an FFI layer gives
            const int64_t ld = O % 8 ? (O + 63) / 64 * 64 : O;
            std::vector<int64_t> strides(logits.dim());
            int64_t step = ld;
            strides.back() = 1;
            for (int64_t k = logits.dim() - 2; k >= 0; --k) {
                strides[k] = step;
                step *= std::max<int64_t>(logits.size(k), 1);
            }
            out[0] = at::empty_strided(
                logits.sizes(), strides,
                at::TensorOptions().dtype(logits.scalar_type()).device(logits.device()));
            call(haste_label_log_probs_bwd(
                ptr(z.t), z.ld, ptr(labels), label_bits(labels), given ? labels.size(-1) : 0,
                static_cast<const float*>(ptr(saved[2])), static_cast<const float*>(ptr(saved[3])),
                static_cast<const float*>(ptr(dlp)), static_cast<const float*>(ptr(dent)),
                out_ptr(out[0]), ld, z.t.size(0), O, dtype_code(logits.scalar_type()),
                stream_of(logits)));
        }
        once_differentiable("label_log_probs", out);
        return out;
    }
};

void check(const at::Tensor& logits, const at::Tensor& labels, int64_t top) {
    check_not_traced("label_log_probs");
    check_no_tangent("label_log_probs", {&logits});
    check_device(logits, "logits");
    TORCH_CHECK(dtype_code(logits.scalar_type()) >= 0, "unsupported dtype ", logits.scalar_type());
    TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) >= 1,
                "label_log_probs: logits must have a last axis of labels (got ", logits.sizes(), ")");
    TORCH_CHECK(top >= 0 && top <= 128 && top <= logits.size(-1),
                "label_log_probs: top must be 0 to 128, and no more than the ", logits.size(-1),
                " labels (got ", top, ")");
    if (!labels.defined()) return;
    check_device(labels, "labels");
    TORCH_CHECK(labels.scalar_type() == at::kLong || labels.scalar_type() == at::kInt,
                "label_log_probs: labels must be int64 or int32 (got ", labels.scalar_type(), ")");
    TORCH_CHECK(labels.device() == logits.device(), "label_log_probs: labels are on ", labels.device(),
                ", logits on ", logits.device());
    TORCH_CHECK(labels.dim() == logits.dim() && labels.sizes().slice(0, labels.dim() - 1) ==
                                                    logits.sizes().slice(0, logits.dim() - 1),
                "label_log_probs: labels must be [..., L] for logits [..., O] (got ", labels.sizes(),
                " for ", logits.sizes(), ")");
    TORCH_CHECK(labels.size(-1) <= HASTE_MAX_GRAD_LABELS || !logits.requires_grad() ||
                    !at::GradMode::is_enabled(),
                "label_log_probs: at most ", HASTE_MAX_GRAD_LABELS, " labels a row with a gradient (got ",
                labels.size(-1), ")");
}

}  // namespace

PyObject* label_log_probs(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(count == 3, "label_log_probs: logits, labels and top are expected");
    const at::Tensor logits = tensor_arg(args[0], "logits", false);
    at::Tensor labels = tensor_arg(args[1], "labels", true);
    const int64_t top = PyLong_AsLongLong(args[2]);
    if (PyErr_Occurred()) return nullptr;
    Forward f;
    {
        pybind11::gil_scoped_release no_gil;
        check(logits, labels, top);
        const c10::DeviceGuard guard(logits.device());
        labels = dense(labels);
        if (at::GradMode::is_enabled() && logits.requires_grad()) {
            const variable_list out =
                LabelLogProbs::apply(logits, std::optional<at::Tensor>(labels), top);
            size_t k = 0;
            f.entropy = out[k++];
            if (labels.defined()) f.log_probs = out[k++];
            if (top > 0) {
                f.top = out[k++];
                f.top_labels = out[k++];
            }
        } else {
            f = forward(logits, labels, top, false);
        }
    }
    PyObject* all = PyTuple_New(4);
    if (!all) return nullptr;
    const at::Tensor* parts[] = {&f.log_probs, &f.entropy, &f.top, &f.top_labels};
    for (int k = 0; k < 4; ++k) {
        PyObject* o = parts[k]->defined() ? THPVariable_Wrap(*parts[k]) : Py_None;
        if (!o) {
            Py_DECREF(all);
            return nullptr;
        }
        if (o == Py_None) Py_INCREF(o);
        PyTuple_SET_ITEM(all, k, o);
    }
    return all;
    END_HANDLE_TH_ERRORS
}

}  // namespace haste_host
