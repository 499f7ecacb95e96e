// The token lookup as a node of torch's autograd: gs_embed_tokens forward, gs_embed_tokens_grad backward.
//
// It is C++ for its host time.  A backward pass over GPU tensors runs in a thread of autograd's own; this one and the caller's wake
// each other and start cold, so that every line of Python in a step counts twice: 512 tokens, 30522 rows of 384 fp32 values, a
// lookup and its gradient 84 us with a function of torch.autograd and 46 with this node, of which the kernels take 19.
//
// gpusparse/embedding.py checks the arguments before it comes here.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/version.h>

#include "gpusparse.h"

namespace {

using torch::autograd::variable_list;

// The exceptions that gpusparse._lib.check raises
void check(int rc, const char *what) {
    if (rc == GS_OK) return;
    TORCH_CHECK_VALUE(rc != GS_EINVAL, what, ": ", gs_last_error());
    TORCH_CHECK(false, what, " failed (", rc, "): ", gs_last_error());
}

void *stream_of(const at::Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

int type_of(const at::Tensor &t) {
    return t.scalar_type() == at::kFloat ? GS_H_F32 : t.scalar_type() == at::kHalf ? GS_H_F16 : GS_H_BF16;
}

gs_lookup lookup_of(const at::Tensor &ids, int64_t vocab, int64_t dim, int type, double scale, int64_t padding) {
    gs_lookup a{};
    a.ids_d = ids.const_data_ptr();
    a.tokens = ids.numel();
    a.padding = padding;
    a.id_bytes = (int32_t)ids.element_size();
    a.type = a.out_type = type;
    a.vocab = (int32_t)vocab;
    a.dim = (int32_t)dim;
    a.scale = (float)scale;
    return a;
}

// The gradient of a table of a's type and sizes; ids are contiguous.  grad: [..., dim] in any strides.
at::Tensor gradient(gs_lookup a, const at::Tensor &ids, at::Tensor grad) {
    const at::NoGradGuard no_grad;
    const c10::DeviceGuard on(grad.device());
    int64_t row = a.dim;
    if (!grad.is_contiguous()) {
        grad = grad.reshape({-1, a.dim});
        if (grad.stride(1) != 1) grad = grad.contiguous();
        row = grad.stride(0);
    }
    a.ids_d = ids.const_data_ptr();
    at::Tensor dweight = at::empty({a.vocab, a.dim}, grad.options()), workspace;
    size_t need = 0;
    check(gs_embed_tokens_grad_workspace(&a, &need), "gs_embed_tokens_grad_workspace");
    if (need) workspace = at::empty({(int64_t)need}, grad.options().dtype(at::kByte));
    check(gs_embed_tokens_grad(&a, grad.const_data_ptr(), row, dweight.mutable_data_ptr(), need ? workspace.mutable_data_ptr() : nullptr, need,
                               stream_of(grad)),
          "gs_embed_tokens_grad");
    return dweight;
}

struct EmbedTokensBackward : torch::autograd::Node {
    gs_lookup a;
    torch::autograd::SavedVariable ids;
    std::vector<int64_t> ids_shape;
    at::ScalarType ids_type;
    at::TensorOptions options;  // of the table

    variable_list apply(variable_list &&grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        if (!task_should_compute_output(0)) return {at::Tensor()};
        at::Tensor at_ids = ids.unpack();
        // hooks on saved tensors may move them, no more
        TORCH_CHECK(at_ids.sizes() == ids_shape && at_ids.scalar_type() == ids_type && at_ids.device() == options.device(),
                    "the saved ids came back as ", at_ids.scalar_type(), " ", at_ids.sizes(), " on ", at_ids.device());
        if (!grads[0].defined()) return {at::zeros({a.vocab, a.dim}, options)};  // as a function of torch.autograd would
        at::Tensor dweight = gradient(a, at_ids.contiguous(), grads[0]);
        if (!at::GradMode::is_enabled() || !grads[0].requires_grad()) return {dweight};
        // a second derivative is refused where it is asked for
        const auto refuse = std::make_shared<torch::autograd::DelayedError>("embed_tokens has first derivatives only", 1);
        return (*refuse)({dweight.detach().set_requires_grad(true)});
    }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        ids.reset_data();
    }
    std::string name() const override { return "EmbedTokensBackward"; }
};

// scale * weight[ids]; ids are contiguous.  Recorded where a gradient may be asked for.
at::Tensor embed_tokens(const at::Tensor &ids, const at::Tensor &weight, double scale, int64_t padding) {
    const c10::DeviceGuard on(weight.device());
    gs_lookup a = lookup_of(ids, weight.size(0), weight.size(1), type_of(weight), scale, padding);
    a.weight_d = weight.const_data_ptr();
    a.weight_row_stride = weight.stride(0);
    a.weight_dim_stride = weight.stride(1);
    c10::SmallVector<int64_t, 8> shape(ids.sizes().begin(), ids.sizes().end());
    shape.push_back(weight.size(1));
    at::Tensor out = at::empty(shape, weight.options());
    check(gs_embed_tokens(&a, out.mutable_data_ptr(), stream_of(weight)), "gs_embed_tokens");
    if (at::GradMode::is_enabled() && weight.requires_grad()) {
        const std::shared_ptr<EmbedTokensBackward> node(new EmbedTokensBackward, torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(weight));
        node->a = a;
        node->a.weight_d = nullptr;  // which the gradient does not read
        node->ids = torch::autograd::SavedVariable(ids, false);
        node->ids_shape = ids.sizes().vec();
        node->ids_type = ids.scalar_type();
        node->options = weight.options();
        torch::autograd::set_history(out, node);
    }
    return out;
}

// Its gradient alone; ids and grad [..., dim] of one device
at::Tensor embed_tokens_grad(const at::Tensor &ids, const at::Tensor &grad, int64_t vocab, double scale, int64_t padding) {
    return gradient(lookup_of(ids, vocab, grad.size(-1), type_of(grad), scale, padding), ids, grad);
}

}  // namespace

PYBIND11_MODULE(_autograd, m) {
    namespace py = pybind11;
    m.attr("ABI_VERSION") = GS_ABI_VERSION;
    m.attr("TORCH_VERSION") = TORCH_VERSION;
    m.def("embed_tokens", &embed_tokens, py::call_guard<py::gil_scoped_release>());
    m.def("embed_tokens_grad", &embed_tokens_grad, py::call_guard<py::gil_scoped_release>());
}
