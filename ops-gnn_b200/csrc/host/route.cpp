// Launch planners of topk_route (with its backward) and route_csr.  No counterpart in the reference.
#include <pybind11/pybind11.h>

#include "ops.h"

namespace opsgnn {
namespace {

OpsgnnRouteDesc RouteDescOf(const at::Tensor& logits, int64_t k, int64_t score, int64_t groups, int64_t kept_groups, int64_t group_top,
                            bool renormalize, double scale, const char* api)
{
    CheckCuda(logits, api, "logits");
    TORCH_CHECK(logits.dim() == 2 && logits.is_contiguous(), api, ": logits must be a contiguous [rows, experts] tensor");
    OpsgnnRouteDesc desc{};
    desc.rows = logits.size(0);
    desc.experts = logits.size(1);
    desc.k = k;
    desc.groups = groups;
    desc.kept_groups = kept_groups;
    desc.scale = static_cast<float>(scale);
    desc.group_top = static_cast<int32_t>(group_top);
    desc.score = static_cast<int32_t>(score);
    desc.renormalize = renormalize ? 1 : 0;
    desc.dtype = DtypeId(logits.scalar_type(), api);
    return desc;
}

}  // namespace

namespace {

// `undefined`: bytes, one per row, for the backward pass; may be null.
std::tuple<at::Tensor, at::Tensor> Forward(const at::Tensor& logits, const std::optional<at::Tensor>& bias, int64_t k, int64_t score,
                                           int64_t groups, int64_t kept_groups, int64_t group_top, bool renormalize, double scale,
                                           at::Tensor* undefined)
{
    const char* api = "topk_route";
    const OpsgnnRouteDesc desc = RouteDescOf(logits, k, score, groups, kept_groups, group_top, renormalize, scale, api);
    if (bias) {
        TORCH_CHECK(bias->device() == logits.device() && bias->scalar_type() == at::kFloat && bias->dim() == 1 &&
                        bias->size(0) == desc.experts && bias->is_contiguous(),
                    api, ": bias must be a contiguous float32 [experts] tensor on the GPU of logits");
    }
    c10::cuda::CUDAGuard guard(logits.device());
    at::Tensor weight = at::empty({desc.rows, k}, logits.options());
    at::Tensor index = at::empty({desc.rows, k}, logits.options().dtype(at::kLong));
    if (undefined != nullptr) {
        *undefined = at::empty({desc.rows}, logits.options().dtype(at::kByte));
    }
    CheckStatus(opsgnn_topk_route_recorded(&desc, logits.const_data_ptr(), bias ? bias->const_data_ptr<float>() : nullptr,
                                           weight.data_ptr(), index.data_ptr<int64_t>(),
                                           undefined != nullptr ? undefined->data_ptr<uint8_t>() : nullptr, CurrentStream(logits)),
                api);
    return {weight, index};
}

at::Tensor Backward(const at::Tensor& logits, const at::Tensor& index, const at::Tensor& undefined, const at::Tensor& grad_weight,
                    int64_t score, bool renormalize, double scale)
{
    const char* api = "topk_route backward";
    const OpsgnnRouteDesc desc = RouteDescOf(logits, index.size(-1), score, 1, 1, 1, renormalize, scale, api);
    TORCH_CHECK(index.device() == logits.device() && grad_weight.device() == logits.device() && index.scalar_type() == at::kLong &&
                    grad_weight.scalar_type() == logits.scalar_type() && index.is_contiguous() && grad_weight.is_contiguous() &&
                    index.dim() == 2 && index.size(0) == desc.rows && grad_weight.sizes() == index.sizes(),
                api, ": index and grad_weight must be contiguous [rows, k] tensors on the GPU of logits");
    c10::cuda::CUDAGuard guard(logits.device());
    at::Tensor grad_logits = at::empty_like(logits);
    CheckStatus(opsgnn_topk_route_backward_recorded(&desc, logits.const_data_ptr(), index.const_data_ptr<int64_t>(),
                                                    undefined.defined() ? undefined.const_data_ptr<uint8_t>() : nullptr,
                                                    grad_weight.const_data_ptr(), grad_logits.data_ptr(), CurrentStream(logits)),
                api);
    return grad_logits;
}

}  // namespace

std::tuple<at::Tensor, at::Tensor> topk_route_forward(const at::Tensor& logits, const std::optional<at::Tensor>& bias, int64_t k,
                                                      int64_t score, int64_t groups, int64_t kept_groups, int64_t group_top,
                                                      bool renormalize, double scale)
{
    return Forward(logits, bias, k, score, groups, kept_groups, group_top, renormalize, scale, nullptr);
}

at::Tensor topk_route_backward(const at::Tensor& logits, const at::Tensor& index, const at::Tensor& grad_weight, int64_t score,
                               bool renormalize, double scale)
{
    return Backward(logits, index, at::Tensor(), grad_weight, score, renormalize, scale);
}

namespace {

// The autograd node lives in C++: a router's pass is a few microseconds of GPU time, which a Python node would exceed.
class TopkRoute : public torch::autograd::Function<TopkRoute> {
public:
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits,
                                                  const std::optional<at::Tensor>& bias, int64_t k, int64_t score, int64_t groups,
                                                  int64_t kept_groups, int64_t group_top, bool renormalize, double scale)
    {
        at::Tensor undefined;
        const bool marks = score == OPSGNN_ROUTE_SOFTMAX && renormalize;
        auto [weight, index] =
            Forward(logits, bias, k, score, groups, kept_groups, group_top, renormalize, scale, marks ? &undefined : nullptr);
        ctx->save_for_backward({logits, index, undefined});
        ctx->saved_data["score"] = score;
        ctx->saved_data["renormalize"] = renormalize;
        ctx->saved_data["scale"] = scale;
        ctx->mark_non_differentiable({index});
        ctx->set_materialize_grads(false);
        return {weight, index};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads)
    {
        torch::autograd::variable_list out(9);
        if (grads[0].defined()) {
            PlannerScope scope;
            const auto saved = ctx->get_saved_variables();
            const at::Tensor grad = Backward(saved[0].detach(), saved[1], saved[2], grads[0].detach().contiguous(),
                                             ctx->saved_data["score"].toInt(), ctx->saved_data["renormalize"].toBool(),
                                             ctx->saved_data["scale"].toDouble());
            out[0] = OnceDifferentiable({grad}, "topk_route")[0];
        }
        return out;
    }
};

}  // namespace

std::tuple<at::Tensor, at::Tensor> topk_route(const at::Tensor& logits, const std::optional<at::Tensor>& bias, int64_t k, int64_t score,
                                              int64_t groups, int64_t kept_groups, int64_t group_top, bool renormalize, double scale)
{
    if (logits.requires_grad() && at::GradMode::is_enabled()) {
        const auto out = TopkRoute::apply(logits, bias, k, score, groups, kept_groups, group_top, renormalize, scale);
        return {out[0], out[1]};
    }
    return topk_route_forward(logits, bias, k, score, groups, kept_groups, group_top, renormalize, scale);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> route_csr(const at::Tensor& index, int64_t experts)
{
    const char* api = "route_csr";
    CheckCuda(index, api, "index");
    TORCH_CHECK(index.is_contiguous() && (index.scalar_type() == at::kInt || index.scalar_type() == at::kLong), api,
                ": index must be a contiguous int32 / int64 tensor");
    c10::cuda::CUDAGuard guard(index.device());
    const auto options = index.options().dtype(at::kLong);
    at::Tensor indptr = at::empty({experts + 1}, options);
    at::Tensor perm = at::empty({index.numel()}, options);
    at::Tensor position = at::empty(index.sizes(), options);
    int64_t bytes = 0;
    CheckStatus(opsgnn_route_csr_workspace_bytes(index.numel(), experts, &bytes), api);
    at::Tensor scratch;
    if (bytes > 0) {
        scratch = Scratch(bytes, index);
    }
    CheckStatus(opsgnn_route_csr(index.const_data_ptr(), DtypeId(index.scalar_type(), api), index.numel(), experts,
                                 indptr.data_ptr<int64_t>(), perm.data_ptr<int64_t>(), position.data_ptr<int64_t>(),
                                 bytes > 0 ? scratch.data_ptr() : nullptr, bytes, CurrentStream(index)),
                api);
    return {indptr, perm, position};
}

}  // namespace opsgnn

namespace py = pybind11;

void BindRoute(py::module_& m)
{
    m.def("topk_route", opsgnn::Scoped(&opsgnn::topk_route), py::arg("logits"), py::arg("bias"), py::arg("k"), py::arg("score"),
          py::arg("groups"), py::arg("kept_groups"), py::arg("group_top"), py::arg("renormalize"), py::arg("scale"),
          "topk_route_forward with its gradient; not part of the reference binding", py::call_guard<py::gil_scoped_release>());
    m.def("topk_route_forward", opsgnn::Scoped(&opsgnn::topk_route_forward), py::arg("logits"), py::arg("bias"), py::arg("k"),
          py::arg("score"), py::arg("groups"), py::arg("kept_groups"), py::arg("group_top"), py::arg("renormalize"), py::arg("scale"),
          "The k best experts of each row and their weights; not part of the reference binding",
          py::call_guard<py::gil_scoped_release>());
    m.def("topk_route_backward", opsgnn::Scoped(&opsgnn::topk_route_backward), py::arg("logits"), py::arg("index"),
          py::arg("grad_weight"), py::arg("score"), py::arg("renormalize"), py::arg("scale"),
          "Gradient of topk_route's weights; not part of the reference binding", py::call_guard<py::gil_scoped_release>());
    m.def("route_csr", opsgnn::Scoped(&opsgnn::route_csr), py::arg("index"), py::arg("experts"),
          "CSR structure (indptr, perm, position) of expert labels; not part of the reference binding",
          py::call_guard<py::gil_scoped_release>());
}
