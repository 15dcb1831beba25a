// Launch planners of the segment products (16 / 32 bits with both gradients, 8 bits with block scales) and of quantize_fp8.
// No counterpart in the reference.  The pointers are never read on the host: the kernels find their tiles on the device and
// clamp what they read, so a call neither synchronises nor reads back and can be captured into a graph.
#include <c10/cuda/CUDAException.h>
#include <cuda_runtime_api.h>
#include <pybind11/pybind11.h>

#include "ops.h"

namespace opsgnn {
namespace {

// A stall of an earlier launch raises here, but not while a graph is captured: the look allocates pinned memory on a device's
// first use.
void LookForStalls(const at::Tensor& t, const char* api)
{
    cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
    C10_CUDA_CHECK(cudaStreamIsCapturing(c10::cuda::getCurrentCUDAStream(t.device().index()).stream(), &capturing));
    if (capturing == cudaStreamCaptureStatusNone) {
        RaiseIfDeviceStalled(t, api);
    }
}

// A matrix whose rows are runs of consecutive elements, at any row distance.
at::Tensor RowMajor(const at::Tensor& t)
{
    const bool fine = (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1));
    return fine ? t : t.contiguous();
}

int64_t RowStride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : std::max<int64_t>(t.size(1), 1); }

// [segments, width, out] with `width` or `out` running along memory and no overlap; anything else is copied.
at::Tensor Matrices(const at::Tensor& t)
{
    const int64_t e = t.size(0), k = t.size(1), n = t.size(2);
    if (t.numel() == 0) {
        return t.contiguous();
    }
    const bool out_fast = (n == 1 || t.stride(2) == 1) && (k == 1 || t.stride(1) >= n);
    const bool width_fast = (k == 1 || t.stride(1) == 1) && (n == 1 || t.stride(2) >= k);
    const int64_t extent = (k - 1) * t.stride(1) + (n - 1) * t.stride(2) + 1;
    return (out_fast || width_fast) && (e == 1 || t.stride(0) >= extent) ? t : t.contiguous();
}

// The tensor cores' loads want rows on 16-byte boundaries.  A product of this many multiply-adds or more is worth a copy of an
// operand that has them elsewhere; smaller ones run as they are, on the kernel for any layout.  bf16 forward, as it is and with both
// operands copied: 32768 x 33 -> 33 (3.6e7) 16 and 25 us, 4096 x 101 -> 77 in 20 segments (3.2e7) 16 and 16 us, 256 x 333 -> 501
// (4.3e7) 28 and 17 us; 2100 x 130 -> 641 (1.7e8) 48 and 27 us.
constexpr double kWorthCopy = 5e7;

bool Wants(const at::Tensor& rows, int64_t width, int64_t out)
{
    return rows.scalar_type() != at::kFloat &&
           static_cast<double>(rows.size(0)) * static_cast<double>(width) * static_cast<double>(out) >= kWorthCopy;
}
bool Wants(const at::Tensor& rows, const at::Tensor& matrices) { return Wants(rows, matrices.size(1), matrices.size(2)); }

// A weight gradient on the kernel for any layout is one block's sum over all rows of a segment, 70 ns a row, however few the
// columns, so there the copies also pay for long segments.  How long these are the host does not know: the mean tells where lengths
// are alike, and from so many rows on one long segment would cost more than the copies.  bf16 33 -> 33, as it is and with copies:
// 512 rows in one segment 38 and 18 us, 64 rows 7 and 14 us; 1024 rows in 8 segments 11 and 15 us, 4096 rows 38 and 18 us; 32768
// rows in 64 segments 38 and 22 us, in 500 segments 18 and 49 us, in one 2238 and 41 us.
bool WantsWeightGrad(const at::Tensor& rows, int64_t segments, int64_t width, int64_t out)
{
    const int64_t m = rows.size(0);
    return Wants(rows, width, out) || (rows.scalar_type() != at::kFloat && ((m >= 256 && m >= 128 * segments) || m >= 16384));
}

// Rows (the last dimension or, `turned`, the one before it) on 16-byte boundaries?
bool IsOnBoundaries(const at::Tensor& t, bool turned = false)
{
    const int64_t vec = 16 / t.element_size(), inner = turned ? t.dim() - 2 : t.dim() - 1;
    bool fine = reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
    for (int64_t d = 0; d < t.dim(); ++d) {
        fine = fine && (d == inner || t.size(d) <= 1 || t.stride(d) % vec == 0);
    }
    return fine;
}

// t itself, or a copy with rows on 16-byte boundaries.
at::Tensor OnBoundaries(const at::Tensor& t, bool turned = false)
{
    if (IsOnBoundaries(t, turned)) {
        return t;
    }
    const int64_t vec = 16 / t.element_size();
    at::Tensor from = turned ? t.transpose(-1, -2) : t;
    auto shape = from.sizes().vec();
    const int64_t width = shape.back();
    shape.back() = (width + vec - 1) / vec * vec;
    at::Tensor copy = at::empty(shape, t.options()).narrow(-1, 0, width);
    copy.copy_(from);
    return turned ? copy.transpose(-1, -2) : copy;
}

bool Turned(const at::Tensor& matrices) { return matrices.size(1) > 1 && matrices.stride(1) == 1 && matrices.stride(2) != 1; }

OpsgnnSegmentMatmulDesc DescOf(const at::Tensor& src, const std::optional<at::Tensor>& indptr, int64_t segments, int64_t out,
                               at::ScalarType out_type, const char* api)
{
    OpsgnnSegmentMatmulDesc desc{};
    desc.rows = src.size(0);
    desc.segments = segments;
    desc.width = src.size(1);
    desc.out = out;
    desc.src_stride = std::max(RowStride(src), src.size(1));
    desc.index_type = indptr ? DtypeId(indptr->scalar_type(), api) : OPSGNN_I64;
    desc.in_type = src.scalar_type() == at::kFloat8_e4m3fn ? OPSGNN_F8E4M3 : DtypeId(src.scalar_type(), api);
    desc.out_type = DtypeId(out_type, api);
    return desc;
}

void SetWeight(OpsgnnSegmentMatmulDesc& desc, const at::Tensor& matrices)
{
    // Strides of dimensions of one element say nothing; give them the values of a contiguous layout.
    const int64_t k = matrices.size(1), n = matrices.size(2);
    const bool width_fast = k > 1 && matrices.stride(1) == 1 && (n == 1 || matrices.stride(2) >= k);
    desc.weight_width_stride = k > 1 ? matrices.stride(1) : (width_fast ? 1 : std::max<int64_t>(n, 1));
    desc.weight_out_stride = n > 1 ? matrices.stride(2) : (width_fast ? std::max<int64_t>(k, 1) : 1);
    desc.weight_segment_stride = matrices.size(0) > 1 ? matrices.stride(0) : std::max<int64_t>(k * n, 1);
}

void CheckPointers(const at::Tensor& indptr, const at::Tensor& src, int64_t segments, const char* api)
{
    TORCH_CHECK(indptr.device() == src.device() && indptr.dim() == 1 && indptr.is_contiguous() && indptr.numel() == segments + 1 &&
                    (indptr.scalar_type() == at::kInt || indptr.scalar_type() == at::kLong),
                api, ": indptr must be a contiguous int32 / int64 vector of segments + 1 pointers on the GPU of src");
}

}  // namespace

at::Tensor segment_matmul_forward(const at::Tensor& src, const at::Tensor& indptr, const at::Tensor& weight)
{
    const char* api = "segment_matmul";
    CheckCuda(src, api, "src");
    TORCH_CHECK(src.dim() == 2 && weight.dim() == 3 && weight.size(1) == src.size(1) && weight.scalar_type() == src.scalar_type() &&
                    weight.device() == src.device(),
                api, ": src must be [rows, width] and weight [segments, width, out] of one dtype on one GPU");
    CheckPointers(indptr, src, weight.size(0), api);
    c10::cuda::CUDAGuard guard(src.device());
    LookForStalls(src, api);
    at::Tensor rows = RowMajor(src), matrices = Matrices(weight);
    if (Wants(rows, matrices)) {
        rows = OnBoundaries(rows);
        matrices = OnBoundaries(matrices, Turned(matrices));
    }
    at::Tensor out = at::empty({src.size(0), weight.size(2)}, src.options());
    OpsgnnSegmentMatmulDesc desc = DescOf(rows, indptr, weight.size(0), weight.size(2), src.scalar_type(), api);
    SetWeight(desc, matrices);
    int64_t bytes = 0;
    CheckStatus(opsgnn_segment_matmul_workspace_bytes(&desc, OPSGNN_SEGMENT_MATMUL_FORWARD, &bytes), api);
    const at::Tensor scratch = bytes > 0 ? Scratch(bytes, src) : at::Tensor();
    CheckStatus(opsgnn_segment_matmul(&desc, indptr.const_data_ptr(), rows.const_data_ptr(), matrices.const_data_ptr(), out.data_ptr(),
                                      bytes > 0 ? scratch.data_ptr() : nullptr, bytes, CurrentStream(src)),
                api);
    return out;
}

at::Tensor segment_matmul_weight_grad(const at::Tensor& src, const at::Tensor& indptr, const at::Tensor& grad)
{
    const char* api = "segment_matmul backward";
    CheckCuda(src, api, "src");
    TORCH_CHECK(src.dim() == 2 && grad.dim() == 2 && grad.size(0) == src.size(0) && grad.scalar_type() == src.scalar_type() &&
                    grad.device() == src.device() && indptr.numel() >= 1,
                api, ": src and grad must be [rows, width] and [rows, out] of one dtype on one GPU");
    const int64_t segments = indptr.numel() - 1;
    CheckPointers(indptr, src, segments, api);
    c10::cuda::CUDAGuard guard(src.device());
    LookForStalls(src, api);
    at::Tensor rows = RowMajor(src), upstream = RowMajor(grad);
    if (WantsWeightGrad(rows, segments, src.size(1), grad.size(1))) {
        rows = OnBoundaries(rows);
        upstream = OnBoundaries(upstream);
    }
    at::Tensor out = at::empty({segments, src.size(1), grad.size(1)}, src.options());
    const OpsgnnSegmentMatmulDesc desc = DescOf(rows, indptr, segments, grad.size(1), src.scalar_type(), api);
    int64_t bytes = 0;
    CheckStatus(opsgnn_segment_matmul_workspace_bytes(&desc, OPSGNN_SEGMENT_MATMUL_WEIGHT_GRAD, &bytes), api);
    const at::Tensor scratch = bytes > 0 ? Scratch(bytes, src) : at::Tensor();
    CheckStatus(opsgnn_segment_matmul_weight_grad(&desc, indptr.const_data_ptr(), rows.const_data_ptr(), upstream.const_data_ptr(),
                                                  std::max(RowStride(upstream), upstream.size(1)), out.data_ptr(),
                                                  bytes > 0 ? scratch.data_ptr() : nullptr, bytes, CurrentStream(src)),
                api);
    return out;
}

namespace {

// grad_src and, in the layout of weight, grad_weight.
std::vector<at::Tensor> Gradients(const at::Tensor& src, const at::Tensor& indptr, const at::Tensor& weight, const at::Tensor& grad)
{
    const char* api = "segment_matmul backward";
    c10::cuda::CUDAGuard guard(src.device());
    LookForStalls(src, api);
    at::Tensor rows = RowMajor(src), matrices = Matrices(weight), upstream = RowMajor(grad);
    if (Wants(rows, matrices)) {
        rows = OnBoundaries(rows);
        matrices = OnBoundaries(matrices, Turned(matrices));
        upstream = OnBoundaries(upstream);
    }
    const bool turned = weight.stride(1) == 1 && weight.stride(2) != 1;
    OpsgnnSegmentMatmulDesc desc = DescOf(rows, indptr, weight.size(0), weight.size(2), src.scalar_type(), api);
    SetWeight(desc, matrices);
    at::Tensor grad_src = at::empty(src.sizes(), src.options());
    at::Tensor grad_weight = turned ? at::empty({weight.size(0), weight.size(2), weight.size(1)}, src.options())
                                    : at::empty(weight.sizes(), src.options());
    int64_t bytes = 0;
    CheckStatus(opsgnn_segment_matmul_workspace_bytes(&desc, OPSGNN_SEGMENT_MATMUL_GRADS, &bytes), api);
    const at::Tensor scratch = bytes > 0 ? Scratch(bytes, src) : at::Tensor();
    CheckStatus(opsgnn_segment_matmul_grads(&desc, indptr.const_data_ptr(), rows.const_data_ptr(), matrices.const_data_ptr(),
                                            upstream.const_data_ptr(), std::max(RowStride(upstream), upstream.size(1)),
                                            grad_src.data_ptr(), grad_weight.data_ptr(), turned ? 1 : 0,
                                            bytes > 0 ? scratch.data_ptr() : nullptr, bytes, CurrentStream(src)),
                api);
    return {grad_src, turned ? grad_weight.transpose(1, 2) : grad_weight};
}

class SegmentMatmul : public torch::autograd::Function<SegmentMatmul> {
public:
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& src, const at::Tensor& indptr,
                              const at::Tensor& weight)
    {
        ctx->save_for_backward({src, indptr, weight});
        return segment_matmul_forward(src, indptr, weight);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads)
    {
        PlannerScope scope;
        const auto saved = ctx->get_saved_variables();
        const bool of_src = ctx->needs_input_grad(0), of_weight = ctx->needs_input_grad(2);
        const at::Tensor indptr = saved[1], weight = saved[2].detach(), grad = RowMajor(grads[0].detach());
        const at::Tensor src = of_weight ? RowMajor(saved[0].detach()) : saved[0].detach();
        // Together, unless only the weight's wants copies: the gradient of src has the bits that it has alone.
        const bool together = of_src && of_weight &&
                              (Wants(src, weight) == WantsWeightGrad(src, weight.size(0), weight.size(1), weight.size(2)) ||
                               (IsOnBoundaries(src) && IsOnBoundaries(grad)));
        std::vector<at::Tensor> out(2);
        if (together) {
            out = Gradients(src, indptr, weight, grad);
        }
        if (of_src && !together) {
            out[0] = segment_matmul_forward(grad, indptr, weight.transpose(1, 2));
        }
        if (of_weight && !together) {  // in the layout of the weight
            out[1] = weight.stride(1) == 1 && weight.stride(2) != 1 ? segment_matmul_weight_grad(grad, indptr, src).transpose(1, 2)
                                                                    : segment_matmul_weight_grad(src, indptr, grad);
        }
        out = OnceDifferentiable(std::move(out), "segment_matmul");
        return {out[0], at::Tensor(), out[1]};
    }
};

}  // namespace

at::Tensor segment_matmul(const at::Tensor& src, const at::Tensor& indptr, const at::Tensor& weight)
{
    if (at::GradMode::is_enabled() && (src.requires_grad() || weight.requires_grad())) {
        return SegmentMatmul::apply(src, indptr, weight);
    }
    return segment_matmul_forward(src, indptr, weight);
}

at::Tensor segment_matmul_fp8(const at::Tensor& src, const at::Tensor& src_scale, const at::Tensor& weight,
                              const at::Tensor& weight_scale, const std::optional<at::Tensor>& indptr, at::ScalarType out_type)
{
    const char* api = "segment_matmul_fp8";
    CheckCuda(src, api, "src");
    TORCH_CHECK(src.dim() == 2 && weight.dim() == 3 && weight.size(2) == src.size(1) && src.scalar_type() == at::kFloat8_e4m3fn &&
                    weight.scalar_type() == at::kFloat8_e4m3fn,
                api, ": src must be [rows, width] and weight [segments, out, width], both float8_e4m3fn");
    for (const auto& tensor : {src_scale, weight, weight_scale}) {
        TORCH_CHECK(tensor.device() == src.device(), api, ": inputs must be on the same GPU");
    }
    const int64_t segments = weight.size(0), blocks = (src.size(1) + 127) / 128, bands = (weight.size(1) + 127) / 128;
    TORCH_CHECK(src_scale.scalar_type() == at::kFloat && src_scale.dim() == 2 && src_scale.size(0) == src.size(0) &&
                    src_scale.size(1) == blocks && weight_scale.scalar_type() == at::kFloat && weight_scale.dim() == 3 &&
                    weight_scale.size(0) == segments && weight_scale.size(1) == bands && weight_scale.size(2) == blocks,
                api, ": scales must be float32, one for each 128 columns of a row of src and each tile of 128 x 128 of weight");
    if (indptr) {
        CheckPointers(*indptr, src, segments, api);
    } else {
        TORCH_CHECK(segments == 1, api, ": without indptr there is one weight");
    }
    c10::cuda::CUDAGuard guard(src.device());
    LookForStalls(src, api);
    at::Tensor rows = RowMajor(src), matrices = weight.contiguous();
    if (Wants(rows, matrices)) {
        rows = OnBoundaries(rows);
        matrices = OnBoundaries(matrices);
    }
    const at::Tensor row_scale = src_scale.contiguous(), tile_scale = weight_scale.contiguous();
    at::Tensor out = at::empty({src.size(0), weight.size(1)}, src.options().dtype(out_type));
    OpsgnnSegmentMatmulDesc desc = DescOf(rows, indptr, segments, weight.size(1), out_type, api);
    desc.weight_width_stride = 1;
    desc.weight_out_stride = matrices.stride(1);
    desc.weight_segment_stride = matrices.stride(0);
    CheckStatus(opsgnn_segment_matmul_fp8(&desc, indptr ? indptr->const_data_ptr() : nullptr, rows.const_data_ptr(),
                                          row_scale.const_data_ptr<float>(), matrices.const_data_ptr(),
                                          tile_scale.const_data_ptr<float>(), out.data_ptr(), CurrentStream(src)),
                api);
    return out;
}

std::tuple<at::Tensor, at::Tensor> quantize_fp8(const at::Tensor& src, int64_t block_rows)
{
    const char* api = "quantize_fp8";
    CheckCuda(src, api, "src");
    TORCH_CHECK(src.dim() >= 2 && src.is_contiguous() && (block_rows == 1 || block_rows == 128), api,
                ": src must be contiguous with at least two dimensions, block_rows 1 or 128");
    c10::cuda::CUDAGuard guard(src.device());
    const int64_t rows = src.size(-2), width = src.size(-1), batch = Product(src.sizes(), 0, src.dim() - 2);
    auto shape = src.sizes().vec();
    shape[shape.size() - 2] = (rows + block_rows - 1) / block_rows;
    shape[shape.size() - 1] = (width + 127) / 128;
    at::Tensor values = at::empty(src.sizes(), src.options().dtype(at::kFloat8_e4m3fn));
    at::Tensor scale = at::empty(shape, src.options().dtype(at::kFloat));
    CheckStatus(opsgnn_quantize_fp8(src.const_data_ptr(), DtypeId(src.scalar_type(), api), batch, rows, width,
                                    static_cast<int>(block_rows), values.data_ptr(), scale.data_ptr<float>(), CurrentStream(src)),
                api);
    return {values, scale};
}

}  // namespace opsgnn

namespace py = pybind11;

void BindSegmentMatmul(py::module_& m)
{
    m.def("segment_matmul", opsgnn::Scoped(&opsgnn::segment_matmul), py::arg("src"), py::arg("indptr"), py::arg("weight"),
          "segment_matmul_forward with both gradients; not part of the reference binding", py::call_guard<py::gil_scoped_release>());
    m.def("segment_matmul_forward", opsgnn::Scoped(&opsgnn::segment_matmul_forward), py::arg("src"), py::arg("indptr"),
          py::arg("weight"), "out[r] = src[r] @ weight[segment of r]; not part of the reference binding",
          py::call_guard<py::gil_scoped_release>());
    m.def("segment_matmul_weight_grad", opsgnn::Scoped(&opsgnn::segment_matmul_weight_grad), py::arg("src"), py::arg("indptr"),
          py::arg("grad"), "out[e] = src[rows of e]^T @ grad[rows of e]; not part of the reference binding",
          py::call_guard<py::gil_scoped_release>());
    m.def(
        "segment_matmul_fp8",
        [](const at::Tensor& src, const at::Tensor& src_scale, const at::Tensor& weight, const at::Tensor& weight_scale,
           const std::optional<at::Tensor>& indptr, int64_t out_type) {
            opsgnn::PlannerScope scope;
            return opsgnn::segment_matmul_fp8(src, src_scale, weight, weight_scale, indptr,
                                              out_type == OPSGNN_F32 ? at::kFloat : (out_type == OPSGNN_F16 ? at::kHalf : at::kBFloat16));
        },
        py::arg("src"), py::arg("src_scale"), py::arg("weight"), py::arg("weight_scale"), py::arg("indptr"), py::arg("out_type"),
        "Block-scaled float8_e4m3 segment product; not part of the reference binding", py::call_guard<py::gil_scoped_release>());
    m.def("quantize_fp8", opsgnn::Scoped(&opsgnn::quantize_fp8), py::arg("src"), py::arg("block_rows"),
          "float8_e4m3 values and their block scales; not part of the reference binding", py::call_guard<py::gil_scoped_release>());
}
