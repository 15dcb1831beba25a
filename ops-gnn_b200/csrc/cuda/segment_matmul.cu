// C ABI of the segment products: argument checks and the choice of a kernel.
#include <algorithm>

#include "segment_matmul.cuh"

namespace opsgnn {
namespace segmm {
namespace {

bool FloatType(int t) { return t == OPSGNN_F32 || t == OPSGNN_F16 || t == OPSGNN_BF16; }

int CheckDesc(const OpsgnnSegmentMatmulDesc* d, bool eight_bits)
{
    if (d == nullptr || d->rows < 0 || d->segments < 0 || d->width < 0 || d->out < 0 || d->src_stride < d->width) {
        return OPSGNN_ERR_INVALID;
    }
    if (d->index_type != OPSGNN_I32 && d->index_type != OPSGNN_I64) {
        return OPSGNN_ERR_INVALID;
    }
    if (eight_bits ? (d->in_type != OPSGNN_F8E4M3 || !FloatType(d->out_type)) : (!FloatType(d->in_type) || d->out_type != d->in_type)) {
        return OPSGNN_ERR_UNSUPPORTED;
    }
    return OPSGNN_OK;
}

// fp32 products that go through bf16 terms on the tensor cores.  Making the terms costs launches and passes over the operands,
// which small products do not earn back: forward 4096 x 128 -> 128 (134 MFLOP) 13.1 us against 11.2 us on the simple kernel,
// 16384 x 101 -> 77 (255 MFLOP) 20.8 against 27.4 us, 32768 x 501 -> 333 157 against 586 us.  The simple weight gradient also
// grows with the rows a block sums alone, a segment's: 1024 x 128 -> 128 in 8 segments 12.5 us in terms against 12.0 us, in one 32 against
// 76; 2000 rows in 8 segments 16 against 21, 4096 x 64 -> 64 20.1 against 38.7.  (Below 2048 rows one long segment could gain, but a
// gradient of src computed alone would no longer have the bits of one computed together with the weight's.)
bool Splits(const OpsgnnSegmentMatmulDesc& d, int what)
{
    if (d.in_type != OPSGNN_F32 || d.rows <= 0 || d.segments <= 0 || d.width <= 0 || d.out <= 0) {
        return false;
    }
    const double flops = 2.0 * static_cast<double>(d.rows) * static_cast<double>(d.width) * static_cast<double>(d.out);
    return flops >= 2e8 || (what != OPSGNN_SEGMENT_MATMUL_FORWARD && d.rows >= 2048);
}

// 16-bit products, which may be summed in pieces.
bool Pieces(const OpsgnnSegmentMatmulDesc& d)
{
    return d.in_type != OPSGNN_F32 && d.rows > 0 && d.segments > 0 && d.width > 0 && d.out > 0;
}

SegmentPointers Pointers(const OpsgnnSegmentMatmulDesc& d, const void* indptr)
{
    SegmentPointers p;
    p.data = indptr;
    p.segments = indptr != nullptr ? d.segments : 1;
    p.rows = d.rows;
    p.wide = d.index_type == OPSGNN_I64;
    return p;
}

// The fastest kernel that takes the problem; fp32 goes through bf16 terms where there is a workspace for them.
int RunRows(const RowsProblem& p, void* workspace, cudaStream_t stream)
{
    int ran = OPSGNN_ERR_UNSUPPORTED;
    if (p.in_type != OPSGNN_F32) {
        ran = RunRowsTensor(p, workspace, stream);
    } else if (workspace != nullptr) {
        ran = RunRowsSplit(p, workspace, stream);
    }
    return ran == OPSGNN_ERR_UNSUPPORTED ? RunRowsSimple(p, stream) : ran;
}

int RunOuter(const OuterProblem& p, void* workspace, cudaStream_t stream)
{
    int ran = OPSGNN_ERR_UNSUPPORTED;
    if (p.type != OPSGNN_F32) {
        ran = RunOuterTensor(p, workspace, stream);
    } else if (workspace != nullptr) {
        ran = RunOuterSplit(p, workspace, stream);
    }
    return ran == OPSGNN_ERR_UNSUPPORTED ? RunOuterSimple(p, stream) : ran;
}

}  // namespace
}  // namespace segmm
}  // namespace opsgnn

using namespace opsgnn;

extern "C" int opsgnn_segment_matmul_workspace_bytes(const OpsgnnSegmentMatmulDesc* desc, int what, int64_t* bytes)
{
    const int status = segmm::CheckDesc(desc, false);
    if (status != OPSGNN_OK) {
        return status;
    }
    if (bytes == nullptr) {
        return OPSGNN_ERR_INVALID;
    }
    const int64_t rows = desc->rows, segments = desc->segments, width = desc->width, out = desc->out;
    const bool split = segmm::Splits(*desc, what);
    *bytes = 0;
    if (what == OPSGNN_SEGMENT_MATMUL_FORWARD) {
        *bytes = split ? segmm::RowsSplitBytes(rows, segments, width, out)
                       : (segmm::Pieces(*desc) ? segmm::RowsPartialBytes(rows, segments, width, out) : 0);
    } else if (what == OPSGNN_SEGMENT_MATMUL_WEIGHT_GRAD) {
        *bytes = split ? segmm::OuterSplitBytes(rows, segments, width, out)
                       : (segmm::Pieces(*desc) ? segmm::OuterPartialBytes(rows, segments, width, out) : 0);
    } else if (what == OPSGNN_SEGMENT_MATMUL_GRADS) {
        *bytes = split ? segmm::GradsSplitBytes(rows, segments, width, out)
                       : (segmm::Pieces(*desc) ? std::max({segmm::RowsPartialBytes(rows, segments, out, width),
                                                           segmm::OuterPartialBytes(rows, segments, width, out),
                                                           segmm::OuterPartialBytes(rows, segments, out, width)})
                                               : 0);
    } else {
        return OPSGNN_ERR_INVALID;
    }
    return OPSGNN_OK;
}

extern "C" int opsgnn_segment_matmul(const OpsgnnSegmentMatmulDesc* desc, const void* indptr, const void* src, const void* weight,
                                     void* out, void* workspace, int64_t workspace_bytes, void* stream)
{
    int64_t need = 0;
    const int status = opsgnn_segment_matmul_workspace_bytes(desc, OPSGNN_SEGMENT_MATMUL_FORWARD, &need);
    if (status != OPSGNN_OK) {
        return status;
    }
    if (desc->rows == 0 || desc->out == 0) {
        return OPSGNN_OK;
    }
    if (indptr == nullptr || out == nullptr || ((src == nullptr || weight == nullptr) && desc->width > 0 && desc->segments > 0)) {
        return OPSGNN_ERR_INVALID;
    }
    segmm::RowsProblem p{};
    p.ptr = segmm::Pointers(*desc, indptr);
    p.a = src;
    p.b = weight;
    p.out = out;
    p.k = desc->width;
    p.n = desc->out;
    p.lda = desc->src_stride;
    p.ldo = desc->out;
    p.b_segment = desc->weight_segment_stride;
    p.b_k = desc->weight_width_stride;
    p.b_n = desc->weight_out_stride;
    p.in_type = desc->in_type;
    p.out_type = desc->out_type;
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !Aligned(workspace, 16))) {
        return OPSGNN_ERR_WORKSPACE;
    }
    return segmm::RunRows(p, need > 0 ? workspace : nullptr, AsStream(stream));
}

extern "C" int opsgnn_segment_matmul_weight_grad(const OpsgnnSegmentMatmulDesc* desc, const void* indptr, const void* src,
                                                 const void* grad, int64_t grad_stride, void* grad_weight, void* workspace,
                                                 int64_t workspace_bytes, void* stream)
{
    int64_t need = 0;
    const int status = opsgnn_segment_matmul_workspace_bytes(desc, OPSGNN_SEGMENT_MATMUL_WEIGHT_GRAD, &need);
    if (status != OPSGNN_OK) {
        return status;
    }
    if (desc->segments == 0 || desc->width == 0 || desc->out == 0) {
        return OPSGNN_OK;
    }
    if (indptr == nullptr || grad_weight == nullptr || grad_stride < desc->out || ((src == nullptr || grad == nullptr) && desc->rows > 0)) {
        return OPSGNN_ERR_INVALID;
    }
    segmm::OuterProblem p{};
    p.ptr = segmm::Pointers(*desc, indptr);
    p.a = src;
    p.b = grad;
    p.out = grad_weight;
    p.k = desc->width;
    p.n = desc->out;
    p.lda = desc->src_stride;
    p.ldb = grad_stride;
    p.type = desc->in_type;
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !Aligned(workspace, 16))) {
        return OPSGNN_ERR_WORKSPACE;
    }
    return segmm::RunOuter(p, need > 0 ? workspace : nullptr, AsStream(stream));
}

extern "C" int opsgnn_segment_matmul_grads(const OpsgnnSegmentMatmulDesc* desc, const void* indptr, const void* src, const void* weight,
                                           const void* grad, int64_t grad_stride, void* grad_src, void* grad_weight, int turned,
                                           void* workspace, int64_t workspace_bytes, void* stream)
{
    int64_t need = 0;
    const int status = opsgnn_segment_matmul_workspace_bytes(desc, OPSGNN_SEGMENT_MATMUL_GRADS, &need);
    if (status != OPSGNN_OK) {
        return status;
    }
    if (indptr == nullptr || grad_stride < desc->out) {
        return OPSGNN_ERR_INVALID;
    }
    const bool rows = desc->rows > 0 && desc->width > 0, outer = desc->segments > 0 && desc->width > 0 && desc->out > 0;
    const bool sums = desc->out > 0 && desc->segments > 0;
    if ((rows && (grad_src == nullptr || (sums && (grad == nullptr || weight == nullptr)))) ||
        (outer && (grad_weight == nullptr || (desc->rows > 0 && (src == nullptr || grad == nullptr))))) {
        return OPSGNN_ERR_INVALID;
    }
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !Aligned(workspace, 16))) {
        return OPSGNN_ERR_WORKSPACE;
    }
    segmm::RowsProblem p{};
    p.ptr = segmm::Pointers(*desc, indptr);
    p.a = grad;
    p.b = weight;
    p.out = grad_src;
    p.k = desc->out;
    p.n = desc->width;
    p.lda = grad_stride;
    p.ldo = desc->width;
    p.b_segment = desc->weight_segment_stride;
    p.b_k = desc->weight_out_stride;
    p.b_n = desc->weight_width_stride;
    p.in_type = desc->in_type;
    p.out_type = desc->out_type;
    segmm::OuterProblem q{};
    q.ptr = p.ptr;
    q.a = turned ? grad : src;
    q.b = turned ? src : grad;
    q.out = grad_weight;
    q.k = turned ? desc->out : desc->width;
    q.n = turned ? desc->width : desc->out;
    q.lda = turned ? grad_stride : desc->src_stride;
    q.ldb = turned ? desc->src_stride : grad_stride;
    q.type = desc->in_type;
    if (rows && outer && segmm::Splits(*desc, OPSGNN_SEGMENT_MATMUL_GRADS)) {
        const int ran = segmm::RunGradsSplit(p, q, turned != 0, workspace, AsStream(stream));
        if (ran != OPSGNN_ERR_UNSUPPORTED) {
            return ran;
        }
    }
    // fp32 that cannot be split goes through the simple kernels: no workspace for it below
    void* scratch = need > 0 && !segmm::Splits(*desc, OPSGNN_SEGMENT_MATMUL_GRADS) ? workspace : nullptr;
    int ran = rows ? segmm::RunRows(p, scratch, AsStream(stream)) : OPSGNN_OK;
    if (ran == OPSGNN_OK && outer) {
        ran = segmm::RunOuter(q, scratch, AsStream(stream));
    }
    return ran;
}

extern "C" int opsgnn_segment_matmul_fp8(const OpsgnnSegmentMatmulDesc* desc, const void* indptr, const void* src, const float* src_scale,
                                         const void* weight, const float* weight_scale, void* out, void* stream)
{
    const int status = segmm::CheckDesc(desc, true);
    if (status != OPSGNN_OK) {
        return status;
    }
    if (desc->rows == 0 || desc->out == 0) {
        return OPSGNN_OK;
    }
    if (out == nullptr || (indptr == nullptr && desc->segments != 1) ||
        ((src == nullptr || src_scale == nullptr || weight == nullptr || weight_scale == nullptr) && desc->width > 0 && desc->segments > 0)) {
        return OPSGNN_ERR_INVALID;
    }
    segmm::RowsProblem p{};
    p.ptr = segmm::Pointers(*desc, indptr);
    p.a = src;
    p.b = weight;
    p.out = out;
    p.a_scale = src_scale;
    p.b_scale = weight_scale;
    p.k = desc->width;
    p.n = desc->out;
    p.lda = desc->src_stride;
    p.ldo = desc->out;
    p.b_segment = desc->weight_segment_stride;
    p.b_k = desc->weight_width_stride;
    p.b_n = desc->weight_out_stride;
    p.in_type = desc->in_type;
    p.out_type = desc->out_type;
    const int ran = segmm::RunRowsFp8(p, AsStream(stream));
    return ran == OPSGNN_ERR_UNSUPPORTED ? segmm::RunRowsSimple(p, AsStream(stream)) : ran;
}
