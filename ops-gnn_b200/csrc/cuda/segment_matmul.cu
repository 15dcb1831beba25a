// C ABI of the segment products: argument checks and the choice of a kernel.
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

// fp32 products that go through bf16 terms on the tensor cores, as far as sizes and strides say (a base address off 16 bytes
// sends the call to the simple kernel all the same).
bool Splits(const OpsgnnSegmentMatmulDesc& d)
{
    return d.in_type == OPSGNN_F32 && d.rows > 0 && d.segments > 0 && d.width > 0 && d.width % 8 == 0 && d.out > 0 && d.out % 8 == 0 &&
           d.src_stride % 4 == 0;
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

}  // namespace
}  // namespace segmm
}  // namespace opsgnn

using namespace opsgnn;

extern "C" int opsgnn_segment_matmul_workspace_bytes(const OpsgnnSegmentMatmulDesc* desc, int weight_grad, int64_t* bytes)
{
    const int status = segmm::CheckDesc(desc, false);
    if (status != OPSGNN_OK) {
        return status;
    }
    if (bytes == nullptr) {
        return OPSGNN_ERR_INVALID;
    }
    *bytes = 0;
    if (segmm::Splits(*desc)) {
        *bytes = weight_grad ? segmm::OuterSplitBytes(desc->rows, desc->segments, desc->width, desc->out)
                             : segmm::RowsSplitBytes(desc->rows, desc->segments, desc->width, desc->out);
    } else if (desc->in_type != OPSGNN_F32 && weight_grad && desc->rows > 0 && desc->segments > 0 && desc->width > 0 && desc->out > 0 &&
               desc->out % 8 == 0) {
        *bytes = segmm::OuterPartialBytes(desc->rows, desc->segments, desc->width, desc->out);
    }
    return OPSGNN_OK;
}

extern "C" int opsgnn_segment_matmul(const OpsgnnSegmentMatmulDesc* desc, const void* indptr, const void* src, const void* weight,
                                     void* out, void* workspace, int64_t workspace_bytes, void* stream)
{
    int64_t need = 0;
    const int status = opsgnn_segment_matmul_workspace_bytes(desc, 0, &need);
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
    const int ran = need > 0 ? segmm::RunRowsSplit(p, workspace, AsStream(stream)) : segmm::RunRowsTensor(p, AsStream(stream));
    return ran == OPSGNN_ERR_UNSUPPORTED ? segmm::RunRowsSimple(p, AsStream(stream)) : ran;
}

extern "C" int opsgnn_segment_matmul_weight_grad(const OpsgnnSegmentMatmulDesc* desc, const void* indptr, const void* src,
                                                 const void* grad, int64_t grad_stride, void* grad_weight, void* workspace,
                                                 int64_t workspace_bytes, void* stream)
{
    int64_t need = 0;
    const int status = opsgnn_segment_matmul_workspace_bytes(desc, 1, &need);
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
    const int ran = p.type == OPSGNN_F32 ? (need > 0 ? segmm::RunOuterSplit(p, workspace, AsStream(stream)) : OPSGNN_ERR_UNSUPPORTED)
                                         : segmm::RunOuterTensor(p, workspace, AsStream(stream));
    return ran == OPSGNN_ERR_UNSUPPORTED ? segmm::RunOuterSimple(p, AsStream(stream)) : ran;
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
