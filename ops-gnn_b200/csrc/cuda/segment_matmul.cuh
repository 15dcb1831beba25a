// Shared declarations of the segment products: launch parameters, and the entry points of their kernels.
#pragma once

#include "common.cuh"
#include "segment_walk.cuh"

namespace opsgnn {
namespace segmm {

// out[r, n] = sum_k a[r, k] * b[e, k, n] for the rows r of segment e; rows of no segment are 0.
struct RowsProblem {
    SegmentPointers ptr;
    const void* a;
    const void* b;
    void* out;
    const float* a_scale;             // 8-bit operands only: [rows, ceil(k / 128)]
    const float* b_scale;             // [segments, ceil(n / 128), ceil(k / 128)]
    int64_t k, n;
    int64_t lda, ldo;                 // row strides, elements
    int64_t b_segment, b_k, b_n;      // strides of b, elements
    int32_t in_type, out_type;
};

// out[e, k, n] = sum over the rows r of segment e of a[r, k] * b[r, n]; 0 for an empty segment.
struct OuterProblem {
    SegmentPointers ptr;
    const void* a;
    const void* b;
    void* out;
    int64_t k, n;
    int64_t lda, ldb;
    int32_t type;
};

// The stride of a dimension as a tensor map takes it: nothing steps over the stride of a single element, so there any run of whole
// 16-byte vectors that holds `extent` values will do.
inline int64_t StrideOf(int64_t stride, int64_t count, int64_t extent, int64_t vec) { return count > 1 ? stride : AlignUp(extent, vec); }

// Any type, size, stride and alignment (segment_matmul_simple.cu).
int RunRowsSimple(const RowsProblem& p, cudaStream_t stream);
int RunOuterSimple(const OuterProblem& p, cudaStream_t stream);
// 16-bit types on the tensor cores (segment_matmul_tc.cu): widths and strides of whole 16-byte vectors, 16-byte aligned
// bases.  OPSGNN_ERR_UNSUPPORTED, with nothing launched, for anything else.
int RunRowsTensor(const RowsProblem& p, void* workspace, cudaStream_t stream);
int RunOuterTensor(const OuterProblem& p, void* workspace, cudaStream_t stream);
// 8-bit and fp32 operands on the tensor cores (segment_matmul_promoted.cu), under the same conditions; fp32 needs a workspace.
int RunRowsFp8(const RowsProblem& p, cudaStream_t stream);
int RunRowsSplit(const RowsProblem& p, void* workspace, cudaStream_t stream);
int RunOuterSplit(const OuterProblem& p, void* workspace, cudaStream_t stream);
int64_t RowsSplitBytes(int64_t rows, int64_t segments, int64_t k, int64_t n);
int64_t OuterSplitBytes(int64_t rows, int64_t segments, int64_t k, int64_t n);
// Both gradients in one call: the terms of the upstream gradient are made once.
int64_t GradsSplitBytes(int64_t rows, int64_t segments, int64_t k, int64_t n);
// `turned`: outer is grad^T src.
int RunGradsSplit(const RowsProblem& rows, const OuterProblem& outer, bool turned, void* workspace, cudaStream_t stream);
// Outer form with few result tiles: rows per piece (0: one piece per segment), fp32 scratch for the pieces, and their sum.
int64_t OuterChunk(int64_t rows, int64_t segments, int64_t k, int64_t n);
int64_t RowsPartialBytes(int64_t rows, int64_t segments, int64_t k, int64_t n);  // the same for the rows form; null: in one piece
int64_t OuterPartialBytes(int64_t rows, int64_t segments, int64_t k, int64_t n);
int JoinPieces(const OuterProblem& p, int64_t chunk, const float* partial, cudaStream_t stream);

}  // namespace segmm
}  // namespace opsgnn
