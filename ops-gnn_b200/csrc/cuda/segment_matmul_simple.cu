// Segment products for every type, size, stride and alignment: tiles of 64 x 64 in shared memory (segment_tile.cuh).
#include <cuda_fp8.h>

#include <algorithm>

#include "segment_matmul.cuh"
#include "segment_tile.cuh"

namespace opsgnn {
namespace segmm {
namespace {

constexpr int kTile = tile::kSize;
constexpr int kThreads = tile::kThreads;

template <class T> __device__ __forceinline__ float ValueOf(const T* p) { return Widen<float, T>(LoadNc(p)); }
template <> __device__ __forceinline__ float ValueOf<__nv_fp8_e4m3>(const __nv_fp8_e4m3* p)
{
    return static_cast<float>(*p);
}

struct BlockSync {
    __device__ __forceinline__ void operator()() const { __syncthreads(); }
};

template <class T, class O> __global__ void __launch_bounds__(kThreads) RowsKernel(RowsProblem p)
{
    __shared__ tile::Operands shared;
    const T* a = static_cast<const T*>(p.a);
    const T* b = static_cast<const T*>(p.b);
    O* out = static_cast<O*>(p.out);
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int64_t across = (p.n + kTile - 1) / kTile;
    SegmentWalk<kTile, int64_t> walk;
    walk.Start(p.ptr);
    for (int64_t t = blockIdx.x;; t += gridDim.x) {
        if (!walk.Seek(p.ptr, t / across)) {
            break;
        }
        const int64_t col0 = t % across * kTile;
        float total[4][4] = {};
        const T* matrix = b + walk.segment * p.b_segment;
        const int64_t row = walk.row, row_end = walk.row_end;
        const int64_t blocks = (p.k + 127) / 128;
        const float* bs = p.b_scale != nullptr
                              ? p.b_scale + (walk.segment * ((p.n + 127) / 128) + col0 / 128) * blocks
                              : nullptr;
        auto multiply = [&](int64_t from, int64_t depth, float (&sum)[4][4]) {
            tile::Multiply(
                shared, threadIdx.x, BlockSync(),
                [&](int r, int64_t d) { return row + r < row_end ? ValueOf(a + (row + r) * p.lda + from + d) : 0.0f; },
                [&](int64_t d, int c) { return col0 + c < p.n ? ValueOf(matrix + (from + d) * p.b_k + (col0 + c) * p.b_n) : 0.0f; }, true,
                p.b_k == 1, depth, sum);
        };
        if (bs == nullptr) {
            multiply(0, p.k, total);
        } else {
            // sum over blocks of 128: (scale of the row) * (scale of the tile of b) * (product of the 8-bit values)
            for (int64_t block = 0; block < blocks; ++block) {
                float sum[4][4] = {};
                multiply(block * 128, p.k - block * 128 < 128 ? p.k - block * 128 : 128, sum);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int64_t r = row + ty * 4 + i;
                    const float scale = r < row_end ? __ldg(p.a_scale + r * blocks + block) * __ldg(bs + block) : 0.0f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        total[i][j] = fmaf(scale, sum[i][j], total[i][j]);
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t r = row + ty * 4 + i;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t c = col0 + tx * 4 + j;
                if (r < row_end && c < p.n) {
                    out[r * p.ldo + c] = Narrow<O, float>(total[i][j]);
                }
            }
        }
    }
    // Rows of no segment.
    const int64_t first = p.ptr.data != nullptr ? p.ptr.Raw(0) : 0;
    const int64_t last = p.ptr.data != nullptr ? p.ptr.Raw(p.ptr.segments) : p.ptr.rows;
    for (int64_t r = blockIdx.x; r < first + (p.ptr.rows - last); r += gridDim.x) {
        const int64_t at = r < first ? r : last + (r - first);
        for (int64_t c = threadIdx.x; c < p.n; c += kThreads) {
            out[at * p.ldo + c] = Narrow<O, float>(0.0f);
        }
    }
}

template <class T> __global__ void __launch_bounds__(kThreads) OuterKernel(OuterProblem p)
{
    __shared__ tile::Operands shared;
    const T* a = static_cast<const T*>(p.a);
    const T* b = static_cast<const T*>(p.b);
    T* out = static_cast<T*>(p.out);
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int64_t down = (p.k + kTile - 1) / kTile, across = (p.n + kTile - 1) / kTile;
    for (int64_t t = blockIdx.x; t < p.ptr.segments * down * across; t += gridDim.x) {
        const int64_t e = t / (down * across), k0 = t / across % down * kTile, n0 = t % across * kTile;
        int64_t begin, end;
        p.ptr.Range<int64_t>(e, begin, end);
        float total[4][4] = {};
        tile::Multiply(
            shared, threadIdx.x, BlockSync(), [&](int r, int64_t d) { return k0 + r < p.k ? ValueOf(a + (begin + d) * p.lda + k0 + r) : 0.0f; },
            [&](int64_t d, int c) { return n0 + c < p.n ? ValueOf(b + (begin + d) * p.ldb + n0 + c) : 0.0f; }, false, false, end - begin,
            total);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t k = k0 + ty * 4 + i, n = n0 + tx * 4 + j;
                if (k < p.k && n < p.n) {
                    out[(e * p.k + k) * p.n + n] = Narrow<T, float>(total[i][j]);
                }
            }
        }
    }
}

template <class T, class O> int LaunchRows(const RowsProblem& p, cudaStream_t stream)
{
    // At most this many tiles; the kernel finds out on the device how many there are.
    const int64_t bound = (p.ptr.rows / kTile + p.ptr.segments) * CeilDiv(p.n, kTile);
    const int grid = static_cast<int>(std::min<int64_t>(std::max<int64_t>(bound, 1), static_cast<int64_t>(SmCount()) * 8));
    RowsKernel<T, O><<<grid, kThreads, 0, stream>>>(p);
    return LaunchStatus();
}

}  // namespace

int RunRowsSimple(const RowsProblem& p, cudaStream_t stream)
{
    if (p.in_type == OPSGNN_F8E4M3) {
        switch (p.out_type) {
            case OPSGNN_F32:
                return LaunchRows<__nv_fp8_e4m3, float>(p, stream);
            case OPSGNN_F16:
                return LaunchRows<__nv_fp8_e4m3, __half>(p, stream);
            default:
                return LaunchRows<__nv_fp8_e4m3, __nv_bfloat16>(p, stream);
        }
    }
    switch (p.in_type) {
        case OPSGNN_F32:
            return LaunchRows<float, float>(p, stream);
        case OPSGNN_F16:
            return LaunchRows<__half, __half>(p, stream);
        default:
            return LaunchRows<__nv_bfloat16, __nv_bfloat16>(p, stream);
    }
}

int RunOuterSimple(const OuterProblem& p, cudaStream_t stream)
{
    const int64_t tiles = p.ptr.segments * CeilDiv(p.k, kTile) * CeilDiv(p.n, kTile);
    const int grid = static_cast<int>(std::min<int64_t>(std::max<int64_t>(tiles, 1), static_cast<int64_t>(SmCount()) * 8));
    switch (p.type) {
        case OPSGNN_F32:
            OuterKernel<float><<<grid, kThreads, 0, stream>>>(p);
            break;
        case OPSGNN_F16:
            OuterKernel<__half><<<grid, kThreads, 0, stream>>>(p);
            break;
        default:
            OuterKernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(p);
            break;
    }
    return LaunchStatus();
}

}  // namespace segmm
}  // namespace opsgnn
