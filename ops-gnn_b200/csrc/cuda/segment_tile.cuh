// A 64 x 64 tile of a product with fp32 multiply-adds, by 256 threads with 4 x 4 results each: any size, stride and alignment.
#pragma once

#include "common.cuh"

namespace opsgnn {
namespace segmm {
namespace tile {

constexpr int kSize = 64;
constexpr int kDepth = 16;
constexpr int kChunk = 128;  // terms added up at a time
constexpr int kThreads = 256;

struct Operands {  // shared memory
    float a[kDepth][kSize + 4], b[kDepth][kSize + 4];
};

// total[i][j] += sum over d < depth of a(row, d) * b(d, col) for the rows thread / 16 * 4 + i and the columns thread % 16 * 4 + j.
// Sums of more than kChunk terms are added up in chunks, which bounds the growth of the rounding error with the length of the
// sum.  fa(row, d) and fb(d, col) give values and 0 outside; *_depth_fast say which index runs along memory, so that
// neighbouring threads read neighbouring addresses.  sync: a barrier of the 256 threads.
template <class Sync, class FA, class FB>
__device__ __forceinline__ void Multiply(Operands& shared, int thread, Sync&& sync, FA&& fa, FB&& fb, bool a_depth_fast, bool b_depth_fast,
                                         int64_t depth, float (&total)[4][4])
{
    const int tx = thread % 16, ty = thread / 16;
    float part[4][4] = {};
    for (int64_t d0 = 0; d0 < depth; d0 += kDepth) {
#pragma unroll
        for (int i = 0; i < kSize * kDepth / kThreads; ++i) {
            const int at = i * kThreads + thread;
            const int da = a_depth_fast ? at % kDepth : at / kSize, ra = a_depth_fast ? at / kDepth : at % kSize;
            shared.a[da][ra] = d0 + da < depth ? fa(ra, d0 + da) : 0.0f;
            const int db = b_depth_fast ? at % kDepth : at / kSize, cb = b_depth_fast ? at / kDepth : at % kSize;
            shared.b[db][cb] = d0 + db < depth ? fb(d0 + db, cb) : 0.0f;
        }
        sync();
#pragma unroll
        for (int d = 0; d < kDepth; ++d) {
            const float4 x = *reinterpret_cast<const float4*>(&shared.a[d][ty * 4]);
            const float4 y = *reinterpret_cast<const float4*>(&shared.b[d][tx * 4]);
            const float xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    part[i][j] = fmaf(xs[i], ys[j], part[i][j]);
                }
            }
        }
        sync();
        if ((d0 + kDepth) % kChunk == 0 || d0 + kDepth >= depth) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    total[i][j] += part[i][j];
                    part[i][j] = 0.0f;
                }
            }
        }
    }
}

}  // namespace tile
}  // namespace segmm
}  // namespace opsgnn
