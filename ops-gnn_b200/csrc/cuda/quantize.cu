// Block-scaled 8-bit values: float8_e4m3 with one fp32 scale for 128 consecutive columns of a row, or for a tile of
// 128 x 128.  The scale is the smallest power of two that brings the block's largest finite magnitude to at most 448 (the
// largest e4m3 value), 1 for a block without a non-zero finite value.  A power of two makes value / scale exact, so every
// value is rounded once (to nearest, ties to even) and no result hangs on how a division rounds.  Infinities saturate at
// 448, NaN stays NaN; neither has a part in the scale.
#include <cuda_fp8.h>

#include <algorithm>

#include "common.cuh"

namespace opsgnn {
namespace quant {

constexpr int kBlock = 128;
constexpr unsigned kFull = 0xffffffffu;

// 2^p and 2^-p with p the smallest exponent for which top <= 448 * 2^p, 448 = 1.75 * 2^8.  With top = m * 2^e, 1 <= m < 2:
// p = e - 8, one more where m > 1.75.  p >= -126 keeps the scale a normal number; top is finite, so p <= 120.
__device__ __forceinline__ void ScaleOf(float top, float& scale, float& inverse)
{
    const uint32_t bits = __float_as_uint(top);
    int p = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    p = top > 0.0f ? max(p, -126) : 0;
    scale = __uint_as_float(static_cast<uint32_t>(p + 127) << 23);
    inverse = __uint_as_float(static_cast<uint32_t>(127 - p) << 23);
}

__device__ __forceinline__ float FiniteAbs(float v)
{
    const float a = fabsf(v);
    return a < INFINITY ? a : 0.0f;  // NaN compares false
}

__device__ __forceinline__ uint16_t Two(float a, float b)
{
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

template <class T, int VEC> __device__ __forceinline__ void StoreBytes(uint8_t* out, const float (&v)[VEC], float inverse)
{
    if constexpr (VEC == 1) {
        *out = static_cast<uint8_t>(Two(v[0] * inverse, 0.0f) & 0xff);
    } else {
        uint32_t words[VEC / 4];
#pragma unroll
        for (int i = 0; i < VEC / 4; ++i) {
            words[i] = Two(v[4 * i] * inverse, v[4 * i + 1] * inverse) |
                       (static_cast<uint32_t>(Two(v[4 * i + 2] * inverse, v[4 * i + 3] * inverse)) << 16);
        }
        if constexpr (VEC == 8) {
            *reinterpret_cast<uint2*>(out) = make_uint2(words[0], words[1]);
        } else {
            *reinterpret_cast<uint32_t*>(out) = words[0];
        }
    }
}

// One scale per row and 128 columns.  Lanes x VEC = 128: a block is one 16-byte (VEC = 16 / sizeof(T)) vector per lane of a
// half warp (16-bit types) or a warp (fp32); the scalar form takes any width and alignment.
template <class T, int VEC>
__global__ void __launch_bounds__(256) RowKernel(const T* __restrict__ src, int64_t rows, int64_t width, uint8_t* __restrict__ values,
                                                 float* __restrict__ scales)
{
    constexpr int PER = VEC == 1 ? 4 : 1;             // strided elements a lane takes in the scalar form
    constexpr int LANES = VEC == 1 ? 32 : kBlock / VEC;
    constexpr int GROUPS = 256 / LANES;
    const int lane = threadIdx.x % LANES;
    const int64_t across = (width + kBlock - 1) / kBlock;
    const int64_t blocks = rows * across;
    // All lanes of a warp stay in the loop together: the shuffles below name the whole warp.
    const int64_t steps = (blocks + static_cast<int64_t>(gridDim.x) * GROUPS - 1) / (static_cast<int64_t>(gridDim.x) * GROUPS);
    for (int64_t s = 0; s < steps; ++s) {
        const int64_t b = (s * gridDim.x + blockIdx.x) * GROUPS + threadIdx.x / LANES;
        const bool real = b < blocks;
        const int64_t row = real ? b / across : 0, block = real ? b % across : 0;
        const int64_t first = row * width + block * kBlock;
        const int left = static_cast<int>(width - block * kBlock < kBlock ? width - block * kBlock : kBlock);
        float v[VEC * PER];
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < VEC * PER; ++i) {
            v[i] = 0.0f;
        }
        if constexpr (VEC == 1) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (real && i * LANES + lane < left) {
                    v[i] = Widen<float, T>(LoadNc(src + first + i * LANES + lane));
                }
            }
        } else {
            if (real && lane * VEC < left) {
                Unpack<float, T, VEC>(LoadGather<T, VEC>(src + first + lane * VEC), v);
            }
        }
#pragma unroll
        for (int i = 0; i < VEC * PER; ++i) {
            top = fmaxf(top, FiniteAbs(v[i]));
        }
#pragma unroll
        for (int d = LANES / 2; d > 0; d >>= 1) {
            top = fmaxf(top, __shfl_xor_sync(kFull, top, d));
        }
        float scale, inverse;
        ScaleOf(top, scale, inverse);
        if (real && lane == 0) {
            scales[b] = scale;
        }
        if constexpr (VEC == 1) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (real && i * LANES + lane < left) {
                    const float one[1] = {v[i]};
                    StoreBytes<T, 1>(values + first + i * LANES + lane, one, inverse);
                }
            }
        } else {
            if (real && lane * VEC < left) {
                StoreBytes<T, VEC>(values + first + lane * VEC, v, inverse);
            }
        }
    }
}

// One scale per tile of 128 x 128: a thread block per tile, the tile's values stay in registers between the maximum and the
// conversion.
template <class T, int VEC>
__global__ void __launch_bounds__(512) TileKernel(const T* __restrict__ src, int64_t rows, int64_t width, int64_t down, int64_t across,
                                                  uint8_t* __restrict__ values, float* __restrict__ scales)
{
    constexpr int LANES = kBlock / VEC;       // threads along a row of the tile
    constexpr int STEP = 512 / LANES;         // rows taken at once
    constexpr int PER = kBlock / STEP;
    __shared__ float tops[16];
    const int lane = threadIdx.x % LANES, line = threadIdx.x / LANES;
    const int64_t tile = blockIdx.x;
    const int64_t batch = tile / (down * across), row0 = tile / across % down * kBlock, col0 = tile % across * kBlock;
    const int64_t at = (batch * rows + row0) * width + col0;
    const int high = static_cast<int>(rows - row0 < kBlock ? rows - row0 : kBlock);
    const int left = static_cast<int>(width - col0 < kBlock ? width - col0 : kBlock);
    float v[PER][VEC];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int r = i * STEP + line;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            v[i][j] = 0.0f;
        }
        if (r < high && lane * VEC < left) {
            const T* from = src + at + r * width + lane * VEC;
            if constexpr (VEC == 1) {
                v[i][0] = Widen<float, T>(LoadNc(from));
            } else {
                Unpack<float, T, VEC>(LoadGather<T, VEC>(from), v[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            top = fmaxf(top, FiniteAbs(v[i][j]));
        }
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(kFull, top, d));
    }
    if ((threadIdx.x & 31) == 0) {
        tops[threadIdx.x >> 5] = top;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        top = fmaxf(top, tops[w]);
    }
    float scale, inverse;
    ScaleOf(top, scale, inverse);
    if (threadIdx.x == 0) {
        scales[tile] = scale;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int r = i * STEP + line;
        if (r < high && lane * VEC < left) {
            StoreBytes<T, VEC>(values + at + r * width + lane * VEC, v[i], inverse);
        }
    }
}

template <class T>
int Run(const void* src, int64_t batch, int64_t rows, int64_t width, int block_rows, uint8_t* values, float* scales, cudaStream_t stream)
{
    constexpr int VEC = 16 / sizeof(T);
    const T* in = static_cast<const T*>(src);
    const bool wide = width % VEC == 0 && Aligned(src, 16) && Aligned(values, VEC);
    const int64_t across = CeilDiv(width, kBlock);
    if (block_rows == 1) {
        const int64_t blocks = batch * rows * across;
        const int64_t groups = wide ? 256 / (kBlock / VEC) : 8;
        const int grid = static_cast<int>(std::min<int64_t>(CeilDiv(blocks, groups), static_cast<int64_t>(SmCount()) * 64));
        if (wide) {
            RowKernel<T, VEC><<<grid, 256, 0, stream>>>(in, batch * rows, width, values, scales);
        } else {
            RowKernel<T, 1><<<grid, 256, 0, stream>>>(in, batch * rows, width, values, scales);
        }
    } else {
        const int64_t down = CeilDiv(rows, kBlock), tiles = batch * down * across;
        if (tiles > INT32_MAX) {
            return OPSGNN_ERR_LIMIT;
        }
        if (wide) {
            TileKernel<T, VEC><<<static_cast<unsigned>(tiles), 512, 0, stream>>>(in, rows, width, down, across, values, scales);
        } else {
            TileKernel<T, 1><<<static_cast<unsigned>(tiles), 512, 0, stream>>>(in, rows, width, down, across, values, scales);
        }
    }
    return LaunchStatus();
}

}  // namespace quant
}  // namespace opsgnn

using namespace opsgnn;

extern "C" int opsgnn_quantize_fp8(const void* src, int dtype, int64_t batch, int64_t rows, int64_t width, int block_rows, void* values,
                                   float* scales, void* stream)
{
    if (batch < 0 || rows < 0 || width < 0 || (block_rows != 1 && block_rows != quant::kBlock)) {
        return OPSGNN_ERR_INVALID;
    }
    if (batch == 0 || rows == 0 || width == 0) {
        return OPSGNN_OK;
    }
    if (src == nullptr || values == nullptr || scales == nullptr) {
        return OPSGNN_ERR_INVALID;
    }
    uint8_t* out = static_cast<uint8_t*>(values);
    switch (dtype) {
        case OPSGNN_F32:
            return quant::Run<float>(src, batch, rows, width, block_rows, out, scales, AsStream(stream));
        case OPSGNN_F16:
            return quant::Run<__half>(src, batch, rows, width, block_rows, out, scales, AsStream(stream));
        case OPSGNN_BF16:
            return quant::Run<__nv_bfloat16>(src, batch, rows, width, block_rows, out, scales, AsStream(stream));
        default:
            return OPSGNN_ERR_UNSUPPORTED;
    }
}
