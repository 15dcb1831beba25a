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

// 16 bytes that are read once.
template <class T, int VEC> __device__ __forceinline__ Pack<T, VEC> LoadStream16(const T* p)
{
    static_assert(sizeof(T) * VEC == 16, "one vector");
    const uint4 raw = __ldcs(reinterpret_cast<const uint4*>(p));
    Pack<T, VEC> out;
    memcpy(&out, &raw, 16);
    return out;
}

// Largest magnitude of a 16-byte vector; NaN has no part.  An infinity shows as +inf.
template <class T, int VEC> __device__ __forceinline__ float TopOf(const Pack<T, VEC>& p)
{
    if constexpr (std::is_same<T, float>::value) {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            top = fmaxf(top, fabsf(p.v[i]));
        }
        return top;
    } else {
        using Two = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        Two pair[VEC / 2];
        memcpy(pair, &p, sizeof(pair));
        Two top = __habs2(pair[0]);
#pragma unroll
        for (int i = 1; i < VEC / 2; ++i) {
            top = __hmax2(top, __habs2(pair[i]));  // of a number and a NaN, the number
        }
        return fmaxf(fmaxf(Widen<float, T>(top.x), Widen<float, T>(top.y)), 0.0f);
    }
}
template <class T, int VEC> __device__ __forceinline__ float FiniteTopOf(const Pack<T, VEC>& p)
{
    float v[VEC], top = 0.0f;
    Unpack<float, T, VEC>(p, v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        top = fmaxf(top, FiniteAbs(v[i]));
    }
    return top;
}
template <int LANES> __device__ __forceinline__ float GroupMax(float top)
{
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(kFull, top, d));
    }
    return top;
}

// One scale per row and 128 columns, whole vectors: a block of 128 is one 16-byte vector per lane of a half warp (16-bit
// types) or a warp (fp32).  Bound by memory: every lane has kAhead vectors in flight (16381 x 4096 bf16: two 33.3 us,
// four 36.1, eight 37.8).  FULL: the width is a multiple of 128, so the blocks lie one after the other.
constexpr int kAhead = 2;

template <class T, bool FULL>
__global__ void __launch_bounds__(256) RowKernel(const T* __restrict__ src, int64_t blocks, int64_t width, int64_t across,
                                                 uint8_t* __restrict__ values, float* __restrict__ scales)
{
    constexpr int VEC = 16 / sizeof(T);
    constexpr int LANES = kBlock / VEC;
    constexpr int GROUPS = 256 / LANES;
    const int lane = threadIdx.x % LANES;
    // kAhead runs of GROUPS blocks, one after the other in memory; every lane of a warp stays in the loop, as the shuffles name
    // the whole warp.
    for (int64_t first = static_cast<int64_t>(blockIdx.x) * (GROUPS * kAhead); first < blocks;
         first += static_cast<int64_t>(gridDim.x) * (GROUPS * kAhead)) {
        const int64_t b0 = first + threadIdx.x / LANES;
        Pack<T, VEC> p[kAhead];
        int64_t at[FULL ? 1 : kAhead];
        unsigned mine = 0;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t b = b0 + i * GROUPS;
            bool here = b < blocks;
            const T* from;
            if constexpr (FULL) {
                from = src + b * kBlock + lane * VEC;
            } else {
                const int64_t row = here ? b / across : 0, column = (b - row * across) * kBlock + lane * VEC;
                at[i] = row * width + column;
                from = src + at[i];
                here = here && column < width;
            }
            mine |= here ? 1u << i : 0u;
            memset(&p[i], 0, sizeof(p[i]));
            if (here) {
                p[i] = LoadStream16<T, VEC>(from);
            }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t b = b0 + i * GROUPS;
            float top = GroupMax<LANES>(TopOf<T, VEC>(p[i]));
            if (__any_sync(kFull, top == INFINITY)) {
                top = GroupMax<LANES>(FiniteTopOf<T, VEC>(p[i]));
            }
            float scale, inverse;
            ScaleOf(top, scale, inverse);
            if (lane == 0 && b < blocks) {
                scales[b] = scale;
            }
            if ((mine >> i) & 1u) {
                float v[VEC];
                Unpack<float, T, VEC>(p[i], v);
                StoreBytes<T, VEC>(values + (FULL ? b * kBlock + lane * VEC : at[FULL ? 0 : i]), v, inverse);
            }
        }
    }
}

// The same for any width and alignment, a block of 128 per warp: single loads and one-byte stores, 2.3 times as long (16381 x 4095
// bf16 85 us, fp32 83 us, against 37 us for 16381 x 4096 bf16).
template <class T>
__global__ void __launch_bounds__(256) RowScalarKernel(const T* __restrict__ src, int64_t blocks, int64_t width, int64_t across,
                                                       uint8_t* __restrict__ values, float* __restrict__ scales)
{
    constexpr int PER = kBlock / 32;
    const int lane = threadIdx.x & 31;
    for (int64_t b = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); b < blocks; b += static_cast<int64_t>(gridDim.x) * 8) {
        const int64_t row = b / across, column = (b - row * across) * kBlock;
        const int64_t first = row * width + column;
        const int left = static_cast<int>(width - column < kBlock ? width - column : kBlock);
        float v[PER], top = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            v[i] = i * 32 + lane < left ? Widen<float, T>(LoadNc(src + first + i * 32 + lane)) : 0.0f;
            top = fmaxf(top, FiniteAbs(v[i]));
        }
        top = GroupMax<32>(top);
        float scale, inverse;
        ScaleOf(top, scale, inverse);
        if (lane == 0) {
            scales[b] = scale;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (i * 32 + lane < left) {
                const float one[1] = {v[i]};
                StoreBytes<T, 1>(values + first + i * 32 + lane, one, inverse);
            }
        }
    }
}

// One scale per tile of 128 x 128: a thread block per tile, the tile stays in registers (as loaded) between the maximum and
// the conversion.  VEC 1: any width and alignment (64 x 1024 x 2047 bf16 197 us, x 2048 in vectors 70 us).
constexpr int kTileThreads = 256;

template <class T, int VEC>
__global__ void __launch_bounds__(kTileThreads) TileKernel(const T* __restrict__ src, int64_t rows, int64_t width, int down, int across,
                                                           uint8_t* __restrict__ values, float* __restrict__ scales)
{
    constexpr int LANES = kBlock / VEC;         // threads along a row of the tile
    constexpr int STEP = kTileThreads / LANES;  // rows taken at once
    constexpr int PER = kBlock / STEP;
    __shared__ float tops[2][kTileThreads / 32];
    const int lane = threadIdx.x % LANES, line = threadIdx.x / LANES;
    const unsigned tile = blockIdx.x;
    const unsigned band = tile / across;
    const int64_t batch = band / down, row0 = static_cast<int64_t>(band % down) * kBlock, col0 = static_cast<int64_t>(tile % across) * kBlock;
    const int64_t at = (batch * rows + row0) * width + col0 + lane * VEC;
    const int high = static_cast<int>(rows - row0 < kBlock ? rows - row0 : kBlock);
    const bool inside = lane * VEC < width - col0;
    Pack<T, VEC> p[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int r = i * STEP + line;
        memset(&p[i], 0, sizeof(p[i]));
        if (r < high && inside) {
            if constexpr (VEC == 1) {
                p[i].v[0] = LoadNc(src + at + r * width);
            } else {
                p[i] = LoadStream16<T, VEC>(src + at + r * width);
            }
        }
    }
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if constexpr (VEC == 1) {
            top = fmaxf(top, fabsf(Widen<float, T>(p[i].v[0])));
        } else {
            top = fmaxf(top, TopOf<T, VEC>(p[i]));
        }
    }
    auto over_block = [&](float mine, float* shared) {
        mine = GroupMax<32>(mine);
        if ((threadIdx.x & 31) == 0) {
            shared[threadIdx.x >> 5] = mine;
        }
        __syncthreads();
        float all = 0.0f;
#pragma unroll
        for (int w = 0; w < kTileThreads / 32; ++w) {
            all = fmaxf(all, shared[w]);
        }
        return all;
    };
    top = over_block(top, tops[0]);
    if (top == INFINITY) {  // the same in every thread
        top = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            top = fmaxf(top, FiniteTopOf<T, VEC>(p[i]));
        }
        top = over_block(top, tops[1]);
    }
    float scale, inverse;
    ScaleOf(top, scale, inverse);
    if (threadIdx.x == 0) {
        scales[tile] = scale;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int r = i * STEP + line;
        if (r < high && inside) {
            float v[VEC];
            Unpack<float, T, VEC>(p[i], v);
            StoreBytes<T, VEC>(values + at + r * width, v, inverse);
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
        const int64_t groups = wide ? 256 / (kBlock / VEC) * kAhead : 8;
        const int grid = static_cast<int>(std::min<int64_t>(CeilDiv(blocks, groups), static_cast<int64_t>(SmCount()) * 64));
        if (!wide) {
            RowScalarKernel<T><<<grid, 256, 0, stream>>>(in, blocks, width, across, values, scales);
        } else if (width % kBlock == 0) {
            RowKernel<T, true><<<grid, 256, 0, stream>>>(in, blocks, width, across, values, scales);
        } else {
            RowKernel<T, false><<<grid, 256, 0, stream>>>(in, blocks, width, across, values, scales);
        }
    } else {
        const int64_t down = CeilDiv(rows, kBlock), tiles = batch * down * across;
        if (tiles > INT32_MAX) {
            return OPSGNN_ERR_LIMIT;
        }
        const unsigned grid = static_cast<unsigned>(tiles);
        if (wide) {
            TileKernel<T, VEC><<<grid, kTileThreads, 0, stream>>>(in, rows, width, static_cast<int>(down), static_cast<int>(across), values, scales);
        } else {
            TileKernel<T, 1><<<grid, kTileThreads, 0, stream>>>(in, rows, width, static_cast<int>(down), static_cast<int>(across), values, scales);
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
