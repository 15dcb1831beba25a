// How the segment products find their work without asking the host: row tiles of a pointer array, numbered on the device.
#pragma once

#include "common.cuh"

namespace opsgnn {

// Pointers as the kernels use them: clamped to the rows there are, an end never before its start, so no pointer content can
// lead an access out of bounds.
struct SegmentPointers {
    const void* data;
    int64_t segments, rows;
    int32_t wide;  // 1: int64, 0: int32

    __device__ __forceinline__ int64_t Raw(int64_t i) const
    {
        const int64_t v = wide ? __ldg(static_cast<const long long*>(data) + i) : __ldg(static_cast<const int*>(data) + i);
        return v < 0 ? 0 : (v > rows ? rows : v);
    }
    __device__ __forceinline__ void Range(int64_t e, int64_t& begin, int64_t& end) const
    {
        if (data == nullptr) {  // one dense segment
            begin = 0;
            end = rows;
            return;
        }
        begin = Raw(e);
        const int64_t last = Raw(e + 1);
        end = last > begin ? last : begin;
    }
};

// Row tiles of all segments in order, TILE rows each (a segment's last one may be short; an empty segment has none).
// Seek(t) is called by a whole warp with ascending t and finds tile t by a running warp scan over 32 segments at a time:
// no tile table, no workspace, no limit on the number of segments.  TILE 0: the number of rows is given to Start.
template <int TILE> struct SegmentWalk {
    SegmentPointers ptr;
    int64_t length;              // rows per tile
    int64_t from, base;          // first segment of the 32 at hand; tiles before them
    int64_t begin, end;          // this lane's segment
    int64_t inclusive;           // tiles of the 32 up to and with this lane's segment
    // what Seek found
    int64_t segment, row, row_end;

    __device__ __forceinline__ int64_t Tiles() const
    {
        const int64_t tile = TILE > 0 ? TILE : length;
        return (end - begin + tile - 1) / tile;
    }
    __device__ __forceinline__ void Load()
    {
        const int lane = threadIdx.x & 31;
        begin = end = 0;
        if (from + lane < ptr.segments) {
            ptr.Range(from + lane, begin, end);
        }
        inclusive = Tiles();
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t up = __shfl_up_sync(0xffffffffu, inclusive, d);
            inclusive += lane >= d ? up : 0;
        }
    }
    __device__ __forceinline__ void Start(const SegmentPointers& p, int64_t tile = TILE)
    {
        ptr = p;
        length = tile;
        from = 0;
        base = 0;
        Load();
    }
    // False past the last tile.
    __device__ __forceinline__ bool Seek(int64_t t)
    {
        while (true) {
            const unsigned there = __ballot_sync(0xffffffffu, t < base + inclusive);
            if (there != 0) {
                const int owner = __ffs(there) - 1;
                const int64_t first = __shfl_sync(0xffffffffu, base + inclusive - Tiles(), owner);
                row_end = __shfl_sync(0xffffffffu, end, owner);
                row = __shfl_sync(0xffffffffu, begin, owner) + (t - first) * (TILE > 0 ? TILE : length);
                segment = from + owner;
                return true;
            }
            base += __shfl_sync(0xffffffffu, inclusive, 31);
            from += 32;
            if (from >= ptr.segments) {
                return false;
            }
            Load();
        }
    }
};

}  // namespace opsgnn
