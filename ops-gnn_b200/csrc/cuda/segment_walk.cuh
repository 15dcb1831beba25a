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
    template <class I> __device__ __forceinline__ void Range(I e, I& begin, I& end) const
    {
        if (data == nullptr) {  // one dense segment
            begin = 0;
            end = static_cast<I>(rows);
            return;
        }
        begin = static_cast<I>(Raw(e));
        const I last = static_cast<I>(Raw(static_cast<int64_t>(e) + 1));
        end = last > begin ? last : begin;
    }
};

// Row tiles of all segments in order, TILE rows each (a segment's last one may be short; an empty segment has none).
// Seek(t) is called by a whole warp with ascending t and finds tile t by a warp scan over 32 segments at a time, from where it
// last stood: no tile table, no workspace, no limit on the number of segments.  Three registers live between two calls (the
// scan is done again each time: the products' summing warps have none to spare).  TILE 0: the number of rows is given to
// Start.  I: the type of rows and tile numbers, int where the host has checked that they fit.
template <int TILE, class I> struct SegmentWalk {
    I from, base;          // first segment of the 32 at hand; tiles before them
    I high;                // largest pointer before them
    I length;              // rows per tile
    // what Seek found
    I segment, row, row_end, begin_row;  // begin_row: the segment's first

    __device__ __forceinline__ I Rows() const { return TILE > 0 ? TILE : length; }
    __device__ __forceinline__ void Start(const SegmentPointers& p, I tile = TILE)
    {
        length = tile;
        from = 0;
        base = 0;
        high = p.data != nullptr ? static_cast<I>(p.Raw(0)) : 0;
    }
    // This lane's segment of the 32 at hand, and the tiles of the 32 up to and with it.
    __device__ __forceinline__ void Scan(const SegmentPointers& p, I& begin, I& end, I& inclusive) const
    {
        const int lane = threadIdx.x & 31;
        end = 0;
        if (from + lane < static_cast<I>(p.segments)) {
            end = p.data != nullptr ? static_cast<I>(p.Raw(static_cast<int64_t>(from) + lane + 1)) : static_cast<I>(p.rows);
        }
        // A pointer below an earlier one counts as that one: segments never overlap, and all tiles together are bounded.
        end = end > high ? end : high;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const I up = __shfl_up_sync(0xffffffffu, end, d);
            end = lane >= d && up > end ? up : end;
        }
        begin = __shfl_up_sync(0xffffffffu, end, 1);
        begin = lane == 0 ? high : begin;
        inclusive = (end - begin + Rows() - 1) / Rows();
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const I up = __shfl_up_sync(0xffffffffu, inclusive, d);
            inclusive += lane >= d ? up : 0;
        }
    }
    __device__ __forceinline__ void Next(I end, I inclusive)
    {
        base += __shfl_sync(0xffffffffu, inclusive, 31);
        high = __shfl_sync(0xffffffffu, end, 31);
        from += 32;
    }
    // False past the last tile.
    __device__ __forceinline__ bool Seek(const SegmentPointers& p, I t)
    {
        while (from < static_cast<I>(p.segments)) {
            I begin, end, inclusive;
            Scan(p, begin, end, inclusive);
            const unsigned there = __ballot_sync(0xffffffffu, t < base + inclusive);
            if (there != 0) {
                const int owner = __ffs(there) - 1;
                const I before = __shfl_sync(0xffffffffu, base + inclusive - (end - begin + Rows() - 1) / Rows(), owner);
                row_end = __shfl_sync(0xffffffffu, end, owner);
                begin_row = __shfl_sync(0xffffffffu, begin, owner);
                row = begin_row + (t - before) * Rows();
                segment = from + owner;
                return true;
            }
            Next(end, inclusive);
        }
        return false;
    }
};

// Sums over a segment's rows, the rows of long segments cut into pieces of `chunk`.  A segment of one piece is written as the
// result; the pieces of longer ones go to slots of a workspace, which the row they start at names: the last piece of a segment
// and the first of the next may start among the same chunk of rows, hence two slots for each.
__device__ __forceinline__ int PieceSlot(int row, bool last, int chunk) { return row / chunk * 2 + (last ? 1 : 0); }
inline int64_t PieceSlots(int64_t rows, int64_t chunk) { return CeilDiv(rows, chunk) * 2; }

// Where a piece that a walk has found goes: twice its slot, or twice its segment and one.
template <class Walk> __device__ __forceinline__ int PieceTarget(const Walk& walk, int chunk)
{
    const bool last = walk.row_end - walk.row <= chunk;
    return last && walk.row == walk.begin_row ? walk.segment * 2 + 1 : PieceSlot(walk.row, last, chunk) * 2;
}

}  // namespace opsgnn
