// Segment products of 16-bit types on the tensor cores (tcgen05.mma, operands by TMA, accumulators in TMEM).
//
// One persistent thread block per SM walks over output tiles of 128 x BN:
//   warp 0      loads the tiles' operands, 64 values of the reduced index at a time, into a ring of shared-memory stages
//   warp 1      issues the matrix instructions; accumulators alternate between two halves of TMEM
//   warps 4-7   move a finished accumulator to memory (32 rows each) while the next tile is multiplied
// Rows form (out and grad_src): tiles are row tiles of one segment times BN columns, found on the device (SegmentWalk).  A
// tile's last rows may belong to the next segment: they are multiplied and not stored, rows do not mix.  The weight is read as
// it lies: its reduced index along memory (K-major operand) or its columns (MN-major).
// Outer form (grad_weight): the rows of a segment are the reduced index, both operands MN-major.  The last load of a segment
// reaches into the next one; those rows are zeroed in shared memory, in both operands (0 * NaN is NaN).
#include <algorithm>

#include "segment_matmul.cuh"
#include "tensor_core.cuh"

namespace opsgnn {

namespace tc {

bool EncodeMap(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base, const uint64_t* sizes, const uint64_t* strides,
               const uint32_t* box)
{
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = []() -> Encode {
        void* entry = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &entry, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess) {
            (void)cudaGetLastError();
            return nullptr;
        }
        return reinterpret_cast<Encode>(entry);
    }();
    if (encode == nullptr) {
        return false;
    }
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    return encode(map, type, static_cast<cuuint32_t>(rank), const_cast<void*>(base), reinterpret_cast<const cuuint64_t*>(sizes),
                  reinterpret_cast<const cuuint64_t*>(strides), box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool EncodeSlabs(CUtensorMap* map, CUtensorMapDataType type, const void* base, int64_t extent, int64_t rows, int64_t depth,
                 int64_t row_bytes, int64_t depth_bytes, int slabs)
{
    const bool whole = WholeSlabs(extent);
    const uint64_t sizes[4] = {static_cast<uint64_t>(whole ? 64 : extent), static_cast<uint64_t>(rows),
                               static_cast<uint64_t>(whole ? extent / 64 : 1), static_cast<uint64_t>(depth)};
    const uint64_t strides[3] = {static_cast<uint64_t>(row_bytes), 128, static_cast<uint64_t>(depth_bytes)};
    const uint32_t box[4] = {64, 64, whole ? static_cast<uint32_t>(slabs) : 1u, 1};
    return EncodeMap(map, type, 4, base, sizes, strides, box);
}

}  // namespace tc

namespace segmm {
namespace {

constexpr int kRows = 128;     // rows of a tile
constexpr int kBoxRows = 32;   // rows of a per load where a tile is not full
constexpr int kDepth = 64;     // reduced index per stage: one 128-byte row of 16-bit values
constexpr int kThreads = 256;
constexpr int kSlab = tc::kSlabBytes;
constexpr int kStagingBytes = 4 * 32 * 128;  // per epilogue warp 32 rows of 64 values

enum Form { kRowsWide, kRowsTurned, kOuter };  // weight's columns along memory; its reduced index along memory; grad_weight

template <int BN> constexpr int Stages() { return BN == 256 ? 4 : (BN == 128 ? 6 : 8); }
template <int BN> constexpr int StageBytes() { return kRows * 128 + BN * 128; }
template <int BN> constexpr int SharedBytes() { return 1024 + Stages<BN>() * StageBytes<BN>() + kStagingBytes + 256; }

struct Params {
    SegmentPointers ptr;
    void* out;
    int64_t m, n, k;   // rows form: n columns, k reduced; outer form: m x n results per segment
    bool whole_a, whole_b;  // MN-major operands: all slabs in one load
    bool vec;               // rows of out start on 16-byte boundaries
    int64_t chunk;     // of the reduced index per partial result; 0: all of it in one piece
    int64_t pieces;    // rows form: pieces of the reduced index
    float* partial;    // outer form [slots][m][n], rows form [pieces][rows][n]
    WaitSettings wait;
};

struct Barriers {
    uint64_t full[8], empty[8], done[2], free[2], drain;
    uint32_t tmem, stop;
};

// Loads of kBoxRows rows that cover the first `rows` of a block's rows.
__device__ __forceinline__ int Boxes(int rows) { return rows <= 0 ? 0 : min(rows + kBoxRows - 1, kRows) / kBoxRows; }

template <class T> __device__ __forceinline__ uint32_t TwoOf(uint32_t a, uint32_t b)
{
    uint32_t word;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(__uint_as_float(a), __uint_as_float(b));
        memcpy(&word, &p, 4);
    } else {
        const __half2 p = __floats2half2_rn(__uint_as_float(a), __uint_as_float(b));
        memcpy(&word, &p, 4);
    }
    return word;
}

template <class T, int BN, int FORM>
__global__ void __launch_bounds__(kThreads, 1)
    TensorKernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_tail,
                 const __grid_constant__ CUtensorMap map_b, const Params p)
{
    constexpr int kStages = Stages<BN>();
    constexpr int kStage = StageBytes<BN>();
    extern __shared__ unsigned char raw[];
    unsigned char* smem = raw + ((1024 - (tc::Shared(raw) & 1023)) & 1023);
    unsigned char* staging = smem + kStages * kStage;
    Barriers& bar = *reinterpret_cast<Barriers*>(staging + kStagingBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            tc::BarInit(&bar.full[i], 1);
            tc::BarInit(&bar.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::BarInit(&bar.done[i], 1);
            tc::BarInit(&bar.free[i], 4);
        }
        tc::BarInit(&bar.drain, 1);
        bar.stop = 0;
        tc::BarInitFence();
    }
    if (warp == 2) {
        tc::TmemAlloc(&bar.tmem);
    }
    tc::FenceBefore();
    __syncthreads();
    tc::FenceAfter();
    const uint32_t tmem = bar.tmem;
    const tc::Waiter wait{&bar.stop, p.wait};

    // Rows, widths and tile numbers fit 32 bits (checked on the host); offsets in memory are formed in 64.
    const int n = static_cast<int>(p.n), m = static_cast<int>(p.m), width = static_cast<int>(p.k), chunk = static_cast<int>(p.chunk);
    const int across = (n + BN - 1) / BN;
    const int down = FORM == kOuter ? (m + kRows - 1) / kRows : 1, pieces = static_cast<int>(p.pieces);
    SegmentWalk<FORM == kOuter ? 0 : kRows, int> walk;
    if (warp != 2 && warp != 3 && (FORM != kOuter || chunk > 0)) {
        walk.Start(p.ptr, FORM == kOuter ? chunk : kRows);
    }
    // Tile t: its segment, first result row and column, and the range of the reduced index.
    int segment = 0, row = 0, row_end = 0, column = 0, from = 0, depth = 0, piece = 0;
    auto find = [&](int t) {
        if constexpr (FORM != kOuter) {
            piece = t % pieces;
            t /= pieces;
        }
        column = t % across * BN;
        t /= across;
        if constexpr (FORM == kOuter) {
            row = t % down * kRows;
            row_end = m;
            segment = t / down;  // in pieces: the piece, then its target
            if (chunk > 0) {
                if (!walk.Seek(p.ptr, segment)) {
                    return false;
                }
                segment = PieceTarget(walk, chunk);
                from = walk.row;
                depth = min(walk.row_end - from, chunk);
                return true;
            }
            if (segment >= p.ptr.segments) {
                return false;
            }
            int end;
            p.ptr.Range<int>(segment, from, end);
            depth = end - from;
            return true;
        } else {
            if (!walk.Seek(p.ptr, t)) {
                return false;
            }
            segment = walk.segment;
            row = walk.row;
            row_end = walk.row_end;
            from = piece * chunk;
            depth = chunk > 0 ? min(chunk, width - from) : width;
            return true;
        }
    };

    uint32_t filled = 0;  // stages the loading warp has asked for
    if (warp == 0) {
        bool going = true;
        for (int t = blockIdx.x; going && find(t); t += gridDim.x) {
            for (int k = 0; k < depth; k += kDepth, ++filled) {
                const uint32_t s = filled % kStages;
                going = wait.Warp(&bar.empty[s], ((filled / kStages) & 1) ^ 1);
                if (!going) {
                    break;
                }
                if (lane == 0) {
                    const uint32_t a = tc::Shared(smem) + s * kStage, b = a + kRows * 128;
                    const uint32_t full = tc::Shared(&bar.full[s]);
                    if constexpr (FORM == kOuter) {
                        tc::BarExpect(&bar.full[s], kStage);
                        tc::LoadSlabs(map_a, full, a, row, from + k, 0, kRows / 64, p.whole_a);
                        tc::LoadSlabs(map_b, full, b, column, from + k, 0, BN / 64, p.whole_b);
                    } else {
                        // Only the rows that are the segment's, to the next 32; what else lies in the stage is multiplied into
                        // rows that are not stored.
                        const int boxes = Boxes(row_end - row);
                        tc::BarExpect(&bar.full[s], boxes * kBoxRows * 128 + BN * 128);
                        if (boxes * kBoxRows == kRows) {
                            tc::LoadTo(map_a, full, a, from + k, row);
                        } else {
                            for (int i = 0; i < boxes; ++i) {
                                tc::LoadTo(map_tail, full, a + i * kBoxRows * 128, from + k, row + i * kBoxRows);
                            }
                        }
                        if constexpr (FORM == kRowsTurned) {
                            tc::LoadTo(map_b, full, b, from + k, column, segment);
                        } else {
                            tc::LoadSlabs(map_b, full, b, column, from + k, segment, BN / 64, p.whole_b);
                        }
                    }
                }
                __syncwarp();
            }
        }
    } else if (warp == 1) {
        constexpr uint32_t shape = tc::Shape(kRows, BN, std::is_same<T, __nv_bfloat16>::value ? 1 : 0, FORM == kOuter, FORM != kRowsTurned);
        // One thread issues.  The tensor cores run dry where it dawdles between two stages, so stage and parity advance without
        // divisions, operand descriptors differ by a constant, and the next stage is looked at before it is needed (18944 x 4096 ->
        // 2048 bf16, a warp-wide loop without these: 235 us; with them 223 us).
        uint32_t s = 0, parity = 0, tiles = 0;
        bool going = true;
        const uint64_t a0 = tc::Operand(tc::Shared(smem), FORM == kOuter ? kSlab : 16, 1024);
        const uint64_t b0 = tc::Operand(tc::Shared(smem) + kRows * 128, FORM == kRowsTurned ? 16 : kSlab, 1024);
        for (int t = blockIdx.x; going && find(t); t += gridDim.x) {
            if (depth == 0) {
                continue;
            }
            const uint32_t half = tiles & 1;
            auto multiply = [&](int k) {  // one stage
                tc::FenceAfter();
                const uint64_t da = a0 + s * (kStage >> 4), db = b0 + s * (kStage >> 4);
#pragma unroll
                for (int i = 0; i < kDepth / 16; ++i) {
                    tc::MmaF16(tmem + half * BN, da + i * (FORM == kOuter ? 2048 >> 4 : 32 >> 4),
                                     db + i * (FORM == kRowsTurned ? 32 >> 4 : 2048 >> 4), shape, k > 0 || i > 0);
                }
                tc::Commit(&bar.empty[s]);
            };
            const int whole = FORM == kOuter ? depth / kDepth * kDepth : depth;
            if (lane == 0) {
                going = wait(&bar.free[half], ((tiles >> 1) & 1) ^ 1);
                tc::FenceAfter();
                bool landed = going && whole > 0 && tc::BarTest(&bar.full[s], parity);
                for (int k = 0; going && k < whole; k += kDepth) {
                    going = landed || wait(&bar.full[s], parity);
                    if (!going) {
                        break;
                    }
                    multiply(k);
                    if (++s == kStages) {
                        s = 0;
                        parity ^= 1;
                    }
                    landed = k + kDepth < whole && tc::BarTest(&bar.full[s], parity);
                }
            }
            going = __shfl_sync(0xffffffffu, going ? 1 : 0, 0) != 0;
            if constexpr (FORM == kOuter) {
                s = __shfl_sync(0xffffffffu, s, 0);
                parity = __shfl_sync(0xffffffffu, parity, 0);
                if (whole < depth && going) {
                    going = wait.Warp(&bar.full[s], parity);
                    if (going) {
                        // Rows of the next segment: zero them in every slab of both operands.
                        unsigned char* stage = smem + s * kStage;
                        for (int i = (depth - whole) * 8 + lane; i < kDepth * 8; i += 32) {
#pragma unroll
                            for (int slab = 0; slab < kStage / kSlab; ++slab) {
                                *reinterpret_cast<uint4*>(stage + slab * kSlab + i * 16) = make_uint4(0, 0, 0, 0);
                            }
                        }
                        tc::FenceAsync();
                        __syncwarp();
                        if (lane == 0) {
                            multiply(whole);
                        }
                        if (++s == kStages) {
                            s = 0;
                            parity ^= 1;
                        }
                    }
                }
            }
            if (lane == 0 && going) {
                tc::Commit(&bar.done[half]);
            }
            __syncwarp();
            ++tiles;
        }
    } else if (warp >= 4) {
        const int quarter = warp - 4;
        unsigned char* mine = staging + quarter * (32 * 128);
        T* out = static_cast<T*>(p.out);
        uint32_t tiles = 0;
        bool going = true;
        for (int t = blockIdx.x; going && find(t); t += gridDim.x) {
            const uint32_t half = tiles & 1;
            if (depth > 0) {
                going = wait.Warp(&bar.done[half], (tiles >> 1) & 1);
                if (!going) {
                    break;
                }
                tc::FenceAfter();
            }
            const bool in_piece = chunk > 0 && (FORM != kOuter || (segment & 1) == 0);  // else a whole sum
            const int64_t result = FORM == kOuter && chunk > 0 ? segment >> 1 : segment;
            T* to = out + (FORM == kOuter ? result * p.m * p.n : 0);
            float* sums = p.partial + (FORM == kOuter ? result * p.m * p.n : piece * p.ptr.rows * p.n);
            const int first = row + quarter * 32;
#pragma unroll 1
            for (int c = 0; c < BN; c += 64) {
                if (column + c >= n) {
                    break;
                }
                uint32_t words[32];
                if (depth > 0) {
                    uint32_t low[32], high[32];
                    const uint32_t at = tmem + half * BN + c + (static_cast<uint32_t>(quarter * 32) << 16);
                    tc::TmemLoad32(at, low);
                    tc::TmemLoad32(at + 32, high);
                    tc::TmemWait();
                    if (in_piece) {
                        // A piece of the sum, kept in fp32: 32 columns are 128 bytes.
#pragma unroll
                        for (int side = 0; side < 2; ++side) {
                            const uint32_t(&v)[32] = side == 0 ? low : high;
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                *reinterpret_cast<uint4*>(mine + tc::Staged<128>(lane, i)) =
                                    make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                            }
                            __syncwarp();
                            const int col = column + c + side * 32;
                            tc::StoreStaged<128>(mine, sums + first * p.n + col, p.n, row_end - first, n - col, n % 4 == 0);
                            __syncwarp();
                        }
                        continue;
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        words[i] = TwoOf<T>(low[2 * i], low[2 * i + 1]);
                        words[16 + i] = TwoOf<T>(high[2 * i], high[2 * i + 1]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        words[i] = 0;
                    }
                }
                // Through shared memory, so that 8 lanes write 128 consecutive bytes of a row.
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    *reinterpret_cast<uint4*>(mine + tc::Staged<128>(lane, i)) =
                        make_uint4(words[4 * i], words[4 * i + 1], words[4 * i + 2], words[4 * i + 3]);
                }
                __syncwarp();
                tc::StoreStaged<128>(mine, to + first * p.n + column + c, p.n, row_end - first, n - column - c, p.vec);
                __syncwarp();
            }
            if (depth > 0) {
                tc::FenceBefore();
                __syncwarp();
                if (lane == 0) {
                    tc::BarArrive(&bar.free[half]);
                }
                ++tiles;
            }
        }
        if constexpr (FORM != kOuter) {
            // Rows of no segment (in pieces, the join writes them).
            const int64_t before = p.ptr.Raw(0), behind = p.ptr.Raw(p.ptr.segments);
            for (int64_t r = blockIdx.x * 4 + quarter; chunk == 0 && r < before + (p.ptr.rows - behind); r += gridDim.x * 4) {
                const int64_t at = r < before ? r : behind + (r - before);
                for (int c = lane; c < n; c += 32) {
                    out[at * p.n + c] = Narrow<T, float>(0.0f);
                }
            }
        }
    }
    __syncwarp();
    tc::FenceBefore();
    __syncthreads();
    // Past this barrier no wait of the block is left, so `stop` is final: a wait that ran out after a warp had issued its last
    // work is seen here, too.  What is in flight must end before the block's shared memory and TMEM are given up.
    if (bar.stop != 0) {
        if (warp == 0 && lane == 0) {
            for (uint32_t f = filled > kStages ? filled - kStages : 0; f < filled; ++f) {
                for (uint32_t i = 0; i < (1u << 15) && !tc::BarTry(&bar.full[f % kStages], (f / kStages) & 1); ++i) {
                }
            }
        } else if (warp == 1 && lane == 0) {
            tc::Commit(&bar.drain);
            for (uint32_t i = 0; i < (1u << 15) && !tc::BarTry(&bar.drain, 0); ++i) {
            }
        }
        __syncwarp();
        __syncthreads();
    }
    if (warp == 2) {
        tc::FenceAfter();
        tc::TmemFree(tmem);
    }
}

// What TMA asks of an operand: 16-byte aligned base and strides, extents that fit its fields.
bool Loadable(const void* base, int64_t stride, int64_t limit)
{
    return Aligned(base, 16) && stride % 8 == 0 && stride < (INT64_C(1) << 38) && limit < (INT64_C(1) << 31) - 512;
}

CUtensorMapDataType TypeOf(int type) { return type == OPSGNN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16; }

bool Map2(CUtensorMap* map, int type, const void* base, int64_t inner, int64_t rows, int64_t stride, int box_inner, int box_rows)
{
    const uint64_t sizes[2] = {static_cast<uint64_t>(inner), static_cast<uint64_t>(rows)};
    const uint64_t strides[1] = {static_cast<uint64_t>(stride) * 2};
    const uint32_t box[2] = {static_cast<uint32_t>(box_inner), static_cast<uint32_t>(box_rows)};
    return tc::EncodeMap(map, TypeOf(type), 2, base, sizes, strides, box);
}

template <class T, int BN, int FORM>
int Launch(const CUtensorMap& a, const CUtensorMap& tail, const CUtensorMap& b, const Params& p, int64_t tiles, cudaStream_t stream)
{
    if (tiles >= INT32_MAX - 4096) {
        return OPSGNN_ERR_UNSUPPORTED;
    }
    constexpr int kShared = SharedBytes<BN>();
    static std::atomic<uint64_t> allowed{0};
    OPSGNN_CUDA_TRY(static_cast<cudaError_t>(AllowShared(TensorKernel<T, BN, FORM>, kShared, allowed)));
    const int grid = static_cast<int>(std::min<int64_t>(std::max<int64_t>(tiles, 1), SmCount()));
    TensorKernel<T, BN, FORM><<<grid, kThreads, kShared, stream>>>(a, tail, b, p);
    return LaunchStatus();
}

// f(type tag, integral constant of a tile's columns); the outer form has no tiles of 64.
template <int FORM, class F> int ByType(int type, int columns, F&& f)
{
    using std::integral_constant;
    auto by_columns = [&](auto tag) {
        if constexpr (FORM != kOuter) {
            if (columns == 64) {
                return f(tag, integral_constant<int, 64>());
            }
        }
        return columns == 128 ? f(tag, integral_constant<int, 128>()) : f(tag, integral_constant<int, 256>());
    };
    return type == OPSGNN_BF16 ? by_columns(__nv_bfloat16()) : by_columns(__half());
}

// Columns of a tile of the rows form: 256, which reads an operand least often, unless that leaves half the SMs without a tile
// (`down`: most row tiles there can be).  2000 x 300 -> 300 in 5 segments: 16.8 us with 64 columns, 29.3 with 256.
int TileColumns(int64_t down, int64_t n)
{
    int columns = n <= 64 ? 64 : (n <= 128 ? 128 : 256);
    while (columns > 64 && down * CeilDiv(n, columns) * 2 <= SmCount()) {
        columns /= 2;
    }
    return columns;
}

int64_t RowTiles(int64_t rows, int64_t segments) { return rows / kRows + std::min(segments, rows); }

// Pieces of the reduced index of the rows form, summed apart and joined: where even narrow tiles leave half the SMs idle and the
// sum is long.  One row x 2048 -> 2048 (32 tiles, four pieces): 16.6 us in one piece, 12.8 us in pieces; 16 rows in 4 segments,
// 2048 -> 1024 (64 tiles, two pieces) 16.8 us either way, hence three pieces at least.
int64_t RowPieces(int64_t rows, int64_t segments, int64_t k, int64_t n)
{
    const int64_t tiles = RowTiles(rows, segments) * CeilDiv(n, 64);
    return tiles * 3 > SmCount() || k < 1536 ? 1 : std::min<int64_t>(SmCount() / std::max<int64_t>(tiles, 1), k / 512);
}

}  // namespace

int64_t RowsPartialBytes(int64_t rows, int64_t segments, int64_t k, int64_t n)
{
    const int64_t pieces = RowPieces(rows, segments, k, n);
    return pieces > 1 ? AlignUp(pieces * rows * n * 4, 256) : 0;
}

namespace {

// out[r] <- the sum of the pieces of row r, in their order; 0 for a row of no segment.
template <class T>
__global__ void __launch_bounds__(256) JoinRowsKernel(SegmentPointers ptr, int64_t n, int64_t pieces, const float* __restrict__ partial,
                                                      T* __restrict__ out)
{
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x, size = ptr.rows * n;
    if (i >= size) {
        return;
    }
    const int64_t row = i / n;
    float sum = 0.0f;
    if (row >= ptr.Raw(0) && row < ptr.Raw(ptr.segments)) {
#pragma unroll 4
        for (int64_t c = 0; c < pieces; ++c) {
            sum += __ldcs(partial + c * size + i);
        }
    }
    out[i] = Narrow<T, float>(sum);
}

}  // namespace

int RunRowsTensor(const RowsProblem& p, void* workspace, cudaStream_t stream)
{
    const bool turned = p.b_k == 1 && p.b_n != 1;
    const int64_t inner = turned ? p.k : p.n, other = turned ? p.n : p.k;
    const int64_t stride = StrideOf(turned ? p.b_n : p.b_k, other, inner, 8), lda = StrideOf(p.lda, p.ptr.rows, p.k, 8);
    const int64_t segment_stride = StrideOf(p.b_segment, p.ptr.segments, stride * other, 8);
    if ((p.in_type != OPSGNN_BF16 && p.in_type != OPSGNN_F16) || p.out_type != p.in_type || p.k < 1 || p.ptr.data == nullptr ||
        p.ptr.segments < 1 || p.ldo != p.n || (!turned && p.b_n != 1) || stride < inner ||
        segment_stride % 8 != 0 || segment_stride >= (INT64_C(1) << 38) || segment_stride < 1 || p.ptr.segments >= (INT64_C(1) << 30) ||
        !Loadable(p.a, lda, std::max(p.k, p.ptr.rows)) || !Loadable(p.b, stride, std::max(inner, other))) {
        return OPSGNN_ERR_UNSUPPORTED;
    }
    Params q{};
    q.ptr = p.ptr;
    q.out = p.out;
    q.n = p.n;
    q.k = p.k;
    q.vec = p.n % 8 == 0 && Aligned(p.out, 16);
    OPSGNN_CUDA_TRY(static_cast<cudaError_t>(CurrentWaitSettings(&q.wait)));
    const int64_t down = RowTiles(p.ptr.rows, p.ptr.segments);
    const int64_t pieces = workspace != nullptr ? RowPieces(p.ptr.rows, p.ptr.segments, p.k, p.n) : 1;
    q.chunk = pieces > 1 ? AlignUp(CeilDiv(p.k, pieces), kDepth) : 0;
    q.pieces = pieces > 1 ? CeilDiv(p.k, q.chunk) : 1;
    q.partial = static_cast<float*>(workspace);
    const int columns = TileColumns(down, p.n);
    q.whole_b = tc::WholeSlabs(p.n);
    CUtensorMap a, tail, b;
    const uint64_t sizes[3] = {static_cast<uint64_t>(inner), static_cast<uint64_t>(other), static_cast<uint64_t>(p.ptr.segments)};
    const uint64_t strides[2] = {static_cast<uint64_t>(stride) * 2, static_cast<uint64_t>(segment_stride) * 2};
    const uint32_t box[3] = {64, static_cast<uint32_t>(columns), 1};
    const CUtensorMapDataType type = TypeOf(p.in_type);
    // (with fewer rows than a full tile's last box reaches, every tile is short and the first map is never used)
    if ((p.ptr.rows > kRows - kBoxRows && !Map2(&a, p.in_type, p.a, p.k, p.ptr.rows, lda, kDepth, kRows)) ||
        !Map2(&tail, p.in_type, p.a, p.k, p.ptr.rows, lda, kDepth, kBoxRows) ||
        !(turned ? tc::EncodeMap(&b, type, 3, p.b, sizes, strides, box)
                 : tc::EncodeSlabs(&b, type, p.b, p.n, p.k, p.ptr.segments, stride * 2, segment_stride * 2, columns / 64))) {
        return OPSGNN_ERR_UNSUPPORTED;
    }
    if (p.ptr.rows <= kRows - kBoxRows) {
        a = tail;
    }
    auto run = [&](auto tag, auto width) {
        using T = decltype(tag);
        constexpr int BN = decltype(width)::value;
        const int64_t tiles = down * CeilDiv(p.n, BN) * q.pieces;
        return turned ? Launch<T, BN, kRowsTurned>(a, tail, b, q, tiles, stream) : Launch<T, BN, kRowsWide>(a, tail, b, q, tiles, stream);
    };
    const int status = ByType<kRowsWide>(p.in_type, columns, run);
    if (status != OPSGNN_OK || q.pieces == 1) {
        return status;
    }
    const unsigned grid = static_cast<unsigned>(CeilDiv(p.ptr.rows * p.n, 256));
    if (p.in_type == OPSGNN_BF16) {
        JoinRowsKernel<<<grid, 256, 0, stream>>>(p.ptr, p.n, q.pieces, q.partial, static_cast<__nv_bfloat16*>(p.out));
    } else {
        JoinRowsKernel<<<grid, 256, 0, stream>>>(p.ptr, p.n, q.pieces, q.partial, static_cast<__half*>(p.out));
    }
    return LaunchStatus();
}

namespace {

// out[e][i] <- the sum of the pieces of segment e, in their order; 0 for an empty one.
template <class T, int VEC>
__global__ void __launch_bounds__(256) JoinKernel(SegmentPointers ptr, int chunk, int per, int64_t size, const float* __restrict__ partial,
                                                  T* __restrict__ out)
{
    // `per` segments at a time, a lane of every warp looks at one; those of one piece are done already.
    const int lane = threadIdx.x & 31;
    const int64_t i = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * VEC;
    for (int64_t e0 = static_cast<int64_t>(blockIdx.y) * per; e0 < ptr.segments; e0 += static_cast<int64_t>(gridDim.y) * per) {
        int begin = 0, pieces = 1;
        if (lane < per && e0 + lane < ptr.segments) {
            int64_t first, end;
            ptr.Range<int64_t>(e0 + lane, first, end);
            begin = static_cast<int>(first);
            pieces = static_cast<int>((end - first + chunk - 1) / chunk);
        }
        unsigned left = __ballot_sync(0xffffffffu, pieces != 1);
        while (left != 0) {
            const int owner = __ffs(left) - 1;
            left &= left - 1;
            const int slot = PieceSlot(__shfl_sync(0xffffffffu, begin, owner), false, chunk);
            const int count = __shfl_sync(0xffffffffu, pieces, owner);
            if (i >= size) {
                continue;
            }
            float sum[VEC] = {};
#pragma unroll 8
            for (int c = 0; c < count; ++c) {
                const int64_t at = slot + 2 * c + (c == count - 1 ? 1 : 0);
                const Pack<float, VEC> v = LoadPlain<float, VEC>(partial + at * size + i);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    sum[j] += v.v[j];
                }
            }
            StorePlain<T, VEC>(out + (e0 + owner) * size + i, Repack<T, float, VEC>(sum));
        }
    }
}

}  // namespace

int64_t OuterChunk(int64_t rows, int64_t segments, int64_t k, int64_t n)
{
    // A result tile is one block's sequential sum over a segment's rows.  With fewer tiles than SMs the rows are cut into
    // pieces (200003 x 256 -> 256 in 13 segments, fp32: one piece each 1271 us, in pieces 303 us); with few rows, partial results
    // would cost more than they give (4096 x 256 -> 256 in 32 segments, bf16: 10.5 us in one piece each, 22.9 us in pieces).  Two
    // rounds of tiles over the SMs where a result is a few tiles (bf16, the first case: 51 us, four rounds 65.6 us), four where it
    // is many and two would leave the second round half empty (two segments, 32768 x 2048 -> 1024: 131 us, two rounds 148 us).  A
    // segment's last piece is half full on average.
    const int64_t tiles = CeilDiv(k, kRows) * CeilDiv(n, n <= 128 ? 128 : 256);
    if (rows < 8192 || segments >= (INT64_C(1) << 30)) {  // (twice a segment's number has to fit 32 bits)
        return 0;
    }
    int64_t length = 0;
    if (tiles * segments < SmCount()) {
        const int64_t rounds = tiles * 8 <= SmCount() ? 2 : 4;
        length = CeilDiv(rows, std::max<int64_t>(1, SmCount() * rounds / tiles - segments / 2));
    } else if (tiles * 4 <= SmCount()) {
        // Enough tiles for all SMs when segments are alike: only those of twice the mean length and more are cut, as one long
        // segment would keep its few SMs busy alone.  bf16, whole against cut: 200003 x 256 -> 256 in 100 segments, half of the
        // rows in one 561 and 61 us, lengths like 1 / i 269 and 74 us, lengths alike 52 and 56 us (finding the pieces, and the
        // join's launch); 65536 x 64 -> 64 in 500 segments 143 and 32 us, 59 and 30 us, 13 and 22 us.  A result of more tiles
        // keeps a quarter of the SMs busy by itself and is not cut: its partial results are large.
        length = std::max(CeilDiv(rows * tiles, 2 * SmCount()), CeilDiv(2 * rows, segments));
    }
    const int64_t chunk = std::max<int64_t>(256, AlignUp(length, kDepth));
    return length == 0 || chunk >= rows ? 0 : chunk;
}

int64_t OuterPartialBytes(int64_t rows, int64_t segments, int64_t k, int64_t n)
{
    const int64_t chunk = OuterChunk(rows, segments, k, n);
    return chunk > 0 ? AlignUp(PieceSlots(rows, chunk) * k * n * 4, 256) : 0;
}

int JoinPieces(const OuterProblem& p, int64_t chunk, const float* partial, cudaStream_t stream)
{
    const int64_t size = p.k * p.n;
    auto run = [&](auto tag) {
        using T = decltype(tag);
        const bool vec = size % 4 == 0 && Aligned(p.out, 16);
        // Enough blocks for the machine; with many segments a block looks at up to 32 of them at once.
        const int64_t across = CeilDiv(size, vec ? 1024 : 256), most = CeilDiv(static_cast<int64_t>(SmCount()) * 32, across);
        const int per = static_cast<int>(std::min<int64_t>(32, CeilDiv(p.ptr.segments, most)));
        const dim3 grid(static_cast<unsigned>(across), static_cast<unsigned>(std::min(CeilDiv(p.ptr.segments, per), 4 * most)));
        if (vec) {
            JoinKernel<T, 4><<<grid, 256, 0, stream>>>(p.ptr, static_cast<int>(chunk), per, size, partial, static_cast<T*>(p.out));
        } else {
            JoinKernel<T, 1><<<grid, 256, 0, stream>>>(p.ptr, static_cast<int>(chunk), per, size, partial, static_cast<T*>(p.out));
        }
        return LaunchStatus();
    };
    switch (p.type) {
        case OPSGNN_F32:
            return run(float());
        case OPSGNN_F16:
            return run(__half());
        default:
            return run(__nv_bfloat16());
    }
}

int RunOuterTensor(const OuterProblem& p, void* workspace, cudaStream_t stream)
{
    const int64_t lda = StrideOf(p.lda, p.ptr.rows, p.k, 8), ldb = StrideOf(p.ldb, p.ptr.rows, p.n, 8);
    if ((p.type != OPSGNN_BF16 && p.type != OPSGNN_F16) || p.ptr.rows < 1 ||
        !Loadable(p.a, lda, std::max(p.k, p.ptr.rows)) || !Loadable(p.b, ldb, std::max(p.n, p.ptr.rows))) {
        return OPSGNN_ERR_UNSUPPORTED;
    }
    Params q{};
    q.ptr = p.ptr;
    q.out = p.out;
    q.m = p.k;
    q.n = p.n;
    q.vec = p.n % 8 == 0 && Aligned(p.out, 16);
    q.chunk = OuterChunk(p.ptr.rows, p.ptr.segments, p.k, p.n);
    q.partial = static_cast<float*>(workspace);
    OPSGNN_CUDA_TRY(static_cast<cudaError_t>(CurrentWaitSettings(&q.wait)));
    const bool narrow = p.n <= 128;
    q.whole_a = tc::WholeSlabs(p.k);
    q.whole_b = tc::WholeSlabs(p.n);
    CUtensorMap a, b;
    if (!tc::EncodeSlabs(&a, TypeOf(p.type), p.a, p.k, p.ptr.rows, 1, lda * 2, 16, kRows / 64) ||
        !tc::EncodeSlabs(&b, TypeOf(p.type), p.b, p.n, p.ptr.rows, 1, ldb * 2, 16, narrow ? 2 : 4)) {
        return OPSGNN_ERR_UNSUPPORTED;
    }
    auto run = [&](auto tag, auto width) {
        using T = decltype(tag);
        constexpr int BN = decltype(width)::value;
        const int64_t results = q.chunk > 0 ? p.ptr.rows / q.chunk + p.ptr.segments : p.ptr.segments;
        return Launch<T, BN, kOuter>(a, a, b, q, results * CeilDiv(p.k, kRows) * CeilDiv(p.n, BN), stream);
    };
    const int status = ByType<kOuter>(p.type, narrow ? 128 : 256, run);
    return status == OPSGNN_OK && q.chunk > 0 ? JoinPieces(p, q.chunk, q.partial, stream) : status;
}

}  // namespace segmm
}  // namespace opsgnn
