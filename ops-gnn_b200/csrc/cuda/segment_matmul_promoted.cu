// Segment products whose tensor-core sums are short and are added up in fp32 registers: block-scaled 8-bit values, and fp32.
//
// 8 bits: a sum over 128 values of the reduced index (one block, one scale per row and one per weight tile) is formed by
// tcgen05.mma in TMEM; the epilogue warps multiply it by the two scales and add it to registers while the next block is
// multiplied into the other half of TMEM.
//
// fp32: every operand value is x = x1 + x2 + x3 with bf16 terms (8 significant bits each, so the three hold all 24), and
//     a b = a1 b1 + (a1 b2 + a2 b1) + (a1 b3 + a2 b2 + a3 b1) + terms below 2^-24 of |a b|, which are left out.
// The six products are exact; 64 values of the reduced index are summed in TMEM, a1 b1 last, so that only the last four
// instructions add at full magnitude, then the sum moves to registers, which round to nearest.  Six bf16 products cost
// 1/6 of the bf16 rate, four times what fp32 multiply-adds reach.  Values below 2^-110 lose low bits, as their third term lies
// below the smallest bf16.  An infinity, a number that rounds to one in bf16 or a sum that overflows breaks the split
// (inf - inf, inf * 0): where the largest magnitudes of the operands, noted as the terms are made, leave one of these possible,
// results that are not finite are computed again from the fp32 operands, after the block's last tile and with nobody waiting
// (Repair).  Where they do not, such a result stems from a NaN and is right.
//
// Layout as in segment_matmul_tc.cu (one persistent block per SM: a loading warp, a multiplying warp), with eight summing
// warps, each 32 rows x half the columns of a tile, whose sums need BN / 2 registers a thread.  The first four warps hand
// registers over, and a warp of these looks the tiles up for the summing warps: a register spilled in their inner loop
// doubles the time, since waiting on a barrier drops the first-level cache that holds it.
//
// What bounds the 8-bit product: reading every block's sums out of TMEM.  128 x 256 sums are 128 KB at 128 bytes per cycle and
// SM, twice the 512 cycles of the block's multiplication.  Measured, 18944 x 4096 -> 2048: 171 us (1.86 PFLOP/s); with the
// sums left unread 130 us, with one sum over all of K 117 us.  Sixteen summing warps in place of eight (187 us) and pairs of
// blocks that halve the operand traffic (170 us) gain nothing.
#include <algorithm>

#include "segment_matmul.cuh"
#include "segment_tile.cuh"
#include "tensor_core.cuh"

namespace opsgnn {
namespace segmm {
namespace {

constexpr int kRows = 128;
constexpr int kBoxRows = 32;  // rows of a per load where a tile is not full
constexpr int kSumWarps = 8;
constexpr int kThreads = 128 + 32 * kSumWarps;
constexpr int kStages = 4;
constexpr int kSlab = tc::kSlabBytes;
constexpr int kStagingBytes = 8 * 32 * 128;
// 384 threads are launched with 168 registers each; 128 * 72 + 256 * 216 = 384 * 168.
constexpr int kRegsIssue = 72, kRegsSum = 216;

enum Form { kRowsWide, kRowsTurned, kOuter };

template <int BN> constexpr int StageBytes() { return kRows * 128 + BN * 128; }
template <int BN> constexpr int SharedBytes() { return 1024 + kStages * StageBytes<BN>() + kStagingBytes + 256; }

struct Params {
    SegmentPointers ptr;
    void* out;
    const float* a_scale;
    const float* b_scale;
    int64_t m, n, k;                 // rows form: n columns, k reduced; outer form: m x n results per segment
    const float* a;                  // fp32: the operands as given, for results that are not finite
    const float* b;
    int64_t lda, ldb;                // outer form: ldb = row stride of b
    int64_t b_segment, b_k, b_n;
    const float* a_tops;             // fp32: largest magnitudes of parts of the operands (NaN left out)
    const float* b_tops;
    int a_parts, b_parts;
    bool whole_a, whole_b;  // MN-major operands: all slabs in one load
    bool vec;               // rows of out start on 16-byte boundaries
    int64_t chunk;     // outer form: rows per partial result; 0: a segment's rows in one piece
    float* partial;    // [slots][m][n]
    WaitSettings wait;
};

struct Barriers {
    uint64_t full[kStages], empty[kStages], done[2], free[2], drain;
    uint64_t told[2], taken[2];
    int32_t tile[2][5];          // for the summing warps: segment, row, row_end, column, depth
    uint32_t fills[kStages];  // loads asked for, per stage (loading warp)
    uint32_t tmem, stop;
    uint32_t odd;             // summing warps: 1 results that are not finite, 2 a wait that ran out
};

// Loads of kBoxRows rows that cover the first `rows` of a block's rows.
__device__ __forceinline__ int Boxes(int rows) { return rows <= 0 ? 0 : min(rows + kBoxRows - 1, kRows) / kBoxRows; }

template <class O> __device__ __forceinline__ uint32_t Word(const float* v)  // one 32-bit word of results
{
    uint32_t word;
    if constexpr (std::is_same<O, float>::value) {
        word = __float_as_uint(v[0]);
    } else if constexpr (std::is_same<O, __nv_bfloat16>::value) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(v[0], v[1]);
        memcpy(&word, &p, 4);
    } else {
        const __half2 p = __floats2half2_rn(v[0], v[1]);
        memcpy(&word, &p, 4);
    }
    return word;
}

// sum[i] += scale * part[i], two at a time.
template <int N> __device__ __forceinline__ void Add(float (&sum)[N], int at, const uint32_t (&part)[32], float scale)
{
    const float2 s = make_float2(scale, scale);
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        const float2 r = __ffma2_rn(s, make_float2(__uint_as_float(part[i]), __uint_as_float(part[i + 1])),
                                    make_float2(sum[at + i], sum[at + i + 1]));
        sum[at + i] = r.x;
        sum[at + i + 1] = r.y;
    }
}

// A tile: its segment, first result row and column, and the range of the reduced index.
struct Tile {
    int segment = 0, row = 0, row_end = 0, column = 0, from = 0, depth = 0;
};
template <int FORM> using Walk = SegmentWalk<FORM == kOuter ? 0 : kRows, int>;

template <int FORM> __device__ __forceinline__ void StartWalk(const Params& p, Walk<FORM>& walk)
{
    if (FORM != kOuter || p.chunk > 0) {
        walk.Start(p.ptr, FORM == kOuter ? static_cast<int>(p.chunk) : kRows);
    }
}

// Tile t of `across` columns and `down` rows of tiles, by a whole warp, with ascending t; false past the last one.  Rows, widths and
// tile numbers fit 32 bits (checked on the host); offsets in memory are formed in 64.
template <int BN, int FORM>
__device__ __forceinline__ bool FindTile(const Params& p, Walk<FORM>& walk, int t, int across, int down, int width, int m, int chunk, Tile& tile)
{
    tile.column = t % across * BN;
    t /= across;
    if constexpr (FORM == kOuter) {
        tile.row = t % down * kRows;
        tile.row_end = m;
        tile.segment = t / down;  // in pieces: the piece, then its target
        if (chunk > 0) {
            if (!walk.Seek(p.ptr, tile.segment)) {
                return false;
            }
            tile.segment = PieceTarget(walk, chunk);
            tile.from = walk.row;
            tile.depth = min(walk.row_end - tile.from, chunk);
            return true;
        }
        if (tile.segment >= p.ptr.segments) {
            return false;
        }
        int end;
        p.ptr.Range<int>(tile.segment, tile.from, end);
        tile.depth = end - tile.from;
        return true;
    } else {
        if (!walk.Seek(p.ptr, t)) {
            return false;
        }
        tile.segment = walk.segment;
        tile.row = walk.row;
        tile.row_end = walk.row_end;
        tile.depth = width;
        return true;
    }
}

// Where the results of a tile go.  Outer form: a piece of a longer sum (fp32 as the result) goes to `partial`.
template <class O, int FORM> __device__ __forceinline__ O* ResultsOf(const Params& p, int segment)
{
    O* to = static_cast<O*>(p.out);
    if constexpr (FORM == kOuter) {
        const bool in_piece = p.chunk > 0 && (segment & 1) == 0;
        to = (in_piece ? reinterpret_cast<O*>(p.partial) : to) + (p.chunk > 0 ? segment >> 1 : segment) * p.m * p.n;
    }
    return to;
}

// Barriers of the summing warps alone.
struct SumSync {
    __device__ __forceinline__ void operator()() const { asm volatile("bar.sync 1, %0;" ::"n"(32 * kSumWarps) : "memory"); }
};
__device__ __forceinline__ bool AnySum(bool mine)
{
    uint32_t any;
    asm volatile(
        "{\n"
        ".reg .pred p, q;\n"
        "setp.ne.u32 p, %1, 0;\n"
        "bar.red.or.pred q, 1, %2, p;\n"
        "selp.u32 %0, 1, 0, q;\n"
        "}\n"
        : "=r"(any)
        : "r"(static_cast<uint32_t>(mine)), "n"(32 * kSumWarps)
        : "memory");
    return any != 0;
}

// fp32, after a block's last tile: its results that are not finite, again from the operands as given, by the eight summing warps
// (thread: of these).  A function of its own, so that nothing of it weighs on the registers of the summing loop.  No wait
// depends on it, and it takes at most what the multiply-add kernel takes for the tiles concerned.  65536 x 512 -> 512 in four
// segments, forward and both gradients: 653 us; with a row of NaN 651 us, with one infinity 2993 us.
template <int BN, int FORM> __device__ __noinline__ void Repair(const Params& p, unsigned char* scratch, int thread)
{
    float a_top = 0.0f, b_top = 0.0f;
    for (int i = thread; i < p.a_parts; i += 32 * kSumWarps) {
        a_top = fmaxf(a_top, p.a_tops[i]);
    }
    for (int i = thread; i < p.b_parts; i += 32 * kSumWarps) {
        b_top = fmaxf(b_top, p.b_tops[i]);
    }
    float* shared_tops = reinterpret_cast<float*>(scratch);
    for (int d = 16; d > 0; d >>= 1) {
        a_top = fmaxf(a_top, __shfl_xor_sync(0xffffffffu, a_top, d));
        b_top = fmaxf(b_top, __shfl_xor_sync(0xffffffffu, b_top, d));
    }
    if ((thread & 31) == 0) {
        shared_tops[thread >> 5] = a_top;
        shared_tops[kSumWarps + (thread >> 5)] = b_top;
    }
    SumSync()();
    for (int w = 0; w < kSumWarps; ++w) {
        a_top = fmaxf(a_top, shared_tops[w]);
        b_top = fmaxf(b_top, shared_tops[kSumWarps + w]);
    }
    SumSync()();
    // The largest bf16 is 2^128 - 2^120.  The products of all terms add up to less than 2^127 where this bound is below 2^126.
    const float largest = __uint_as_float(0x7f7f0000u);
    const float terms = static_cast<float>(FORM == kOuter ? p.ptr.rows : p.k);
    if (a_top <= largest && b_top <= largest && a_top * b_top * terms < 0x1p126f) {
        return;
    }
    tile::Operands& shared = *reinterpret_cast<tile::Operands*>(scratch);
    const int n = static_cast<int>(p.n), m = static_cast<int>(p.m), width = static_cast<int>(p.k), chunk = static_cast<int>(p.chunk);
    const int across = (n + BN - 1) / BN, down = (m + kRows - 1) / kRows, below = thread / 16 * 4, right = thread % 16 * 4;
    // One warp finds the tiles for all eight, whose barriers have to agree.
    Walk<FORM> walk;
    if (thread < 32) {
        StartWalk<FORM>(p, walk);
    }
    Tile at;
    Tile* told = reinterpret_cast<Tile*>(scratch + sizeof(tile::Operands));
    for (int t = blockIdx.x;; t += gridDim.x) {
        if (thread < 32) {
            if (!FindTile<BN, FORM>(p, walk, t, across, down, width, m, chunk, at)) {
                at.segment = -1;
            }
            if (thread == 0) {
                *told = at;
            }
        }
        SumSync()();
        at = *told;
        SumSync()();
        if (at.segment < 0) {
            break;
        }
        float* to = ResultsOf<float, FORM>(p, at.segment);
        for (int part = 0; part < kRows / tile::kSize * (BN / tile::kSize); ++part) {
            const int64_t r0 = at.row + part / (BN / tile::kSize) * tile::kSize, c0 = at.column + part % (BN / tile::kSize) * tile::kSize;
            uint32_t odd = 0;  // which of the thread's 4 x 4 results
            for (int i = 0; i < 16; ++i) {
                const int64_t r = r0 + below + i / 4, c = c0 + right + i % 4;
                if (r < at.row_end && c < n && !(fabsf(to[r * n + c]) < INFINITY)) {
                    odd |= 1u << i;
                }
            }
            if (!AnySum(odd != 0)) {
                continue;
            }
            float sum[4][4] = {};
            if constexpr (FORM == kOuter) {
                tile::Multiply(
                    shared, thread, SumSync(), [&](int r, int64_t d) { return r0 + r < p.m ? p.a[(at.from + d) * p.lda + r0 + r] : 0.0f; },
                    [&](int64_t d, int c) { return c0 + c < n ? p.b[(at.from + d) * p.ldb + c0 + c] : 0.0f; }, false, false, at.depth,
                    sum);
            } else {
                const float* matrix = p.b + at.segment * p.b_segment;
                tile::Multiply(
                    shared, thread, SumSync(), [&](int r, int64_t d) { return r0 + r < at.row_end ? p.a[(r0 + r) * p.lda + d] : 0.0f; },
                    [&](int64_t d, int c) { return c0 + c < n ? matrix[d * p.b_k + (c0 + c) * p.b_n] : 0.0f; }, true, p.b_k == 1,
                    at.depth, sum);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if ((odd >> i) & 1u) {
                    to[(r0 + below + i / 4) * n + c0 + right + i % 4] = sum[i / 4][i % 4];
                }
            }
        }
    }
}

template <bool F8, class O, int BN, int FORM>
__global__ void __launch_bounds__(kThreads, 1)
    PromotedKernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_tail,
                   const __grid_constant__ CUtensorMap map_b, const __grid_constant__ Params p)
{
    constexpr int kStage = StageBytes<BN>();
    constexpr int kDepth = F8 ? 128 : 64;  // values of the reduced index in one 128-byte row
    extern __shared__ unsigned char raw[];
    unsigned char* smem = raw + ((1024 - (tc::Shared(raw) & 1023)) & 1023);
    unsigned char* staging = smem + kStages * kStage;
    Barriers& bar = *reinterpret_cast<Barriers*>(staging + kStagingBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            tc::BarInit(&bar.full[i], 1);
            tc::BarInit(&bar.empty[i], 1);
            bar.fills[i] = 0;
        }
        for (int i = 0; i < 2; ++i) {
            tc::BarInit(&bar.done[i], 1);
            tc::BarInit(&bar.free[i], kSumWarps);
            tc::BarInit(&bar.told[i], 1);
            tc::BarInit(&bar.taken[i], kSumWarps);
        }
        tc::BarInit(&bar.drain, 1);
        bar.stop = 0;
        bar.odd = 0;
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

    const int n = static_cast<int>(p.n), m = static_cast<int>(p.m), width = static_cast<int>(p.k), chunk = static_cast<int>(p.chunk);
    const int across = (n + BN - 1) / BN, down = (m + kRows - 1) / kRows;
    Walk<FORM> walk;
    if (warp != 2 && warp < 4) {
        StartWalk<FORM>(p, walk);
    }
    Tile at;
    const int &segment = at.segment, &row = at.row, &row_end = at.row_end, &column = at.column, &from = at.from, &depth = at.depth;
    auto find = [&](int t) { return FindTile<BN, FORM>(p, walk, t, across, down, width, m, chunk, at); };

    // 8 bits: the stages are a ring.  fp32: stages 0 and 1 take turns with the first terms of both operands, stage 2 holds the
    // second, stage 3 the third; every term is loaded once per 64 values of the reduced index and used in up to three products
    // (a ring of operand pairs per product read 288 KB in place of 144).  The single stages are read first and refilled while
    // the other products run; a1 b1 comes last, see above.
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue));
        if (warp == 0) {
            // One stage: rows and columns of the tile at k, terms pa and pb.
            auto load = [&](uint32_t s, uint32_t use, int k, int pa, int pb) {
                if (!wait.Warp(&bar.empty[s], (use & 1) ^ 1)) {
                    return false;
                }
                if (lane == 0) {
                    const uint32_t a = tc::Shared(smem) + s * kStage, b = a + kRows * 128;
                    const uint32_t full = tc::Shared(&bar.full[s]);
                    bar.fills[s] = use + 1;
                    if constexpr (FORM == kOuter) {
                        tc::BarExpect(&bar.full[s], kStage);
                        tc::LoadSlabs(map_a, full, a, row, from + k, pa, kRows / 64, p.whole_a);
                        tc::LoadSlabs(map_b, full, b, column, from + k, pb, BN / 64, p.whole_b);
                    } else {
                        // Only the rows that are the segment's, to the next 32; what else lies in the stage is multiplied into
                        // rows that are not stored.
                        const int boxes = Boxes(row_end - row);
                        const int matrix = pb * static_cast<int>(p.ptr.segments) + segment;
                        tc::BarExpect(&bar.full[s], boxes * kBoxRows * 128 + BN * 128);
                        if (boxes * kBoxRows == kRows) {
                            tc::LoadTo(map_a, full, a, k, row, pa);
                        } else {
                            for (int i = 0; i < boxes; ++i) {
                                tc::LoadTo(map_tail, full, a + i * kBoxRows * 128, k, row + i * kBoxRows, pa);
                            }
                        }
                        if constexpr (FORM == kRowsTurned) {
                            tc::LoadTo(map_b, full, b, k, column, matrix);
                        } else {
                            tc::LoadSlabs(map_b, full, b, column, k, matrix, BN / 64, p.whole_b);
                        }
                    }
                }
                __syncwarp();
                return true;
            };
            uint32_t blocks = 0;
            bool going = true;
            for (int t = blockIdx.x; going && find(t); t += gridDim.x) {
                for (int k = 0; going && k < depth; k += kDepth, ++blocks) {
                    if constexpr (F8) {
                        going = load(blocks % kStages, blocks / kStages, k, 0, 0);
                    } else {
                        going = load(blocks & 1, blocks >> 1, k, 0, 0) && load(3, blocks, k, 2, 2) && load(2, blocks, k, 1, 1);
                    }
                }
            }
        } else if (warp == 1) {
            constexpr uint32_t shape = tc::Shape(kRows, BN, F8 ? 0 : 1, FORM == kOuter, FORM != kRowsTurned);
            // One thread issues (but for the zeroing); see segment_matmul_tc.cu on why its loop is lean.
            bool going = true;
            const uint64_t a0 = tc::Operand(tc::Shared(smem), FORM == kOuter ? kSlab : 16, 1024);
            const uint64_t b0 = tc::Operand(tc::Shared(smem) + kRows * 128, FORM == kRowsTurned ? 16 : kSlab, 1024);
            // One product of kDepth values: a of one stage, b of another.
            auto multiply = [&](uint32_t sa, uint32_t sb, uint32_t half, bool add) {
                const uint64_t da = a0 + sa * (kStage >> 4), db = b0 + sb * (kStage >> 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint64_t ai = da + i * (FORM == kOuter ? 2048 >> 4 : 32 >> 4);
                    const uint64_t bi = db + i * (FORM == kRowsTurned ? 32 >> 4 : 2048 >> 4);
                    if constexpr (F8) {
                        tc::MmaF8(tmem + half * BN, ai, bi, shape, add || i > 0);
                    } else {
                        tc::MmaF16(tmem + half * BN, ai, bi, shape, add || i > 0);
                    }
                }
            };
            if constexpr (F8) {
                uint32_t s = 0, parity = 0, half = 0, half_parity = 1;
                for (int t = blockIdx.x; going && find(t); t += gridDim.x) {
                    if (lane == 0) {
                        bool landed = tc::BarTest(&bar.full[s], parity), freed = tc::BarTest(&bar.free[half], half_parity);
                        for (int k = 0; k < depth; k += kDepth) {
                            going = (freed || wait(&bar.free[half], half_parity)) && (landed || wait(&bar.full[s], parity));
                            if (!going) {
                                break;
                            }
                            tc::FenceAfter();
                            multiply(s, s, half, false);
                            tc::Commit(&bar.empty[s]);
                            tc::Commit(&bar.done[half]);
                            if (++s == kStages) {
                                s = 0;
                                parity ^= 1;
                            }
                            half ^= 1;
                            half_parity ^= half == 0 ? 1 : 0;
                            landed = k + kDepth < depth && tc::BarTest(&bar.full[s], parity);
                            freed = k + kDepth < depth && tc::BarTest(&bar.free[half], half_parity);
                        }
                    }
                    going = __shfl_sync(0xffffffffu, going ? 1 : 0, 0) != 0;
                }
            } else {
                uint32_t blocks = 0;
                // The six products of 64 values, with a wait (one thread's or the warp's) where a stage is first read.
                auto products = [&](auto&& ready) {
                    const uint32_t half = blocks & 1, s = blocks & 1;
                    if (!ready(&bar.free[half], ((blocks >> 1) & 1) ^ 1, -1) || !ready(&bar.full[s], (blocks >> 1) & 1, s) ||
                        !ready(&bar.full[3], blocks & 1, 3)) {
                        return false;
                    }
                    tc::FenceAfter();
                    if (lane == 0) {
                        multiply(3, s, half, false);     // a3 b1
                        multiply(s, 3, half, true);      // a1 b3
                        tc::Commit(&bar.empty[3]);
                    }
                    if (!ready(&bar.full[2], blocks & 1, 2)) {
                        return false;
                    }
                    tc::FenceAfter();
                    if (lane == 0) {
                        multiply(2, 2, half, true);      // a2 b2
                        multiply(2, s, half, true);      // a2 b1
                        multiply(s, 2, half, true);      // a1 b2
                        tc::Commit(&bar.empty[2]);
                        multiply(s, s, half, true);      // a1 b1
                        tc::Commit(&bar.empty[s]);
                        tc::Commit(&bar.done[half]);
                    }
                    return true;
                };
                for (int t = blockIdx.x; going && find(t); t += gridDim.x) {
                    const int whole = FORM == kOuter ? depth / kDepth : (depth + kDepth - 1) / kDepth;
                    const uint32_t before = blocks;
                    if (lane == 0) {
                        for (int i = 0; going && i < whole; ++i, ++blocks) {
                            going = products([&](uint64_t* barrier, uint32_t parity, int) { return wait(barrier, parity); });
                        }
                    }
                    going = __shfl_sync(0xffffffffu, going ? 1 : 0, 0) != 0;
                    blocks = before + whole;
                    if (FORM == kOuter && whole * kDepth < depth && going) {
                        // Rows of the next segment in the last stages are zeroed.
                        going = products([&](uint64_t* barrier, uint32_t parity, int stage) {
                            if (!wait.Warp(barrier, parity)) {
                                return false;
                            }
                            if (stage >= 0) {
                                unsigned char* data = smem + stage * kStage;
                                for (int i = (depth - whole * kDepth) * 8 + lane; i < kDepth * 8; i += 32) {
#pragma unroll
                                    for (int slab = 0; slab < kStage / kSlab; ++slab) {
                                        *reinterpret_cast<uint4*>(data + slab * kSlab + i * 16) = make_uint4(0, 0, 0, 0);
                                    }
                                }
                                tc::FenceAsync();
                                __syncwarp();
                            }
                            return true;
                        });
                        ++blocks;
                        __syncwarp();
                    }
                }
            }
        } else if (warp == 3) {
            // The tiles, looked up for the summing warps, whose registers hold nothing but sums.
            uint32_t turn = 0;
            bool going = true, more = true;
            for (int t = blockIdx.x; going && more; t += gridDim.x, ++turn) {
                more = find(t);
                going = wait.Warp(&bar.taken[turn & 1], ((turn >> 1) & 1) ^ 1);
                if (going && lane == 0) {
                    int32_t* tile = bar.tile[turn & 1];
                    tile[0] = more ? segment : -1;
                    tile[1] = row;
                    tile[2] = row_end;
                    tile[3] = column;
                    tile[4] = depth;
                    tc::BarArrive(&bar.told[turn & 1]);
                }
                __syncwarp();
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSum));
        constexpr int kMine = BN / 2;  // columns of this warp
        const int quarter = warp & 3, side = (warp - 4) >> 2;
        unsigned char* mine = staging + (warp - 4) * (32 * 128);
        const int scale_blocks = F8 ? (width + 127) / 128 : 0, scale_bands = F8 ? (n + 127) / 128 : 0;
        uint32_t blocks = 0, turn = 0;
        bool going = true;
        for (;; ++turn) {
            going = wait.Warp(&bar.told[turn & 1], (turn >> 1) & 1);
            if (!going) {
                break;
            }
            const volatile int32_t* tile = bar.tile[turn & 1];
            const int segment = tile[0], row = tile[1], row_end = tile[2], column = tile[3], depth = tile[4];
            __syncwarp();
            if (lane == 0) {
                tc::BarArrive(&bar.taken[turn & 1]);
            }
            if (segment < 0) {
                break;
            }
            float sum[kMine];
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                sum[i] = 0.0f;
            }
            const int col0 = column + side * kMine;
            const bool some = col0 < n;
            const int r0 = row + quarter * 32;
            const float* sa = nullptr;
            const float* sb = nullptr;
            float scale = 1.0f;
            if constexpr (F8) {
                sa = p.a_scale + static_cast<int64_t>(r0 + lane < row_end ? r0 + lane : row) * scale_blocks;
                sb = p.b_scale + (static_cast<int64_t>(segment) * scale_bands + (some ? col0 / 128 : 0)) * scale_blocks;
            }
            float next_a = 1.0f, next_b = 1.0f;  // the next block's scales, asked for one block ahead
            if constexpr (F8) {
                next_a = __ldg(sa);
                next_b = __ldg(sb);
            }
            const int last = (depth + kDepth - 1) / kDepth - 1;
            for (int kb = 0; kb <= last; ++kb, ++blocks) {
                const uint32_t half = blocks & 1;
                if constexpr (F8) {
                    scale = next_a * next_b;
                    next_a = __ldg(sa + min(kb + 1, last));
                    next_b = __ldg(sb + min(kb + 1, last));
                }
                going = wait.Warp(&bar.done[half], (blocks >> 1) & 1);
                if (!going) {
                    break;
                }
                tc::FenceAfter();
                const uint32_t at = tmem + half * BN + side * kMine + (static_cast<uint32_t>(quarter * 32) << 16);
                // Two loads in flight at a time; the half is handed back as soon as the last one is in registers.
                uint32_t low[32], high[32];
                if (some) {
                    tc::TmemLoad32(at, low);
                    tc::TmemLoad32(at + 32, high);
                    tc::TmemWait();
                    if constexpr (kMine == 128) {
                        Add(sum, 0, low, scale);
                        tc::TmemLoad32(at + 64, low);
                        Add(sum, 32, high, scale);
                        tc::TmemLoad32(at + 96, high);
                        tc::TmemWait();
                    }
                }
                tc::FenceBefore();
                __syncwarp();
                if (lane == 0) {
                    tc::BarArrive(&bar.free[half]);
                }
                if (some) {
                    Add(sum, kMine - 64, low, scale);
                    Add(sum, kMine - 32, high, scale);
                }
            }
            if (!going) {
                break;
            }
            O* to = ResultsOf<O, FORM>(p, segment);
            constexpr int kLine = 128 / sizeof(O);       // columns in 128 bytes
            constexpr int kPerWord = 4 / sizeof(O);
#pragma unroll
            for (int c = 0; c < kMine; c += kLine) {
                if (col0 + c < n) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        uint4 v;
                        v.x = Word<O>(&sum[c + (4 * i) * kPerWord]);
                        v.y = Word<O>(&sum[c + (4 * i + 1) * kPerWord]);
                        v.z = Word<O>(&sum[c + (4 * i + 2) * kPerWord]);
                        v.w = Word<O>(&sum[c + (4 * i + 3) * kPerWord]);
                        *reinterpret_cast<uint4*>(mine + tc::Staged<128>(lane, i)) = v;
                    }
                    __syncwarp();
                    tc::StoreStaged<128>(mine, to + r0 * p.n + col0 + c, p.n, row_end - r0, n - col0 - c, p.vec);
                    __syncwarp();
                }
            }
            if constexpr (!F8) {
                bool odd = false;
#pragma unroll
                for (int i = 0; i < kMine; ++i) {
                    odd |= !(fabsf(sum[i]) < INFINITY);
                }
                if (odd && r0 + lane < row_end) {  // what lies past the segment's rows is not a result
                    atomicOr(&bar.odd, 1u);
                }
            }
        }
        if constexpr (!F8) {
            if (!going) {
                atomicOr(&bar.odd, 2u);
            }
            SumSync()();
            if (bar.odd == 1) {
                Repair<BN, FORM>(p, staging, threadIdx.x - 128);
            }
        }
        if constexpr (FORM != kOuter) {
            // Rows of no segment.
            O* out = static_cast<O*>(p.out);
            const int64_t before = p.ptr.data != nullptr ? p.ptr.Raw(0) : 0;
            const int64_t behind = p.ptr.data != nullptr ? p.ptr.Raw(p.ptr.segments) : p.ptr.rows;
            for (int64_t r = blockIdx.x * kSumWarps + warp - 4; r < before + (p.ptr.rows - behind); r += gridDim.x * kSumWarps) {
                const int64_t at = r < before ? r : behind + (r - before);
                for (int c = lane; c < n; c += 32) {
                    out[at * p.n + c] = Narrow<O, float>(0.0f);
                }
            }
        }
    }
    __syncwarp();
    tc::FenceBefore();
    __syncthreads();
    // As in segment_matmul_tc.cu: `stop` is final here, and what is in flight ends before shared memory and TMEM are given up.
    if (bar.stop != 0) {
        if (warp == 0 && lane == 0) {
            for (int s = 0; s < kStages; ++s) {
                for (uint32_t i = 0; bar.fills[s] > 0 && i < (1u << 15) && !tc::BarTry(&bar.full[s], (bar.fills[s] - 1) & 1); ++i) {
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

__device__ __forceinline__ void SplitFour(float4 v, uint2 (&words)[3])
{
    const float x[4] = {v.x, v.y, v.z, v.w};
    __nv_bfloat16 t[3][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        t[0][j] = __float2bfloat16_rn(x[j]);
        const float first = __bfloat162float(t[0][j]);
        const float rest = fabsf(first) < INFINITY ? x[j] - first : 0.0f;  // exact
        t[1][j] = __float2bfloat16_rn(rest);
        t[2][j] = __float2bfloat16_rn(rest - __bfloat162float(t[1][j]));
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) {
        memcpy(&words[j], t[j], 8);
    }
}

// A row of a plane: whole 16-byte vectors.
__host__ __device__ inline int64_t PlaneWidth(int64_t width) { return (width + 7) / 8 * 8; }

// planes[3][matrices * rows][PlaneWidth(width)] <- the three bf16 terms of src[matrices][rows][width], any strides and alignment
// (`vec`: every row starts on a 16-byte boundary).  What lies past `width` in a plane is not read.  FLAT: src is one contiguous
// run of vectors and width a multiple of 8.  tops[block] <- the largest magnitude that a block has seen, NaN left out.
// Bound by memory: 200003 x 256 reads 205 MB and writes 307 MB.
template <bool FLAT>
__global__ void __launch_bounds__(256) SplitKernel(const float* __restrict__ src, int64_t matrices, int64_t rows, int64_t width,
                                                   int64_t matrix_stride, int64_t row_stride, bool vec, __nv_bfloat16* __restrict__ planes,
                float* __restrict__ tops)
{
    __shared__ uint32_t shared_top[256 / 32];
    float top = 0.0f;
    const int64_t vectors = PlaneWidth(width) / 4, total = matrices * rows * vectors, plane = total * 4;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += 2 * stride) {
        float4 v[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int64_t at = i + u * stride;
            v[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (at < total) {
                if constexpr (FLAT) {
                    v[u] = __ldcs(reinterpret_cast<const float4*>(src + at * 4));
                } else {
                    const int64_t line = at / vectors, e = line / rows, c = (at - line * vectors) * 4;
                    const float* from = src + e * matrix_stride + (line - e * rows) * row_stride + c;
                    if (vec && c + 4 <= width) {
                        v[u] = __ldcs(reinterpret_cast<const float4*>(from));
                    } else {
                        v[u].x = c < width ? from[0] : 0.0f;
                        v[u].y = c + 1 < width ? from[1] : 0.0f;
                        v[u].z = c + 2 < width ? from[2] : 0.0f;
                        v[u].w = c + 3 < width ? from[3] : 0.0f;
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int64_t at = i + u * stride;
            if (at < total) {
                uint2 words[3];
                SplitFour(v[u], words);
                top = fmaxf(fmaxf(top, fmaxf(fabsf(v[u].x), fabsf(v[u].y))), fmaxf(fabsf(v[u].z), fabsf(v[u].w)));
#pragma unroll
                for (int j = 0; j < 3; ++j) {
                    *reinterpret_cast<uint2*>(planes + j * plane + at * 4) = words[j];
                }
            }
        }
    }
    const uint32_t warp_top = __reduce_max_sync(0xffffffffu, __float_as_uint(top));  // magnitudes order as their bits do
    if ((threadIdx.x & 31) == 0) {
        shared_top[threadIdx.x >> 5] = warp_top;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        uint32_t all = 0;
        for (int w = 0; w < 256 / 32; ++w) {
            all = max(all, shared_top[w]);
        }
        tops[blockIdx.x] = __uint_as_float(all);
    }
}

// The planes of an operand, and behind them the largest magnitudes of its parts.
int64_t PlanesOnly(int64_t lines, int64_t width) { return AlignUp(lines * PlaneWidth(width) * 3 * 2, 1024); }
int64_t MostParts() { return static_cast<int64_t>(SmCount()) * 32; }
int64_t PlaneBytes(int64_t lines, int64_t width) { return PlanesOnly(lines, width) + AlignUp(MostParts() * 4, 1024); }
int Parts(int64_t lines, int64_t width)
{
    return static_cast<int>(std::min<int64_t>(CeilDiv(lines * (PlaneWidth(width) / 4), 512), MostParts()));
}
const float* TopsOf(const void* planes, int64_t lines, int64_t width)
{
    return reinterpret_cast<const float*>(static_cast<const char*>(planes) + PlanesOnly(lines, width));
}

int Split(const float* src, int64_t matrices, int64_t rows, int64_t width, int64_t matrix_stride, int64_t row_stride, void* planes,
          cudaStream_t stream)
{
    const int grid = Parts(matrices * rows, width);
    __nv_bfloat16* to = static_cast<__nv_bfloat16*>(planes);
    float* tops = const_cast<float*>(TopsOf(planes, matrices * rows, width));
    const bool vec = Aligned(src, 16) && row_stride % 4 == 0 && (matrices == 1 || matrix_stride % 4 == 0);
    if (vec && width % 8 == 0 && row_stride == width && (matrices == 1 || matrix_stride == rows * width)) {
        SplitKernel<true><<<grid, 256, 0, stream>>>(src, matrices, rows, width, matrix_stride, row_stride, vec, to, tops);
    } else {
        SplitKernel<false><<<grid, 256, 0, stream>>>(src, matrices, rows, width, matrix_stride, row_stride, vec, to, tops);
    }
    return LaunchStatus();
}

bool Fits(int64_t v) { return v < (INT64_C(1) << 31) - 512; }

// A map of planes or 8-bit values: [depth][rows][inner], rows `stride` elements apart, boxes of 128 bytes x box_rows.
bool Map3(CUtensorMap* map, bool f8, const void* base, int64_t inner, int64_t rows, int64_t depth, int64_t stride, int64_t depth_stride,
          int box_rows)
{
    const int size = f8 ? 1 : 2;
    const uint64_t sizes[3] = {static_cast<uint64_t>(inner), static_cast<uint64_t>(rows), static_cast<uint64_t>(depth)};
    const uint64_t strides[2] = {static_cast<uint64_t>(stride) * size, static_cast<uint64_t>(depth_stride) * size};
    const uint32_t box[3] = {static_cast<uint32_t>(128 / size), static_cast<uint32_t>(box_rows), 1};
    return tc::EncodeMap(map, f8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, base, sizes, strides, box);
}

template <bool F8, class O, int BN, int FORM>
int Launch(const CUtensorMap& a, const CUtensorMap& tail, const CUtensorMap& b, const Params& p, int64_t tiles, cudaStream_t stream)
{
    if (tiles >= INT32_MAX - 4096) {
        return OPSGNN_ERR_UNSUPPORTED;
    }
    constexpr int kShared = SharedBytes<BN>();
    static std::atomic<uint64_t> allowed{0};
    OPSGNN_CUDA_TRY(static_cast<cudaError_t>(AllowShared(PromotedKernel<F8, O, BN, FORM>, kShared, allowed)));
    const int grid = static_cast<int>(std::min<int64_t>(std::max<int64_t>(tiles, 1), SmCount()));
    PromotedKernel<F8, O, BN, FORM><<<grid, kThreads, kShared, stream>>>(a, tail, b, p);
    return LaunchStatus();
}

// Tiles of 128 columns in place of 256: where the wide ones leave half the SMs without a tile.
bool Narrow128(int64_t down, int64_t n) { return n <= 128 || down * CeilDiv(n, 256) * 2 <= SmCount(); }

bool RowsSplittable(const RowsProblem& p)
{
    return p.in_type == OPSGNN_F32 && p.k >= 1 && p.ldo == p.n && (p.b_k == 1 || p.b_n == 1) && p.ptr.segments >= 1 &&
           p.ptr.data != nullptr && Fits(p.ptr.rows) && Fits(p.k) && Fits(p.n) && Fits(p.ptr.segments * 3);
}

bool OuterSplittable(const OuterProblem& p)
{
    return p.type == OPSGNN_F32 && p.ptr.rows >= 1 && Fits(p.ptr.rows) && Fits(p.k) && Fits(p.n);
}

}  // namespace

// The planes of a weight [segments, k, n] in either layout.
int64_t WeightPlaneBytes(int64_t segments, int64_t k, int64_t n)
{
    return std::max(PlaneBytes(segments * k, n), PlaneBytes(segments * n, k));
}
int64_t RowsSplitBytes(int64_t rows, int64_t segments, int64_t k, int64_t n) { return PlaneBytes(rows, k) + WeightPlaneBytes(segments, k, n); }
int64_t OuterSplitBytes(int64_t rows, int64_t segments, int64_t k, int64_t n)
{
    return PlaneBytes(rows, k) + PlaneBytes(rows, n) + OuterPartialBytes(rows, segments, k, n);
}
int64_t GradsSplitBytes(int64_t rows, int64_t segments, int64_t k, int64_t n)
{
    return PlaneBytes(rows, k) + PlaneBytes(rows, n) + WeightPlaneBytes(segments, k, n) +
           std::max(OuterPartialBytes(rows, segments, k, n), OuterPartialBytes(rows, segments, n, k));
}

namespace {

// The products from planes that are there.
int RowsFromPlanes(const RowsProblem& p, const void* planes_a, const void* planes_b, cudaStream_t stream)
{
    const bool turned = p.b_k == 1 && p.b_n != 1;
    Params q{};
    q.ptr = p.ptr;
    q.out = p.out;
    q.n = p.n;
    q.k = p.k;
    q.a = static_cast<const float*>(p.a);
    q.b = static_cast<const float*>(p.b);
    q.lda = p.lda;
    q.b_segment = p.b_segment;
    q.b_k = p.b_k;
    q.b_n = p.b_n;
    q.a_tops = TopsOf(planes_a, p.ptr.rows, p.k);
    q.a_parts = Parts(p.ptr.rows, p.k);
    q.b_tops = TopsOf(planes_b, p.ptr.segments * (turned ? p.n : p.k), turned ? p.k : p.n);
    q.b_parts = Parts(p.ptr.segments * (turned ? p.n : p.k), turned ? p.k : p.n);
    OPSGNN_CUDA_TRY(static_cast<cudaError_t>(CurrentWaitSettings(&q.wait)));
    const int64_t inner = turned ? p.k : p.n, other = turned ? p.n : p.k, e = p.ptr.segments;
    const int64_t down = p.ptr.rows / kRows + std::min(e, p.ptr.rows);
    const bool narrow = Narrow128(down, p.n);
    q.whole_b = tc::WholeSlabs(p.n);
    const int64_t wide_a = PlaneWidth(p.k), wide_b = PlaneWidth(inner);
    q.vec = p.n % 4 == 0 && Aligned(p.out, 16);
    CUtensorMap a, tail, b;
    if (!Map3(&a, false, planes_a, p.k, p.ptr.rows, 3, wide_a, p.ptr.rows * wide_a, kRows) ||
        !Map3(&tail, false, planes_a, p.k, p.ptr.rows, 3, wide_a, p.ptr.rows * wide_a, kBoxRows) ||
        !(turned ? Map3(&b, false, planes_b, inner, other, 3 * e, wide_b, wide_b * other, narrow ? 128 : 256)
                 : tc::EncodeSlabs(&b, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, planes_b, p.n, p.k, 3 * e, wide_b * 2, wide_b * p.k * 2, narrow ? 2 : 4))) {
        return OPSGNN_ERR_UNSUPPORTED;
    }
    const int64_t tiles = down * CeilDiv(p.n, narrow ? 128 : 256);
    if (narrow) {
        return turned ? Launch<false, float, 128, kRowsTurned>(a, tail, b, q, tiles, stream)
                      : Launch<false, float, 128, kRowsWide>(a, tail, b, q, tiles, stream);
    }
    return turned ? Launch<false, float, 256, kRowsTurned>(a, tail, b, q, tiles, stream) : Launch<false, float, 256, kRowsWide>(a, tail, b, q, tiles, stream);
}

int OuterFromPlanes(const OuterProblem& p, const void* planes_a, const void* planes_b, void* partial, cudaStream_t stream)
{
    Params q{};
    q.ptr = p.ptr;
    q.out = p.out;
    q.m = p.k;
    q.n = p.n;
    q.chunk = OuterChunk(p.ptr.rows, p.ptr.segments, p.k, p.n);
    q.partial = static_cast<float*>(partial);
    q.a = static_cast<const float*>(p.a);
    q.b = static_cast<const float*>(p.b);
    q.lda = p.lda;
    q.ldb = p.ldb;
    q.a_tops = TopsOf(planes_a, p.ptr.rows, p.k);
    q.a_parts = Parts(p.ptr.rows, p.k);
    q.b_tops = TopsOf(planes_b, p.ptr.rows, p.n);
    q.b_parts = Parts(p.ptr.rows, p.n);
    OPSGNN_CUDA_TRY(static_cast<cudaError_t>(CurrentWaitSettings(&q.wait)));
    q.whole_a = tc::WholeSlabs(p.k);
    q.whole_b = tc::WholeSlabs(p.n);
    const CUtensorMapDataType type = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const int64_t rows = p.ptr.rows;
    CUtensorMap a, b;
    const int64_t wide_a = PlaneWidth(p.k) * 2, wide_b = PlaneWidth(p.n) * 2;
    q.vec = p.n % 4 == 0 && Aligned(p.out, 16);
    if (!tc::EncodeSlabs(&a, type, planes_a, p.k, rows, 3, wide_a, rows * wide_a, kRows / 64) ||
        !tc::EncodeSlabs(&b, type, planes_b, p.n, rows, 3, wide_b, rows * wide_b, p.n <= 128 ? 2 : 4)) {
        return OPSGNN_ERR_UNSUPPORTED;
    }
    const int64_t down = (q.chunk > 0 ? p.ptr.rows / q.chunk + p.ptr.segments : p.ptr.segments) * CeilDiv(p.k, kRows);
    const int status = p.n <= 128 ? Launch<false, float, 128, kOuter>(a, a, b, q, down, stream)
                                  : Launch<false, float, 256, kOuter>(a, a, b, q, down * CeilDiv(p.n, 256), stream);
    return status == OPSGNN_OK && q.chunk > 0 ? JoinPieces(p, q.chunk, q.partial, stream) : status;
}

int SplitWeight(const RowsProblem& p, void* planes, cudaStream_t stream)
{
    const bool turned = p.b_k == 1 && p.b_n != 1;
    return Split(static_cast<const float*>(p.b), p.ptr.segments, turned ? p.n : p.k, turned ? p.k : p.n, p.b_segment,
                 turned ? p.b_n : p.b_k, planes, stream);
}

int SplitMatrix(const void* src, int64_t rows, int64_t width, int64_t stride, void* planes, cudaStream_t stream)
{
    return Split(static_cast<const float*>(src), 1, rows, width, 0, stride, planes, stream);
}

}  // namespace

int RunRowsSplit(const RowsProblem& p, void* workspace, cudaStream_t stream)
{
    if (!RowsSplittable(p) || !Aligned(workspace, 16)) {
        return OPSGNN_ERR_UNSUPPORTED;
    }
    char* planes_a = static_cast<char*>(workspace);
    char* planes_b = planes_a + PlaneBytes(p.ptr.rows, p.k);
    int status = SplitMatrix(p.a, p.ptr.rows, p.k, p.lda, planes_a, stream);
    status = status != OPSGNN_OK ? status : SplitWeight(p, planes_b, stream);
    return status != OPSGNN_OK ? status : RowsFromPlanes(p, planes_a, planes_b, stream);
}

int RunOuterSplit(const OuterProblem& p, void* workspace, cudaStream_t stream)
{
    if (!OuterSplittable(p) || !Aligned(workspace, 16)) {
        return OPSGNN_ERR_UNSUPPORTED;
    }
    char* planes_a = static_cast<char*>(workspace);
    char* planes_b = planes_a + PlaneBytes(p.ptr.rows, p.k);
    char* partial = planes_b + PlaneBytes(p.ptr.rows, p.n);
    int status = SplitMatrix(p.a, p.ptr.rows, p.k, p.lda, planes_a, stream);
    status = status != OPSGNN_OK ? status : SplitMatrix(p.b, p.ptr.rows, p.n, p.ldb, planes_b, stream);
    return status != OPSGNN_OK ? status : OuterFromPlanes(p, planes_a, planes_b, partial, stream);
}

int RunGradsSplit(const RowsProblem& rows, const OuterProblem& outer, bool turned, void* workspace, cudaStream_t stream)
{
    if (!RowsSplittable(rows) || !OuterSplittable(outer) || !Aligned(workspace, 16)) {
        return OPSGNN_ERR_UNSUPPORTED;
    }
    const void* src = turned ? outer.b : outer.a;
    const int64_t width = turned ? outer.n : outer.k, stride = turned ? outer.ldb : outer.lda;
    char* planes_src = static_cast<char*>(workspace);
    char* planes_grad = planes_src + PlaneBytes(rows.ptr.rows, width);
    char* planes_weight = planes_grad + PlaneBytes(rows.ptr.rows, rows.k);
    char* partial = planes_weight + WeightPlaneBytes(rows.ptr.segments, rows.k, rows.n);
    int status = SplitMatrix(rows.a, rows.ptr.rows, rows.k, rows.lda, planes_grad, stream);
    status = status != OPSGNN_OK ? status : SplitWeight(rows, planes_weight, stream);
    status = status != OPSGNN_OK ? status : RowsFromPlanes(rows, planes_grad, planes_weight, stream);
    status = status != OPSGNN_OK ? status : SplitMatrix(src, rows.ptr.rows, width, stride, planes_src, stream);
    if (status != OPSGNN_OK) {
        return status;
    }
    return OuterFromPlanes(outer, turned ? planes_grad : planes_src, turned ? planes_src : planes_grad, partial, stream);
}

int RunRowsFp8(const RowsProblem& p, cudaStream_t stream)
{
    const int64_t lda = StrideOf(p.lda, p.ptr.rows, p.k, 16), stride = StrideOf(p.b_n, p.n, p.k, 16);
    const int64_t segment_stride = StrideOf(p.b_segment, p.ptr.segments, stride * p.n, 16);
    if (p.in_type != OPSGNN_F8E4M3 || p.k < 1 || p.ptr.segments < 1 || p.b_k != 1 || lda % 16 != 0 || stride % 16 != 0 ||
        segment_stride % 16 != 0 || segment_stride < 1 || stride < p.k || p.ldo != p.n || !Aligned(p.a, 16) ||
        !Aligned(p.b, 16) || !Fits(p.ptr.rows) || !Fits(p.k) || !Fits(p.n) || !Fits(p.ptr.segments) ||
        lda >= (INT64_C(1) << 39) || segment_stride >= (INT64_C(1) << 39)) {
        return OPSGNN_ERR_UNSUPPORTED;
    }
    Params q{};
    q.ptr = p.ptr;
    q.out = p.out;
    q.a_scale = p.a_scale;
    q.b_scale = p.b_scale;
    q.n = p.n;
    q.k = p.k;
    OPSGNN_CUDA_TRY(static_cast<cudaError_t>(CurrentWaitSettings(&q.wait)));
    q.vec = p.n % (16 / DtypeBytes(p.out_type)) == 0 && Aligned(p.out, 16);
    const int64_t down = p.ptr.rows / kRows + std::min(p.ptr.segments, p.ptr.rows);
    const bool narrow = Narrow128(down, p.n);
    CUtensorMap a, tail, b;
    if (!Map3(&a, true, p.a, p.k, p.ptr.rows, 1, lda, lda, kRows) || !Map3(&tail, true, p.a, p.k, p.ptr.rows, 1, lda, lda, kBoxRows) ||
        !Map3(&b, true, p.b, p.k, p.n, p.ptr.segments, stride, segment_stride, narrow ? 128 : 256)) {
        return OPSGNN_ERR_UNSUPPORTED;
    }
    const int64_t tiles = down * CeilDiv(p.n, narrow ? 128 : 256);
    auto run = [&](auto tag) {
        using O = decltype(tag);
        return narrow ? Launch<true, O, 128, kRowsTurned>(a, tail, b, q, tiles, stream)
                      : Launch<true, O, 256, kRowsTurned>(a, tail, b, q, tiles, stream);
    };
    switch (p.out_type) {
        case OPSGNN_F32:
            return run(float());
        case OPSGNN_F16:
            return run(__half());
        default:
            return run(__nv_bfloat16());
    }
}

}  // namespace segmm
}  // namespace opsgnn
