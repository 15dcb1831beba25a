// Thin wrappers of the sm_100a instructions the segment products are built from: mbarriers, TMA tile loads, TMEM and
// tcgen05.mma, and the descriptors these take.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace opsgnn {

namespace tc {

// ---- mbarriers -------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t Shared(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void BarInit(uint64_t* bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(Shared(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void BarInitFence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void BarArrive(uint64_t* bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(Shared(bar)) : "memory");
}
__device__ __forceinline__ void BarExpect(uint64_t* bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(Shared(bar)), "r"(bytes) : "memory");
}
// One poll; it may suspend the thread for a while and returns as soon as the phase completes.
__device__ __forceinline__ bool BarTry(uint64_t* bar, uint32_t parity)
{
    uint32_t done;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(done)
        : "r"(Shared(bar)), "r"(parity), "r"(100000u)
        : "memory");
    return done != 0;
}

// A look that does not wait.
__device__ __forceinline__ bool BarTest(uint64_t* bar, uint32_t parity)
{
    uint32_t done;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(done)
        : "r"(Shared(bar)), "r"(parity)
        : "memory");
    return done != 0;
}

// A bounded wait.  One that runs out marks the launch as stopped (every other wait of the block then ends too) and reports
// to the host; the block leaves its remaining tiles unwritten, waits for what it has in flight and returns.
struct Waiter {
    volatile uint32_t* stop;  // shared
    WaitSettings settings;

    __device__ __forceinline__ bool operator()(uint64_t* bar, uint32_t parity) const
    {
        for (uint32_t i = 0; i < settings.polls; ++i) {
            if (BarTry(bar, parity)) {
                return true;
            }
            if (*stop != 0) {
                return false;
            }
        }
        *stop = 1;
        if (settings.sink != nullptr) {
            *reinterpret_cast<volatile unsigned long long*>(settings.sink) = 1ULL;
        }
        return false;
    }
    // For a whole warp: the same answer in every lane.
    __device__ __forceinline__ bool Warp(uint64_t* bar, uint32_t parity) const
    {
        return __all_sync(0xffffffffu, (*this)(bar, parity));
    }
};

// ---- TMA -------------------------------------------------------------------------------------------------------------------

// Tile loads into the own block's shared memory.  x counts elements and is a multiple of 16 bytes at every call site.
__device__ __forceinline__ void LoadTo(const CUtensorMap& map, uint32_t bar, uint32_t to, int x, int y)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(to),
                 "l"(&map), "r"(bar), "r"(x), "r"(y)
                 : "memory");
}
__device__ __forceinline__ void LoadTo(const CUtensorMap& map, uint32_t bar, uint32_t to, int x, int y, int z)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
                     to),
                 "l"(&map), "r"(bar), "r"(x), "r"(y), "r"(z)
                 : "memory");
}
__device__ __forceinline__ void LoadTo(const CUtensorMap& map, uint32_t bar, uint32_t to, int x, int y, int z, int w)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(to),
        "l"(&map), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}
// Writes to shared memory by this thread become visible to tcgen05.mma and TMA.
__device__ __forceinline__ void FenceAsync() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- TMEM and tcgen05 ------------------------------------------------------------------------------------------------------

constexpr uint32_t kTmemColumns = 512;

// By one whole warp; the base address lands in *to.
__device__ __forceinline__ void TmemAlloc(uint32_t* to)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(Shared(to)), "r"(kTmemColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void TmemFree(uint32_t base)
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(kTmemColumns) : "memory");
}
__device__ __forceinline__ void FenceBefore() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void FenceAfter() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// The barrier gets one arrival when all tcgen05.mma this thread issued so far are done.
__device__ __forceinline__ void Commit(uint64_t* bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(Shared(bar)) : "memory");
}

// D[tmem] (+)= A[smem] * B[smem]; 16-bit operands, K = 16 per instruction.
__device__ __forceinline__ void MmaF16(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add)
{
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(shape), "r"(static_cast<uint32_t>(add))
        : "memory");
}
// The same for 8-bit operands, K = 32 per instruction.
__device__ __forceinline__ void MmaF8(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add)
{
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(shape), "r"(static_cast<uint32_t>(add))
        : "memory");
}

// 32 columns of the warp's 32 TMEM lanes; complete after TmemWait.
__device__ __forceinline__ void TmemLoad32(uint32_t at, uint32_t (&r)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
        "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
}
__device__ __forceinline__ void TmemWait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Shared-memory operand in 128-byte swizzled rows (the layout a TMA load with SWIZZLE_128B writes), 1024-byte aligned.
//   K-major (the reduced index runs along the 128-byte row): groups of 8 rows are 1024 bytes apart (`step`); the other
//   stride has no meaning.  K advances inside the row: + 32 bytes per instruction.
//   MN-major (the kept index runs along the row): 8 values of k make 1024 bytes (`step`); the next 128 bytes' worth of the
//   kept index start `lead` bytes further.  K advances by whole groups: + 2048 bytes per 16-bit instruction.
__device__ __forceinline__ uint64_t Operand(uint32_t address, uint32_t lead, uint32_t step)
{
    return static_cast<uint64_t>((address & 0x3ffffu) >> 4) | (static_cast<uint64_t>(lead >> 4) << 16) |
           (static_cast<uint64_t>(step >> 4) << 32) | (1ULL << 46) | (2ULL << 61);
}

// Instruction descriptor: fp32 accumulators; type 0 / 1 = fp16 / bf16 (16-bit kind), 0 = e4m3 (8-bit kind).
constexpr uint32_t Shape(int m, int n, int type, bool a_mn, bool b_mn)
{
    return (1u << 4) | (static_cast<uint32_t>(type) << 7) | (static_cast<uint32_t>(type) << 10) | (a_mn ? 1u << 15 : 0u) |
           (b_mn ? 1u << 16 : 0u) | (static_cast<uint32_t>(n / 8) << 17) | (static_cast<uint32_t>(m / 16) << 24);
}

// ---- results ---------------------------------------------------------------------------------------------------------------

// A warp writes 32 rows of BYTES bytes from its staging area, whose 16-byte pieces are permuted by the row's number against
// bank conflicts (Staged gives a piece's place), to `to` + row * stride; rows and columns past the limits are left out.  VEC:
// rows of the result start on 16-byte boundaries, so neighbouring lanes write neighbouring 16-byte pieces; else single values.
template <int BYTES> __device__ __forceinline__ int Staged(int row, int piece)
{
    constexpr int PIECES = BYTES / 16;
    return row * BYTES + ((piece ^ ((PIECES == 8 ? row : row >> 1) & (PIECES - 1))) << 4);
}
template <int BYTES, class O>
__device__ __forceinline__ void StoreStaged(const unsigned char* staging, O* to, int64_t stride, int rows, int columns, bool vec)
{
    constexpr int PIECES = BYTES / 16, PER = 16 / sizeof(O), LINE = BYTES / sizeof(O);
    const int lane = threadIdx.x & 31;
    if (vec) {
        const int piece = lane % PIECES;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int r = i * (32 / PIECES) + lane / PIECES;
            const uint4 value = *reinterpret_cast<const uint4*>(staging + Staged<BYTES>(r, piece));
            if (r < rows && piece * PER < columns) {
                *reinterpret_cast<uint4*>(to + r * stride + piece * PER) = value;
            }
        }
    } else {
#pragma unroll 1
        for (int r = 0; r < 32 && r < rows; ++r) {
#pragma unroll 1
            for (int c = lane; c < LINE; c += 32) {
                if (c < columns) {
                    to[r * stride + c] = *reinterpret_cast<const O*>(staging + Staged<BYTES>(r, c / PER) + c % PER * sizeof(O));
                }
            }
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------

// An MN-major operand is a row of slabs, 64 values of the kept index by 64 of the reduced one.  Where the kept extent is a
// multiple of 64 one load takes `slabs` of them (dimensions 64, rows, slab, depth); else each slab is a load of its own, with
// the map's bounds filling zeros past the extent (dimensions extent, rows, 1, depth).  Loads are issued by one thread and
// their number matters: four 32-row loads and four slabs a stage in place of one each cost a quarter of the rate.
constexpr int kSlabBytes = 64 * 128;
__device__ __forceinline__ void LoadSlabs(const CUtensorMap& map, uint32_t bar, uint32_t to, int column, int row, int depth, int slabs,
                                          bool whole)
{
    if (whole) {
        LoadTo(map, bar, to, 0, row, column / 64, depth);
    } else {
        for (int i = 0; i < slabs; ++i) {
            LoadTo(map, bar, to + i * kSlabBytes, column + i * 64, row, 0, depth);
        }
    }
}
inline bool WholeSlabs(int64_t extent) { return extent % 64 == 0; }
bool EncodeSlabs(CUtensorMap* map, CUtensorMapDataType type, const void* base, int64_t extent, int64_t rows, int64_t depth,
                 int64_t row_bytes, int64_t depth_bytes, int slabs);

// A tile map of up to 4 dimensions with 128-byte swizzle; strides[i] (bytes, multiples of 16) belong to dimension i + 1.
// False where the driver refuses it.
bool EncodeMap(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base, const uint64_t* sizes, const uint64_t* strides,
               const uint32_t* box);

}  // namespace tc
}  // namespace opsgnn
