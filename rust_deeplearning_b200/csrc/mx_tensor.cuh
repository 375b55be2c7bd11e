// What the two tensor-core kernels for 4-bit weights share: barriers, TMA, the block-scaled product, and a weight as they take it.
//
// tcgen05.mma.kind::mxf8f6f4.block_scale multiplies 32 columns at a time, applies a power of two a row and group on both sides and
// sums in float in tensor memory.  TMA spreads 4-bit codes to a byte each on their way to shared memory (the 16U4_ALIGN16B type: 16 codes
// in 8 of every 16 bytes, the form the instruction reads 4-bit operands in), so that no thread unpacks anything.
//
// Scales go to tensor memory by tcgen05.cp (32 lanes of 16 bytes), issued by the thread that issues the products and in
// order with them.  Word 4 l + c of 128 lands in lane l, column c, where the product looks for the scales of operand row 32 c + l.
// A weight's scales lie in memory in that order.
#pragma once

#include <cuda.h>

#include "common.cuh"
#include "microscaling.cuh"

// Tensor memory.  A block whose columns are taken waits in tcgen05.alloc until a block that has them ends, for as long as that takes.  Blocks of
// a cluster wait for one another, so two clusters on the same multiprocessors, each with the columns the other one's block waits for,
// would never end.  So: what blocks of clusters can be on one multiprocessor together never wants more than its 512 columns.  Few rows: 128
// columns, at most three blocks by their threads (16 float32 rows: 256, one block by its registers).  Up to 128 rows, shared by a
// cluster: 256 columns, and shared memory of three stages, so that there is room for two of them, or for one beside blocks of few rows, of which
// registers allow one.  Pairs of many rows: 512, and no room in shared memory beside them.  Blocks without a cluster may take what
// they want: they wait for nobody once they have it.

// A 4-bit weight on the host's side: made once, when the weight is laid out.
struct alignas(64) Mx4Matrix {
    CUtensorMap codes_map;                       // [tile x block x row][128 codes], a box is a tile
    CUtensorMap scales_map;                      // [tile x block][128 words], a box is a tile's
    const uint8_t* codes; const uint8_t* scales;
    int rows, columns, gated;                    // as packed (gated: rows / 2 outputs)
    int blocks, tiles;                           // of 128 columns, of 128 rows
};

// Blocks that share a tile, each with its part of the columns: as many as keep every tile on the device at once (in clusters of up to 8),
// each with two blocks of columns or more.
int mx_split(int tiles, int blocks, int sms);
bool mx_some_rows_pay(const Mx4Matrix& w, int m);

namespace {

constexpr int MX_TILE_BYTES = MX_ROWS * MX_BLOCK, MX_TILE_TX = MX_TILE_BYTES / 2;      // in shared memory; read (what a 4-bit transfer counts)
constexpr int MX_SCALE_BYTES = MX_ROWS * 4;

__device__ __forceinline__ uint32_t mx_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mx_bar_init(uint32_t bar, int count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void mx_bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mx_bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool mx_bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// false where the phase did not complete in time, or where another warp of the block has given up
__device__ __forceinline__ bool mx_bar_wait(uint32_t bar, uint32_t parity, long long limit, volatile int* gave_up) {
    if (mx_bar_try(bar, parity)) return true;
    const long long t0 = clock64();
    while (!mx_bar_try(bar, parity)) {
        if (*gave_up) return false;
        if (clock64() - t0 > limit) { *gave_up = 1; return false; }
    }
    return true;
}
// One thread of a warp that has come here as a whole.  What tcgen05 and TMA instructions take has to be uniform over the warp: behind this
// choice the compiler knows that one thread issues them; behind `lane == 0` it does not and goes through the lanes, which cost 90
// clock cycles an instruction (a block of 128 columns, four products and two copies of scales: 538 cycles, and 185 so).
__device__ __forceinline__ bool mx_elect() {
    uint32_t one;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(one));
    return one != 0;
}
// the wait of a whole warp; the same answer in all of its lanes
__device__ __forceinline__ bool mx_warp_wait(uint32_t bar, uint32_t parity, long long limit, volatile int* gave_up) {
    return __all_sync(0xffffffffu, mx_bar_wait(bar, parity, limit, gave_up));
}
// Two barriers at once: a wait takes 110 to 190 cycles to answer even if it is long over, as long as the products of a block, and these
// two answer together.
__device__ __forceinline__ bool mx_bar_wait_both(uint32_t bar0, uint32_t parity0, uint32_t bar1, uint32_t parity1, long long limit, volatile int* gave_up) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p, q;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\nmbarrier.test_wait.parity.shared::cta.b64 q, [%3], %4;\n"
                 "and.pred p, p, q;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(bar0), "r"(parity0), "r"(bar1), "r"(parity1) : "memory");
    return ok != 0 || (mx_bar_wait(bar0, parity0, limit, gave_up) && mx_bar_wait(bar1, parity1, limit, gave_up));
}
__device__ __forceinline__ void mx_tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar) : "memory");
}
// K-major operand tile, rows of 128 bytes, 128-byte swizzle: groups of 8 rows are 1024 bytes apart
__device__ __forceinline__ uint64_t mx_operand_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// scales as tcgen05.cp reads them: no swizzle, 8 lanes of 16 bytes are 128 bytes, the next eight right behind
__device__ __forceinline__ uint64_t mx_scale_desc(uint32_t addr) { return (uint64_t)((addr & 0x3FFFF) >> 4) | (8ull << 32) | (1ull << 46); }
constexpr uint32_t MX_E4M3 = 0, MX_E2M1 = 5;
// instruction descriptor of the block-scaled kinds: formats of A and B at bits 7 and 10, N >> 3 at bit 17, scales are powers of two (bit 23),
// M >> 7 at bit 27; which byte of the scale words counts: of B at bit 4, of A at bit 29
__host__ __device__ constexpr uint32_t mx_idesc(uint32_t a, uint32_t b, int m, int n, int byte) {
    return ((uint32_t)byte << 4) | (a << 7) | (b << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 7) << 27) | ((uint32_t)byte << 29);
}
__device__ __forceinline__ void mx_tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void mx_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void mx_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

typedef CUresult (*MxEncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

struct MxMapShape {
    CUtensorMapDataType type; int rank;
    cuuint64_t dims[3], strides[2];              // elements; bytes
    cuuint32_t box[3];
    CUtensorMapSwizzle swizzle;
};

// the driver's encoder is looked up at run time, so that the library loads where there is no driver
inline int mx_make_map(CUtensorMap* map, const void* p, const MxMapShape& s, const char* what) {
    static MxEncodeTiled encode = nullptr;
    if (!encode) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        RDL_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found), "looking up cuTensorMapEncodeTiled");
        RDL_REQUIRE(found == cudaDriverEntryPointSuccess && fn, "this driver has no cuTensorMapEncodeTiled");
        encode = (MxEncodeTiled)fn;
    }
    const cuuint32_t one[3] = {1, 1, 1};
    const CUresult r = encode(map, s.type, (cuuint32_t)s.rank, const_cast<void*>(p), s.dims, s.strides, s.box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              s.swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    RDL_REQUIRE(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with driver error %d for %s", (int)r, what);
    return 0;
}

// The maps of 8-bit rows: values as [4][rows / 4][columns] in boxes of 4 x 32 rows, scales as [blocks][rows] words in boxes of 128.
struct MxRowsMaps { CUtensorMap values, scales; };
inline int mx_rows_maps(MxRowsMaps* maps, const void* x, const void* row_scales, long long blocks, long long rows4) {
    const cuuint64_t cols = (cuuint64_t)blocks * MX_BLOCK, rows = (cuuint64_t)rows4;
    if (int e = mx_make_map(&maps->values, x, {CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, {cols, rows / 4, 4}, {cols * 4, cols}, {MX_BLOCK, 32, 4}, CU_TENSOR_MAP_SWIZZLE_128B}, "8-bit rows")) return e;
    return mx_make_map(&maps->scales, row_scales, {CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, {rows, (cuuint64_t)blocks}, {rows * 4}, {MX_ROWS, 1}, CU_TENSOR_MAP_SWIZZLE_NONE},
                       "the scales of 8-bit rows");
}

}  // namespace
