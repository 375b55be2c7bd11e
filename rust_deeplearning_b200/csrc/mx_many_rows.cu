// Many rows of 8 bits times a 4-bit weight matrix (microscaling.cuh) on the fifth-generation tensor cores:
//   out[m, n] = epilogue(sum_k x[m, k] w[n, k]),  x e4m3 and w e2m1, each with a power of two a group of 32 columns.
//
// The block-scaled tcgen05 product (mx_tensor.cuh) at twice the rate of bfloat16; TMA brings both operands in the form it reads.
//
// The rows' scales lie in memory row by row, and word 4 l + c of 128 reaches the place where the product looks for the scales of
// operand row 32 c + l.  So operand row 32 c + l has to be row 4 l + c of the tile.  The rows' tensor map does that: the matrix
// is described as [4][rows / 4][columns], and a box of 4 x 32 rows arrives in that order.  The epilogue undoes it: lane l of
// quarter c holds row 4 l + c.
//
// A tile is 128 CTAS x 256.  CTAS 2: a pair of blocks on two multiprocessors (cta_group::2) computes 256 x 256; each holds its half of the
// rows and one of the two weight tiles, and the products, issued by a thread of block 0, read both halves.  A multiprocessor
// then fetches 24 KB for 8.4 MFLOP, where a block on its own fetches 32 KB, more than L2 delivers to all of them at the
// tensor cores' rate (gate and up of the 2B shape, 2,048 rows: 64 us on its own).  CTAS 1: few rows, or few tiles.
//
// Persistent: warp 0 loads, warp 1 copies scales and issues the products, sixteen warps take the accumulator out of tensor memory
// at once, all of it into registers, so that the next tile's products can start, and then apply the epilogue and store.  The gated
// form's tile is 128 gate and 128 up rows of the same 128 outputs; its result may leave as 8-bit rows with scales: 32 outputs of a
// row lie in one thread, which is a group.
//
// Measured: gate and up of the 2B shape, 2,048 rows to 8 bits, 56.5 us, 3.1 PFLOP/s; 8,192 rows x 36,864 x 4,608 outputs 865 us, 3.2 PFLOP/s
// (1,020 to 1,050 us, 2.7 PFLOP/s, when such calls go on for seconds and the power limit lowers the clock).
// The tensor cores bound it: 530 cycles a block of columns, of which the products take 513, at the clock that the power limit leaves; between
// two tiles they wait 1,100 cycles, from their end until the accumulator is in registers.
//
// Every wait is bounded; a block that gives up sets `status` and every path ends in the common tear-down.
#include "activations.cuh"
#include "api.h"
#include "launch.cuh"
#include "mx_tensor.cuh"

namespace {

constexpr int BM = 128, BN = 256, BK = MX_BLOCK, EPI_WARPS = 16, THREADS = 64 + EPI_WARPS * 32;
constexpr int A_BYTES = BM * BK;
constexpr int EPI_STAGE_BYTES = 32 * 64;                  // 32 rows of 64 bytes: of one epilogue warp
// shared memory of a stage: rows | one or both weight tiles | the rows' scales | both weight tiles' scales
__host__ __device__ constexpr int stages(int ctas) { return ctas == 2 ? 5 : 3; }
__host__ __device__ constexpr int scales_at(int ctas) { return A_BYTES + (3 - ctas) * MX_TILE_BYTES; }
__host__ __device__ constexpr int stage_pitch(int ctas) { return (scales_at(ctas) + 3 * MX_SCALE_BYTES + 1023) / 1024 * 1024; }
__host__ __device__ constexpr int stage_tx(int ctas) { return A_BYTES + (3 - ctas) * MX_TILE_TX + 3 * MX_SCALE_BYTES; }
__host__ __device__ constexpr int smem_bytes(int ctas) { return stages(ctas) * stage_pitch(ctas) + EPI_WARPS * EPI_STAGE_BYTES + 1024; }
constexpr int SCALE_COLS = 16, SCALE_BUFS = 4;            // tensor memory: 4 + 8 columns of scales a buffer, behind the accumulator
constexpr int TMEM_COLS = 512;
constexpr int RASTER_GROUP = 8;                           // row tiles that share a weight tile and run together

struct ManyArgs {
    void* out; int out_kind;                              // RDL_F32, RDL_BF16, or RDL_MX8 with out_scales
    uint8_t* out_scales;
    int M, N, blocks;                                     // blocks of 128 columns
    int out_blocks, out_padded_rows;                      // RDL_MX8
    int activation; float act_param, softcap;
    long long wait_cycles; int test_extra_tx;
    int* status;
};

// loads into this block's shared memory; of a pair they report to a barrier in block 0
template <int CTAS>
__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if constexpr (CTAS == 1)
        mx_tma_2d(dst, map, x, y, bar);
    else
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar) : "memory");
}
template <int CTAS>
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if constexpr (CTAS == 1)
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                     ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(0), "r"(bar) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                     ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(0), "r"(bar) : "memory");
}
#define MX_CTA_GROUP(CTAS, ONE, TWO) do { if constexpr (CTAS == 1) { ONE; } else { TWO; } } while (0)
template <int CTAS>
__device__ __forceinline__ void mma_mx(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
    MX_CTA_GROUP(CTAS,
        asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\ntcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory"),
        asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\ntcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory"));
}
// of a pair: each block's scales into its own tensor memory
template <int CTAS>
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
    MX_CTA_GROUP(CTAS, asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory"),
                 asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory"));
}
// arrives at `bar` when the products so far are done; of a pair in both blocks
template <int CTAS>
__device__ __forceinline__ void commit(uint32_t bar) {
    MX_CTA_GROUP(CTAS, asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory"),
                 asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((unsigned short)3) : "memory"));
}
__device__ __forceinline__ uint32_t map_to_block(uint32_t addr, uint32_t rank) {      // the same place in the shared memory of block `rank`
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// Relaxed: what it orders, this warp's reads of tensor memory, has completed before (tcgen05.wait::ld), and no memory is handed over.  A
// release at cluster scope cost 1,750 cycles from the last read to the next product, and this 250.
__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) { asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory"); }
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory"); }
// 16 accumulator columns of the warp's lanes, as bits; there after mx_tmem_wait_ld
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr) : "memory");
}

// The 32 outputs [n, n + 32) of one row, in order: epilogue and store.
template <bool GATED>
__device__ __forceinline__ void finish(const ManyArgs& a, float (&y)[32], const float (&u)[32]) {
    if (GATED) {
        if (a.out_kind == RDL_F32) {
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = rdl_gated(y[i], u[i], a.activation, a.act_param);
        } else if (a.activation == RDL_ACT_GELU_TANH) {      // the choice is made once a piece
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = rdl_gated_near(y[i], u[i], RDL_ACT_GELU_TANH, 0.f);
        } else if (a.activation == RDL_ACT_SILU) {
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = rdl_gated_near(y[i], u[i], RDL_ACT_SILU, 0.f);
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = rdl_gated_near(y[i], u[i], RDL_ACT_SWISH_LIMIT, a.act_param);
        }
    } else if (a.activation >= 16) {
#pragma unroll
        for (int i = 0; i < 32; ++i) y[i] = rdl_unary(y[i], a.activation);
    }
    if (a.softcap > 0.f) {
#pragma unroll
        for (int i = 0; i < 32; ++i) y[i] = a.softcap * tanhf(y[i] / a.softcap);
    }
}

// one group of a row of 8-bit results; columns beyond N become zeros, groups beyond the padded width are not there
__device__ __forceinline__ void store_group(const ManyArgs& a, int m, int n, float (&y)[32]) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        if (n + i >= a.N) y[i] = 0.f;
        top = mx_larger(top, y[i]);
    }
    const uint32_t c = mx8_scale_code(top);
    const float inv = mx_inverse_scale(c);
    const int block = n / MX_BLOCK;
    if (block >= a.out_blocks) return;
    uint4* o = reinterpret_cast<uint4*>((uint8_t*)a.out + (long long)m * a.out_blocks * MX_BLOCK + n);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = mx_to_e4m3(y[h * 16 + i * 4] * inv, y[h * 16 + i * 4 + 1] * inv, y[h * 16 + i * 4 + 2] * inv, y[h * 16 + i * 4 + 3] * inv);
        o[h] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    a.out_scales[((long long)block * a.out_padded_rows + m) * 4 + n % MX_BLOCK / MX_GROUP] = (uint8_t)c;
}

template <bool GATED, int CTAS>
__global__ void __launch_bounds__(THREADS, 1) mx_many_rows_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_xs,
                                                                  const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_ws,
                                                                  const __grid_constant__ ManyArgs a) {
    constexpr int OUT_BN = GATED ? BN / 2 : BN, TILE_M = BM * CTAS;
    constexpr int STAGES = stages(CTAS), PITCH = stage_pitch(CTAS), SCALES = scales_at(CTAS);
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) unsigned long long full_bar[STAGES], empty_bar[STAGES], acc_full, acc_empty;
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up;
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;      // the compiler may know it uniform
    const int rank = CTAS == 1 ? 0 : (int)(blockIdx.x & 1), first_tile = blockIdx.x / CTAS, tile_step = gridDim.x / CTAS;
    const int tiles_m = (a.M + TILE_M - 1) / TILE_M, tiles_n = (a.N + OUT_BN - 1) / OUT_BN, n_tiles = tiles_m * tiles_n;
    auto tile_origin = [&](int tile, int& m0, int& n0) {          // m0: of this block's rows
        const int per_group = RASTER_GROUP * tiles_n;
        const int group = tile / per_group, in_group = tile - group * per_group;
        const int first_m = group * RASTER_GROUP;
        const int gm = tiles_m - first_m < RASTER_GROUP ? tiles_m - first_m : RASTER_GROUP;
        m0 = (first_m + in_group % gm) * TILE_M + rank * BM;
        n0 = (in_group / gm) * OUT_BN;
    };
    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int s = 0; s < STAGES; ++s) {
            mx_bar_init(mx_smem(&full_bar[s]), 1);
            mx_bar_init(mx_smem(&empty_bar[s]), 1);
        }
        mx_bar_init(mx_smem(&acc_full), 1);
        mx_bar_init(mx_smem(&acc_empty), EPI_WARPS * CTAS);       // of a pair: used in block 0
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        MX_CTA_GROUP(CTAS, asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(mx_smem(&tmem_slot)), "r"(TMEM_COLS) : "memory"),
                     asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(mx_smem(&tmem_slot)), "r"(TMEM_COLS) : "memory"));
        MX_CTA_GROUP(CTAS, asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory"),
                     asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory"));
    }
    mx_fence_before();
    __syncthreads();
    if (CTAS == 2) cluster_sync();       // both blocks have their barriers and their tensor memory before anything crosses
    mx_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
    volatile int* gave_up_v = &gave_up;
    bool ok = true;
    rdl_grid_wait();
    rdl_grid_launch_dependents();

    if (warp == 0) {
        // ---- loader, in every block: its rows, its weight tiles, the scales of both ----
        int s = 0;
        uint32_t parity = 1, extra = (uint32_t)a.test_extra_tx;      // the first round finds every place free
        for (int tile = first_tile; tile < n_tiles && ok; tile += tile_step) {
            int m0, n0;
            tile_origin(tile, m0, n0);
            // the tile's two weight tiles; where their number is odd the last second one is not there, and arrives as zeros
            const int piece = (GATED ? 2 * n0 : n0) / MX_ROWS * a.blocks, piece1 = piece + a.blocks;
            for (int kb = 0; kb < a.blocks; ++kb) {
                if (!mx_warp_wait(mx_smem(&empty_bar[s]), parity, a.wait_cycles, gave_up_v)) { ok = false; break; }
                if (mx_elect()) {
                    const uint32_t own = mx_smem(&full_bar[s]), full = CTAS == 1 ? own : map_to_block(own, 0), st = mx_smem(smem + (size_t)s * PITCH);
                    if (rank == 0) mx_bar_expect(own, CTAS * stage_tx(CTAS) + extra);
                    load_3d<CTAS>(st, &map_x, kb * BK, m0 / 4, full);
                    if (CTAS == 1) {
                        load_2d<CTAS>(st + A_BYTES, &map_w, 0, (piece + kb) * MX_ROWS, full);
                        load_2d<CTAS>(st + A_BYTES + MX_TILE_BYTES, &map_w, 0, (piece1 + kb) * MX_ROWS, full);
                    } else {
                        load_2d<CTAS>(st + A_BYTES, &map_w, 0, ((rank ? piece1 : piece) + kb) * MX_ROWS, full);
                    }
                    load_2d<CTAS>(st + SCALES, &map_xs, m0, kb, full);
                    load_2d<CTAS>(st + SCALES + MX_SCALE_BYTES, &map_ws, 0, piece + kb, full);
                    load_2d<CTAS>(st + SCALES + 2 * MX_SCALE_BYTES, &map_ws, 0, piece1 + kb, full);
                }
                __syncwarp();
                extra = 0;
                if (++s == STAGES) { s = 0; parity ^= 1; }
            }
        }
    } else if (warp == 1) {
        // ---- scales to tensor memory, and the products: one thread, of a pair in block 0 ----
        int s = 0, lt = 0, scale_buf = 0;
        uint32_t parity = 0;
        for (int tile = first_tile; tile < n_tiles && ok && rank == 0; tile += tile_step, ++lt) {
            if (!mx_warp_wait(mx_smem(&acc_empty), (lt & 1) ^ 1, a.wait_cycles, gave_up_v)) { ok = false; break; }
            mx_fence_after();
            for (int kb = 0; kb < a.blocks; ++kb) {
                if (!mx_warp_wait(mx_smem(&full_bar[s]), parity, a.wait_cycles, gave_up_v)) { ok = false; break; }
                mx_fence_after();
                if (mx_elect()) {
                    const uint32_t st = mx_smem(smem + (size_t)s * PITCH);
                    const uint32_t sa = tmem + BN + (uint32_t)scale_buf * SCALE_COLS, sb = sa + 4;
                    copy_scales<CTAS>(sa, mx_scale_desc(st + SCALES));
                    copy_scales<CTAS>(sb, mx_scale_desc(st + SCALES + MX_SCALE_BYTES));
                    copy_scales<CTAS>(sb + 4, mx_scale_desc(st + SCALES + 2 * MX_SCALE_BYTES));
                    const uint64_t ad = mx_operand_desc(st), bd = mx_operand_desc(st + A_BYTES);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_mx<CTAS>(tmem, ad + (uint32_t)(k * 2), bd + (uint32_t)(k * 2), mx_idesc(MX_E4M3, MX_E2M1, TILE_M, BN, k), sa, sb, (kb | k) != 0);
                    commit<CTAS>(mx_smem(&empty_bar[s]));
                }
                __syncwarp();
                scale_buf = (scale_buf + 1) & (SCALE_BUFS - 1);
                if (++s == STAGES) { s = 0; parity ^= 1; }
            }
            if (ok && mx_elect()) commit<CTAS>(mx_smem(&acc_full));
            __syncwarp();
        }
    } else {
        // ---- epilogue: warp q of four has the lanes of rows 4 l + q; four warps share them, 64 columns of the accumulator each ----
        const int q = warp & 3, part = (warp - 2) >> 2;
        unsigned char* stage = smem + (size_t)STAGES * PITCH + (size_t)(warp - 2) * EPI_STAGE_BYTES;
        const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + 64 * part;
        const bool vec = a.N % 8 == 0;
        int lt = 0;
        const uint32_t to_issuer = CTAS == 1 ? mx_smem(&acc_empty) : map_to_block(mx_smem(&acc_empty), 0);
        for (int tile = first_tile; tile < n_tiles; tile += tile_step, ++lt) {
            int m0, n0;
            tile_origin(tile, m0, n0);
            if (!mx_bar_wait(mx_smem(&acc_full), lt & 1, a.wait_cycles, gave_up_v)) { ok = false; break; }
            mx_fence_after();
            uint32_t v[64];                                               // weight rows 64 part + i of the tile
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld16(lanes + 16 * c, &v[16 * c]);
            mx_tmem_wait_ld();
            mx_fence_before();
            __syncwarp();
            if (lane == 0) arrive_at(to_issuer);                          // the next tile's products may begin
            const int m = m0 + 4 * lane + q, nb = n0 + (GATED ? 32 : 64) * part;
            constexpr int PIECES = GATED ? 1 : 2;                         // of 32 outputs
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                const int n = nb + 32 * p;
                if (n >= a.N && a.out_kind != RDL_MX8) break;             // the same for the whole warp
                float y[32], u[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    // gated: 16 gate rows, then the 16 up rows of the same outputs
                    const int r = GATED ? (i >> 4) * 32 + (i & 15) : 32 * p + i;
                    y[i] = __uint_as_float(v[r]);
                    u[i] = GATED ? __uint_as_float(v[(r + 16) & 63]) : 0.f;
                }
                // rows that are not there are zeros, and zeros take the long way through a division: 64 rows of 128, 256,000 capped
                // outputs took 159 us with their epilogue and take 90 without
                if (m < a.M) finish<GATED>(a, y, u);
                if (a.out_kind == RDL_MX8) {
                    if (m < a.M) store_group(a, m, n, y);
                    continue;
                }
                // Through shared memory, 64 bytes of 32 rows at a time, so that neighbouring lanes store neighbouring bytes.  The 16-byte
                // piece c of row r lies at piece c ^ (r >> 1 & 3): the lanes of a row each write without conflicts.
                const int swz = (lane >> 1) & 3;
                if (a.out_kind == RDL_BF16) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint4 raw;
                        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
                        for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(y[8 * i + 2 * e], y[8 * i + 2 * e + 1]);
                        *reinterpret_cast<uint4*>(stage + lane * 64 + ((i ^ swz) << 4)) = raw;
                    }
                    __syncwarp();
                    if (vec) {
                        const int c = lane & 3, col = n + c * 8;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int r = j * 8 + (lane >> 2), row = m0 + 4 * r + q;
                            const uint4 raw = *reinterpret_cast<const uint4*>(stage + r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
                            if (row < a.M && col < a.N) *reinterpret_cast<uint4*>((__nv_bfloat16*)a.out + (long long)row * a.N + col) = raw;
                        }
                    } else {                                              // rows that begin anywhere: a column a lane, 16 rows in flight
                        __nv_bfloat16* o = (__nv_bfloat16*)a.out + (long long)(m0 + q) * a.N + n + lane;
                        const long long step = 4LL * a.N;
                        const int there = n + lane < a.N ? (a.M - m0 - q + 3) / 4 : 0;      // rows 4 r + q of the tile that are there
#pragma unroll
                        for (int r0 = 0; r0 < 32; r0 += 16) {
                            __nv_bfloat16 e[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                const int r = r0 + j;
                                e[j] = *reinterpret_cast<const __nv_bfloat16*>(stage + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4) + (lane & 7) * 2);
                            }
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                if (r0 + j < there) o[(r0 + j) * step] = e[j];
                        }
                    }
                    __syncwarp();
                } else {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {                // 16 columns of float
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            *reinterpret_cast<float4*>(stage + lane * 64 + ((i ^ swz) << 4)) =
                                make_float4(y[16 * half + 4 * i], y[16 * half + 4 * i + 1], y[16 * half + 4 * i + 2], y[16 * half + 4 * i + 3]);
                        __syncwarp();
#pragma unroll 8
                        for (int j = 0; j < 16; ++j) {
                            const int r = j * 2 + (lane >> 4), row = m0 + 4 * r + q, col = n + 16 * half + (lane & 15);
                            const float e = *reinterpret_cast<const float*>(stage + r * 64 + ((((lane & 15) >> 2) ^ ((r >> 1) & 3)) << 4) + (lane & 3) * 4);
                            if (row < a.M && col < a.N) ((float*)a.out)[(long long)row * a.N + col] = e;
                        }
                        __syncwarp();
                    }
                }
            }
        }
    }
    if (!ok && a.status) atomicExch(a.status, RDL_FAULT_MX_MANY);
    if (*gave_up_v && threadIdx.x == 0) mx_drain();
    // ---- tear-down, reached by every thread ----
    mx_fence_before();
    __syncthreads();
    if (CTAS == 2) cluster_sync();       // neither block leaves while the other may still read its shared memory or report to its barriers
    if (warp == 1)
        MX_CTA_GROUP(CTAS, asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory"),
                     asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory"));
}

template <bool GATED, int CTAS>
int launch(const MxRowsMaps& maps, const Mx4Matrix& w, const ManyArgs& a, cudaStream_t st) {
    constexpr int OUT_BN = GATED ? BN / 2 : BN;
    const long long tiles = (long long)((a.N + OUT_BN - 1) / OUT_BN) * ((a.M + BM * CTAS - 1) / (BM * CTAS));
    RDL_REQUIRE(tiles <= 0x3fffffffLL, "mx_many_rows: %lld tiles are too many", tiles);
    const int at_once = rdl_sm_count() / CTAS > 0 ? rdl_sm_count() / CTAS : 1;
    RDL_CUDA((rdl_allow_shared<mx_many_rows_kernel<GATED, CTAS>>(smem_bytes(CTAS))), "mx_many_rows");
    RDL_CHECK_EX(rdl_launch_cluster(mx_many_rows_kernel<GATED, CTAS>, dim3((tiles < at_once ? (int)tiles : at_once) * CTAS), dim3(THREADS), CTAS,
                                    (size_t)smem_bytes(CTAS), st, maps.values, maps.scales, w.codes_map, w.scales_map, a), "mx_many_rows");
    return 0;
}

}  // namespace

extern "C" int rdl_mx_many_rows(void* out, int out_kind, void* out_scales, const void* x, const void* row_scales, const void* weight, int m,
                                int activation, float act_param, float softcap, int* status, void* stream) {
    const Mx4Matrix* w = (const Mx4Matrix*)weight;
    RDL_REQUIRE(w && w->codes, "mx_many_rows: missing weight");
    RDL_REQUIRE(m >= 0, "mx_many_rows: %d rows", m);
    if (m == 0) return 0;
    RDL_REQUIRE(out && x && row_scales, "mx_many_rows: missing operand");
    RDL_REQUIRE(rdl_valid_dtype(out_kind) || (out_kind == RDL_MX8 && out_scales), "mx_many_rows: bad output (kind %d)", out_kind);
    RDL_REQUIRE((uintptr_t)x % 16 == 0 && (uintptr_t)row_scales % 16 == 0 && (uintptr_t)out % 16 == 0, "mx_many_rows: operands must start on 16-byte boundaries");
    RDL_REQUIRE(!w->gated || rdl_gated_known(activation), "mx_many_rows: unknown activation %d", activation);
    RDL_REQUIRE(softcap >= 0.f, "mx_many_rows: soft-cap must not be negative");
    if (m <= 128 && out_kind != RDL_MX8 && mx_some_rows_pay(*w, m))
        return rdl_mx_some_rows(out, out_kind, x, row_scales, weight, m, activation, act_param, softcap, status, stream);
    const int n = w->gated ? w->rows / 2 : w->rows;
    const long long blocks = w->blocks, rows4 = (m + 3LL) / 4 * 4;
    MxRowsMaps maps;
    if (int e = mx_rows_maps(&maps, x, row_scales, blocks, rows4)) return e;
    ManyArgs a{};
    a.out = out; a.out_kind = out_kind; a.out_scales = (uint8_t*)out_scales;
    a.M = m; a.N = n; a.blocks = (int)blocks;
    a.out_blocks = mx_blocks(n); a.out_padded_rows = (int)rows4;
    a.activation = activation; a.act_param = act_param; a.softcap = softcap;
    a.wait_cycles = rdl_wait_cycles_for(RDL_FAULT_MX_MANY); a.test_extra_tx = rdl_test_extra_tx_for(RDL_FAULT_MX_MANY);
    a.status = status;
    cudaStream_t st = (cudaStream_t)stream;
    if (m > BM) return w->gated ? launch<true, 2>(maps, *w, a, st) : launch<false, 2>(maps, *w, a, st);
    return w->gated ? launch<true, 1>(maps, *w, a, st) : launch<false, 1>(maps, *w, a, st);
}
