// Many rows of 8 bits times a 4-bit weight matrix (microscaling.cuh) on the fifth-generation tensor cores:
//   out[m, n] = epilogue(sum_k x[m, k] w[n, k]),  x e4m3 and w e2m1, each with a power of two a group of 32 columns.
//
// tcgen05.mma.kind::mxf8f6f4.block_scale multiplies 32 columns at a time, applies both groups' scales and sums in float in tensor
// memory, at twice the rate of bfloat16.  TMA brings the rows as they lie and the codes spread to a byte each (the
// 16U4_ALIGN16B type: 16 codes in 8 of every 16 bytes, the form the instruction reads 4-bit operands in), so nothing is
// unpacked by threads.  Scales reach shared memory as words of a row's four groups and tensor memory by tcgen05.cp, issued
// by the thread that issues the products, ahead of them and in order with them.
//
// tcgen05.cp takes 32 lanes of 16 bytes: word 4 l + c of 128 lands in lane l, column c, where the instruction looks for the scales of
// operand row 32 c + l.  The scales lie in memory row by row, so operand row 32 c + l has to be row 4 l + c of the tile.
// The tensor maps do that: a matrix is described as [4][rows / 4][columns] and a box of 4 x 32 rows arrives in that order.
// The epilogue undoes it: lane l of quarter c holds row 4 l + c, accumulator column 32 c + l is output 4 l + c.
//
// A block computes 128 x 256 tiles, one after another (persistent): warp 0 loads, warp 1 copies scales and issues the products, eight
// warps take the accumulator out of tensor memory at once, all of it into registers, so that the next tile's products can
// start, and then apply the epilogue and store.  The gated form's tile is 128 gate and 128 up rows of the same 128 outputs; its result
// may leave as 8-bit rows with scales: 32 outputs of a row lie in one thread, which is a group.
//
// Every wait is bounded; a block that gives up sets `status` and every path ends in the common tear-down.
#include <cuda.h>

#include "activations.cuh"
#include "api.h"
#include "launch.cuh"
#include "microscaling.cuh"

namespace {

constexpr int BM = 128, BN = 256, BK = MX_BLOCK, STAGES = 3, THREADS = 320, EPI_WARPS = 8;
constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK, SA_BYTES = BM * 4, SB_BYTES = BN * 4;
constexpr int STAGE_PITCH = (A_BYTES + B_BYTES + SA_BYTES + SB_BYTES + 1023) / 1024 * 1024;
constexpr int STAGE_TX = A_BYTES + B_BYTES / 2 + SA_BYTES + SB_BYTES;      // the codes' transfers count the bytes they read, not those they fill
constexpr int EPI_STAGE_BYTES = 32 * 128;
constexpr int SMEM_BYTES = STAGES * STAGE_PITCH + EPI_WARPS * EPI_STAGE_BYTES + 1024;
constexpr int SCALE_COLS = 16, SCALE_BUFS = 4;            // tensor memory: 4 + 8 columns of scales a buffer, behind the accumulator
constexpr int TMEM_COLS = 512;
constexpr int RASTER_GROUP = 8;                           // row tiles that share a weight tile and run together

struct MxTcArgs {
    void* out; int out_kind;                              // RDL_F32, RDL_BF16, or RDL_MX8 with out_scales
    uint8_t* out_scales;
    int M, N, blocks;                                     // blocks of 128 columns
    int half_padded;                                      // gated: weight row where the up rows begin
    int out_blocks, out_padded_rows;                      // RDL_MX8
    int activation; float act_param, softcap;
    long long wait_cycles; int test_extra_tx;
    int* status;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar, int count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// false where the phase did not complete in time, or where another warp of the block has given up
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, long long limit, volatile int* gave_up) {
    if (bar_try(bar, parity)) return true;
    const long long t0 = clock64();
    while (!bar_try(bar, parity)) {
        if (*gave_up) return false;
        if (clock64() - t0 > limit) { *gave_up = 1; return false; }
    }
    return true;
}
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
// K-major operand tile, rows of 128 bytes, 128-byte swizzle: groups of 8 rows are 1024 bytes apart
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// scales as tcgen05.cp reads them: no swizzle, 8 lanes of 16 bytes are 128 bytes, the next eight right behind
__device__ __forceinline__ uint64_t scale_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | (8ull << 32) | (1ull << 46);
}
// instruction descriptor of the block-scaled kinds: A e4m3 (0), B e2m1 (5) at bit 10, N >> 3 at bit 17, scales are powers of two (bit
// 23), M >> 7 at bit 27; which byte of the scale words counts: B at bit 4, A at bit 29
__host__ __device__ constexpr uint32_t mx_idesc(int m, int n, int byte) {
    return ((uint32_t)byte << 4) | (5u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 7) << 27) | ((uint32_t)byte << 29);
}
__device__ __forceinline__ void mma_mx(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// 16 accumulator columns of the warp's lanes; complete after tmem_wait
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float* v) {
    uint32_t r[16];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr) : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// The 32 outputs [n, n + 32) of one row, in order: epilogue and store.
template <bool GATED>
__device__ __forceinline__ void finish(const MxTcArgs& a, float (&y)[32], const float (&u)[32]) {
    if (GATED) {
        if (a.out_kind == RDL_F32) {
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = rdl_gated(y[i], u[i], a.activation, a.act_param);
        } else if (a.activation == RDL_ACT_GELU_TANH) {      // rounded to 8 bits and fewer: the fast forms; the choice once a piece
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = rdl_activation_fast(y[i], RDL_ACT_GELU_TANH) * u[i];
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = rdl_gated_fast(y[i], u[i], a.activation, a.act_param);
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
__device__ __forceinline__ void store_group(const MxTcArgs& a, int m, int n, float (&y)[32]) {
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

template <bool GATED>
__global__ void __launch_bounds__(THREADS, 1) mx_tc_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_xs,
                                                           const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_ws,
                                                           const __grid_constant__ MxTcArgs a) {
    constexpr int OUT_BN = GATED ? BN / 2 : BN;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) unsigned long long full_bar[STAGES], empty_bar[STAGES], acc_full, acc_empty;
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles_m = (a.M + BM - 1) / BM, tiles_n = (a.N + OUT_BN - 1) / OUT_BN, n_tiles = tiles_m * tiles_n;
    auto tile_origin = [&](int tile, int& m0, int& n0) {
        const int per_group = RASTER_GROUP * tiles_n;
        const int group = tile / per_group, in_group = tile - group * per_group;
        const int first_m = group * RASTER_GROUP;
        const int gm = tiles_m - first_m < RASTER_GROUP ? tiles_m - first_m : RASTER_GROUP;
        m0 = (first_m + in_group % gm) * BM;
        n0 = (in_group / gm) * OUT_BN;
    };
    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int s = 0; s < STAGES; ++s) {
            bar_init(smem_u32(&full_bar[s]), 1);
            bar_init(smem_u32(&empty_bar[s]), 1);
        }
        bar_init(smem_u32(&acc_full), 1);
        bar_init(smem_u32(&acc_empty), EPI_WARPS);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;
    volatile int* gave_up_v = &gave_up;
    bool ok = true;
    rdl_grid_wait();
    rdl_grid_launch_dependents();

    if (warp == 0) {
        if (lane == 0) {
            // ---- loader ----
            int it = 0;
            for (int tile = blockIdx.x; tile < n_tiles && ok; tile += gridDim.x) {
                int m0, n0;
                tile_origin(tile, m0, n0);
                const int w0 = n0, w1 = GATED ? a.half_padded + n0 : n0 + 128;      // weight rows of the tile's two halves
                for (int kb = 0; kb < a.blocks; ++kb, ++it) {
                    const int s = it % STAGES;
                    if (!bar_wait(smem_u32(&empty_bar[s]), ((it / STAGES) & 1) ^ 1, a.wait_cycles, gave_up_v)) { ok = false; break; }
                    const uint32_t full = smem_u32(&full_bar[s]), st = smem_u32(smem + (size_t)s * STAGE_PITCH);
                    bar_expect(full, STAGE_TX + (it == 0 ? (uint32_t)a.test_extra_tx : 0u));
                    tma_3d(st, &map_x, kb * BK, m0 / 4, 0, full);
                    tma_3d(st + A_BYTES, &map_w, kb * BK, w0 / 4, 0, full);
                    tma_3d(st + A_BYTES + B_BYTES / 2, &map_w, kb * BK, w1 / 4, 0, full);
                    tma_2d(st + A_BYTES + B_BYTES, &map_xs, m0, kb, full);
                    tma_3d(st + A_BYTES + B_BYTES + SA_BYTES, &map_ws, 0, kb, w0 / MX_UNIT, full);
                    tma_3d(st + A_BYTES + B_BYTES + SA_BYTES + SB_BYTES / 2, &map_ws, 0, kb, w1 / MX_UNIT, full);
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            // ---- scales to tensor memory, and the products ----
            int it = 0, lt = 0;
            for (int tile = blockIdx.x; tile < n_tiles && ok; tile += gridDim.x, ++lt) {
                if (!bar_wait(smem_u32(&acc_empty), (lt & 1) ^ 1, a.wait_cycles, gave_up_v)) { ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int kb = 0; kb < a.blocks; ++kb, ++it) {
                    const int s = it % STAGES;
                    if (!bar_wait(smem_u32(&full_bar[s]), (it / STAGES) & 1, a.wait_cycles, gave_up_v)) { ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t st = smem_u32(smem + (size_t)s * STAGE_PITCH);
                    const uint32_t sa = tmem + BN + (uint32_t)(it % SCALE_BUFS) * SCALE_COLS, sb = sa + 4;
                    copy_scales(sa, scale_desc(st + A_BYTES + B_BYTES));
                    copy_scales(sb, scale_desc(st + A_BYTES + B_BYTES + SA_BYTES));
                    copy_scales(sb + 4, scale_desc(st + A_BYTES + B_BYTES + SA_BYTES + SB_BYTES / 2));
                    const uint64_t ad = operand_desc(st), bd = operand_desc(st + A_BYTES);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_mx(tmem, ad + (uint32_t)(k * 2), bd + (uint32_t)(k * 2), mx_idesc(BM, BN, k), sa, sb, (kb | k) != 0);
                    commit(smem_u32(&empty_bar[s]));
                }
                if (ok) commit(smem_u32(&acc_full));
            }
        }
    } else {
        // ---- epilogue: warp q of four has the lanes of rows 4 l + q; two warps share them ----
        const int q = warp & 3, half = (warp - 2) >> 2;
        unsigned char* stage = smem + (size_t)STAGES * STAGE_PITCH + (size_t)(warp - 2) * EPI_STAGE_BYTES;
        const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
        const bool vec = a.N % 8 == 0;
        int lt = 0;
        for (int tile = blockIdx.x; tile < n_tiles; tile += gridDim.x, ++lt) {
            int m0, n0;
            tile_origin(tile, m0, n0);
            if (!bar_wait(smem_u32(&acc_full), lt & 1, a.wait_cycles, gave_up_v)) { ok = false; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            // plain: this half's 128 columns; gated: outputs [64 half, 64 half + 64) as 64 gate and 64 up columns.
            // v[c][i]: output 4 i + c from the first of them (i < 32; gated: i < 16 gate, then 16 up)
            float v[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if (GATED) {
                    tmem_ld16(lanes + 32 * c + 16 * half, &v[c][0]);
                    tmem_ld16(lanes + 128 + 32 * c + 16 * half, &v[c][16]);
                } else {
                    tmem_ld16(lanes + 128 * half + 32 * c, &v[c][0]);
                    tmem_ld16(lanes + 128 * half + 32 * c + 16, &v[c][16]);
                }
            }
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) bar_arrive(smem_u32(&acc_empty));             // the next tile's products may begin
            const int m = m0 + 4 * lane + q, nb = n0 + (GATED ? 64 : 128) * half;
            constexpr int PIECES = GATED ? 2 : 4;                         // of 32 outputs
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                const int n = nb + 32 * p;
                float y[32], u[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    y[i] = v[i & 3][8 * p + (i >> 2)];
                    u[i] = GATED ? v[i & 3][16 + 8 * p + (i >> 2)] : 0.f;
                }
                finish<GATED>(a, y, u);
                if (a.out_kind == RDL_MX8) {
                    if (m < a.M) store_group(a, m, n, y);
                } else if (a.out_kind == RDL_BF16 && vec) {
                    // through shared memory: two pieces are 128 bytes of a row, which leave as whole lines
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint4 raw;
                        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
                        for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(y[8 * i + 2 * e], y[8 * i + 2 * e + 1]);
                        *reinterpret_cast<uint4*>(stage + lane * 128 + ((((p & 1) * 4 + i) ^ (lane & 7)) << 4)) = raw;
                    }
                    if (p & 1) {
                        __syncwarp();
                        const int c = lane & 7, col = n - 32 + c * 8;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const int r = j * 4 + (lane >> 3), row = m0 + 4 * r + q;
                            const uint4 raw = *reinterpret_cast<const uint4*>(stage + r * 128 + ((c ^ (r & 7)) << 4));
                            if (row < a.M && col < a.N) *reinterpret_cast<uint4*>((__nv_bfloat16*)a.out + (long long)row * a.N + col) = raw;
                        }
                        __syncwarp();
                    }
                } else if (m < a.M) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (n + i < a.N) rdl_store(a.out, (long long)m * a.N + n + i, a.out_kind, y[i]);
                }
            }
        }
    }
    if (!ok && a.status) atomicExch(a.status, RDL_FAULT_MX_TC);
    if (*gave_up_v && threadIdx.x == 0)                   // copies that are on their way still write to this block's shared memory
        for (const long long t0 = clock64(); clock64() - t0 < RDL_COPY_DRAIN_CYCLES;) {}
    // ---- tear-down, reached by every thread ----
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// the driver's encoder, looked up at run time so that the library loads where there is no driver
int encoder(EncodeTiled* out) {
    static EncodeTiled encode = nullptr;
    if (!encode) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        RDL_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found), "mx_tc: looking up cuTensorMapEncodeTiled");
        RDL_REQUIRE(found == cudaDriverEntryPointSuccess && fn, "mx_tc: this driver has no cuTensorMapEncodeTiled");
        encode = (EncodeTiled)fn;
    }
    *out = encode;
    return 0;
}

struct MapShape {
    CUtensorMapDataType type; int rank;
    cuuint64_t dims[3], strides[2];                       // elements; bytes
    cuuint32_t box[3];
    CUtensorMapSwizzle swizzle;
};

int make_map(CUtensorMap* map, const void* p, const MapShape& s, const char* what) {
    EncodeTiled encode;
    if (int e = encoder(&encode)) return e;
    const cuuint32_t one[3] = {1, 1, 1};
    const CUresult r = encode(map, s.type, (cuuint32_t)s.rank, const_cast<void*>(p), s.dims, s.strides, s.box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              s.swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    RDL_REQUIRE(r == CUDA_SUCCESS, "mx_tc: cuTensorMapEncodeTiled failed with driver error %d for %s", (int)r, what);
    return 0;
}

}  // namespace

extern "C" int rdl_mx_tc(void* out, int out_kind, void* out_scales, const void* x, const void* row_scales, const void* codes, const void* scales,
                         int m, int n, int k, int gated, int activation, float act_param, float softcap, int* status, void* stream) {
    RDL_REQUIRE(out && x && row_scales && codes && scales, "mx_tc: missing operand");
    RDL_REQUIRE(rdl_valid_dtype(out_kind) || (out_kind == RDL_MX8 && out_scales), "mx_tc: bad output (kind %d)", out_kind);
    RDL_REQUIRE(m >= 0 && n > 0 && k > 0, "mx_tc: m=%d n=%d k=%d", m, n, k);
    RDL_REQUIRE((uintptr_t)x % 16 == 0 && (uintptr_t)row_scales % 16 == 0 && (uintptr_t)codes % 32 == 0 && (uintptr_t)scales % 16 == 0 && (uintptr_t)out % 16 == 0,
                "mx_tc: operands must start on 16-byte boundaries, the codes on a 32-byte boundary");
    RDL_REQUIRE(!gated || rdl_gated_known(activation), "mx_tc: unknown activation %d", activation);
    RDL_REQUIRE(softcap >= 0.f, "mx_tc: soft-cap must not be negative");
    if (m == 0) return 0;
    const long long blocks = mx_blocks(k), cols = blocks * MX_BLOCK, rows4 = (m + 3) / 4 * 4;
    const long long half = (n + MX_UNIT - 1) / MX_UNIT * MX_UNIT, wrows = gated ? 2 * half : half;
    CUtensorMap mx, mxs, mw, mws;
    if (int e = make_map(&mx, x, {CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, {(cuuint64_t)cols, (cuuint64_t)rows4 / 4, 4}, {(cuuint64_t)cols * 4, (cuuint64_t)cols},
                                  {BK, 32, 4}, CU_TENSOR_MAP_SWIZZLE_128B}, "the rows")) return e;
    if (int e = make_map(&mxs, row_scales, {CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, {(cuuint64_t)rows4, (cuuint64_t)blocks}, {(cuuint64_t)rows4 * 4},
                                            {BM, 1}, CU_TENSOR_MAP_SWIZZLE_NONE}, "the rows' scales")) return e;
    if (int e = make_map(&mw, codes, {CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, 3, {(cuuint64_t)cols, (cuuint64_t)wrows / 4, 4}, {(cuuint64_t)cols * 2, (cuuint64_t)cols / 2},
                                      {BK, 32, 4}, CU_TENSOR_MAP_SWIZZLE_128B}, "the codes")) return e;
    if (int e = make_map(&mws, scales, {CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, {64, (cuuint64_t)blocks, (cuuint64_t)wrows / MX_UNIT}, {64, (cuuint64_t)blocks * 64},
                                        {64, 1, 8}, CU_TENSOR_MAP_SWIZZLE_NONE}, "the scales")) return e;
    MxTcArgs a{};
    a.out = out; a.out_kind = out_kind; a.out_scales = (uint8_t*)out_scales;
    a.M = m; a.N = n; a.blocks = (int)blocks;
    a.half_padded = gated ? (int)half : 0;
    a.out_blocks = mx_blocks(n); a.out_padded_rows = (int)rows4;
    a.activation = activation; a.act_param = act_param; a.softcap = softcap;
    a.wait_cycles = rdl_wait_cycles_for(RDL_FAULT_MX_TC); a.test_extra_tx = rdl_test_extra_tx_for(RDL_FAULT_MX_TC);
    a.status = status;
    const int out_bn = gated ? BN / 2 : BN;
    const long long tiles = (long long)((n + out_bn - 1) / out_bn) * ((m + BM - 1) / BM);
    RDL_REQUIRE(tiles <= 0x3fffffffLL, "mx_tc: %lld tiles are too many", tiles);
    const int grid = tiles < rdl_sm_count() ? (int)tiles : rdl_sm_count();
    cudaStream_t st = (cudaStream_t)stream;
    if (gated) {
        RDL_CUDA(rdl_allow_shared<mx_tc_kernel<true>>(SMEM_BYTES), "mx_tc");
        RDL_CHECK_EX(rdl_launch(mx_tc_kernel<true>, dim3(grid), dim3(THREADS), (size_t)SMEM_BYTES, st, mx, mxs, mw, mws, a), "mx_tc");
    } else {
        RDL_CUDA(rdl_allow_shared<mx_tc_kernel<false>>(SMEM_BYTES), "mx_tc");
        RDL_CHECK_EX(rdl_launch(mx_tc_kernel<false>, dim3(grid), dim3(THREADS), (size_t)SMEM_BYTES, st, mx, mxs, mw, mws, a), "mx_tc");
    }
    return 0;
}
