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
// A block computes 128 x 256 tiles, one after another (persistent): warp 0 loads, warp 1 copies scales and issues the products, eight
// warps take the accumulator out of tensor memory at once, all of it into registers, so that the next tile's products can
// start, and then apply the epilogue and store.  The gated form's tile is 128 gate and 128 up rows of the same 128 outputs; its result
// may leave as 8-bit rows with scales: 32 outputs of a row lie in one thread, which is a group.
//
// Every wait is bounded; a block that gives up sets `status` and every path ends in the common tear-down.
#include "activations.cuh"
#include "api.h"
#include "launch.cuh"
#include "mx_tensor.cuh"

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

struct ManyArgs {
    void* out; int out_kind;                              // RDL_F32, RDL_BF16, or RDL_MX8 with out_scales
    uint8_t* out_scales;
    const uint8_t* scales;                                // of the weight
    int M, N, blocks, weight_tiles;                       // blocks of 128 columns, weight tiles of 128 rows
    int out_blocks, out_padded_rows;                      // RDL_MX8
    int activation; float act_param, softcap;
    long long wait_cycles; int test_extra_tx;
    int* status;
};

__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
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
        } else if (a.activation == RDL_ACT_GELU_TANH) {
            // 0.5 (1 + tanh z) = 1 / (1 + exp(-2 z)): the fast exponential and quotient are good to 2^-20, where the hardware's tanh, at
            // 2^-11, would move one 8-bit code in a thousand
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const float z = 0.7978845608028654f * (y[i] + 0.044715f * y[i] * y[i] * y[i]);
                y[i] = __fdividef(y[i], 1.0f + __expf(fminf(-2.0f * z, 80.0f))) * u[i];
            }
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

template <bool GATED>
__global__ void __launch_bounds__(THREADS, 1) mx_many_rows_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_xs,
                                                           const __grid_constant__ CUtensorMap map_w, const __grid_constant__ ManyArgs a) {
    constexpr int OUT_BN = GATED ? BN / 2 : BN;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) unsigned long long full_bar[STAGES], empty_bar[STAGES], acc_full, acc_empty;
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up;
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;      // the compiler may know it uniform
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
            mx_bar_init(mx_smem(&full_bar[s]), 1);
            mx_bar_init(mx_smem(&empty_bar[s]), 1);
        }
        mx_bar_init(mx_smem(&acc_full), 1);
        mx_bar_init(mx_smem(&acc_empty), EPI_WARPS);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(mx_smem(&tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    mx_fence_before();
    __syncthreads();
    mx_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
    volatile int* gave_up_v = &gave_up;
    bool ok = true;
    rdl_grid_wait();
    rdl_grid_launch_dependents();

    if (warp == 0) {
        // ---- loader ----
        int s = 0;
        uint32_t parity = 1, extra = (uint32_t)a.test_extra_tx;      // the first round finds every place free
        for (int tile = blockIdx.x; tile < n_tiles && ok; tile += gridDim.x) {
            int m0, n0;
            tile_origin(tile, m0, n0);
            const int w_tile = (GATED ? 2 * n0 : n0) / MX_ROWS;
            // the tile's two weight tiles; where their number is odd the last second one is not there: its codes arrive as zeros
            const int piece = w_tile * a.blocks, piece1 = piece + a.blocks, scales1 = w_tile + 1 < a.weight_tiles ? piece1 : piece;
            for (int kb = 0; kb < a.blocks; ++kb) {
                if (!mx_warp_wait(mx_smem(&empty_bar[s]), parity, a.wait_cycles, gave_up_v)) { ok = false; break; }
                if (mx_elect()) {
                    const uint32_t full = mx_smem(&full_bar[s]), st = mx_smem(smem + (size_t)s * STAGE_PITCH);
                    mx_bar_expect(full, STAGE_TX + extra);
                    tma_3d(st, &map_x, kb * BK, m0 / 4, 0, full);
                    mx_tma_2d(st + A_BYTES, &map_w, 0, (piece + kb) * MX_ROWS, full);
                    mx_tma_2d(st + A_BYTES + B_BYTES / 2, &map_w, 0, (piece1 + kb) * MX_ROWS, full);
                    mx_tma_2d(st + A_BYTES + B_BYTES, &map_xs, m0, kb, full);
                    mx_bulk(st + A_BYTES + B_BYTES + SA_BYTES, a.scales + (long long)(piece + kb) * MX_SCALE_BYTES, MX_SCALE_BYTES, full);
                    mx_bulk(st + A_BYTES + B_BYTES + SA_BYTES + SB_BYTES / 2, a.scales + (long long)(scales1 + kb) * MX_SCALE_BYTES, MX_SCALE_BYTES, full);
                }
                __syncwarp();
                extra = 0;
                if (++s == STAGES) { s = 0; parity ^= 1; }
            }
        }
    } else if (warp == 1) {
        // ---- scales to tensor memory, and the products ----
        int s = 0, lt = 0, scale_buf = 0;
        uint32_t parity = 0;
        for (int tile = blockIdx.x; tile < n_tiles && ok; tile += gridDim.x, ++lt) {
            if (!mx_warp_wait(mx_smem(&acc_empty), (lt & 1) ^ 1, a.wait_cycles, gave_up_v)) { ok = false; break; }
            mx_fence_after();
            for (int kb = 0; kb < a.blocks; ++kb) {
                if (!mx_warp_wait(mx_smem(&full_bar[s]), parity, a.wait_cycles, gave_up_v)) { ok = false; break; }
                mx_fence_after();
                if (mx_elect()) {
                    const uint32_t st = mx_smem(smem + (size_t)s * STAGE_PITCH);
                    const uint32_t sa = tmem + BN + (uint32_t)scale_buf * SCALE_COLS, sb = sa + 4;
                    copy_scales(sa, mx_scale_desc(st + A_BYTES + B_BYTES));
                    copy_scales(sb, mx_scale_desc(st + A_BYTES + B_BYTES + SA_BYTES));
                    copy_scales(sb + 4, mx_scale_desc(st + A_BYTES + B_BYTES + SA_BYTES + SB_BYTES / 2));
                    const uint64_t ad = mx_operand_desc(st), bd = mx_operand_desc(st + A_BYTES);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_mx(tmem, ad + (uint32_t)(k * 2), bd + (uint32_t)(k * 2), mx_idesc(MX_E4M3, MX_E2M1, BM, BN, k), sa, sb, (kb | k) != 0);
                    commit(mx_smem(&empty_bar[s]));
                }
                __syncwarp();
                scale_buf = (scale_buf + 1) & (SCALE_BUFS - 1);
                if (++s == STAGES) { s = 0; parity ^= 1; }
            }
            if (ok && mx_elect()) commit(mx_smem(&acc_full));
            __syncwarp();
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
            if (!mx_bar_wait(mx_smem(&acc_full), lt & 1, a.wait_cycles, gave_up_v)) { ok = false; break; }
            mx_fence_after();
            // this half's 128 columns; v[c][i]: weight row 32 c + i of them
            uint32_t v[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                tmem_ld16(lanes + 128 * half + 32 * c, &v[c][0]);
                tmem_ld16(lanes + 128 * half + 32 * c + 16, &v[c][16]);
            }
            mx_tmem_wait_ld();
            mx_fence_before();
            __syncwarp();
            if (lane == 0) mx_bar_arrive(mx_smem(&acc_empty));             // the next tile's products may begin
            const int m = m0 + 4 * lane + q, nb = n0 + (GATED ? 64 : 128) * half;
            constexpr int PIECES = GATED ? 2 : 4;                         // of 32 outputs
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                const int n = nb + 32 * p;
                float y[32], u[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    // gated: 16 gate rows, then the 16 up rows of the same outputs
                    const int r = GATED ? 64 * p + (i >> 4) * 32 + (i & 15) : 32 * p + i;
                    y[i] = __uint_as_float(v[r >> 5][r & 31]);
                    u[i] = GATED ? __uint_as_float(v[r >> 5][(r + 16) & 31]) : 0.f;
                }
                finish<GATED>(a, y, u);
                if (a.out_kind == RDL_MX8) {
                    if (m < a.M) store_group(a, m, n, y);
                } else if (a.out_kind == RDL_BF16) {
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
                        const int n1 = n - 32;                           // the first of 64 columns
                        if (vec) {
                            const int c = lane & 7, col = n1 + c * 8;
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const int r = j * 4 + (lane >> 3), row = m0 + 4 * r + q;
                                const uint4 raw = *reinterpret_cast<const uint4*>(stage + r * 128 + ((c ^ (r & 7)) << 4));
                                if (row < a.M && col < a.N) *reinterpret_cast<uint4*>((__nv_bfloat16*)a.out + (long long)row * a.N + col) = raw;
                            }
                        } else {                                         // rows that begin anywhere: 32 neighbouring columns an instruction
#pragma unroll 4
                            for (int r = 0; r < 32; ++r) {
                                const int row = m0 + 4 * r + q;
                                if (row >= a.M) break;                   // the same for the whole warp
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    const int c = h * 32 + lane;
                                    const __nv_bfloat16 e = *reinterpret_cast<const __nv_bfloat16*>(stage + r * 128 + (((c >> 3) ^ (r & 7)) << 4) + (c & 7) * 2);
                                    if (n1 + c < a.N) ((__nv_bfloat16*)a.out)[(long long)row * a.N + n1 + c] = e;
                                }
                            }
                        }
                        __syncwarp();
                    }
                } else {                                                 // float: 32 columns are 128 bytes of a row
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        *reinterpret_cast<float4*>(stage + lane * 128 + ((i ^ (lane & 7)) << 4)) = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
                    __syncwarp();
#pragma unroll 4
                    for (int r = 0; r < 32; ++r) {
                        const int row = m0 + 4 * r + q;
                        if (row >= a.M) break;
                        const float e = *reinterpret_cast<const float*>(stage + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
                        if (n + lane < a.N) ((float*)a.out)[(long long)row * a.N + n + lane] = e;
                    }
                    __syncwarp();
                }
            }
        }
    }
    if (!ok && a.status) atomicExch(a.status, RDL_FAULT_MX_MANY);
    if (*gave_up_v && threadIdx.x == 0) mx_drain();
    // ---- tear-down, reached by every thread ----
    mx_fence_before();
    __syncthreads();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
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
    const int n = w->gated ? w->rows / 2 : w->rows;
    const cuuint64_t blocks = w->blocks, cols = blocks * MX_BLOCK, rows4 = (m + 3LL) / 4 * 4;
    CUtensorMap mx, mxs;
    if (int e = mx_make_map(&mx, x, {CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, {cols, rows4 / 4, 4}, {cols * 4, cols}, {BK, 32, 4}, CU_TENSOR_MAP_SWIZZLE_128B}, "8-bit rows")) return e;
    if (int e = mx_make_map(&mxs, row_scales, {CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, {rows4, blocks}, {rows4 * 4}, {BM, 1}, CU_TENSOR_MAP_SWIZZLE_NONE},
                            "the scales of 8-bit rows")) return e;
    ManyArgs a{};
    a.out = out; a.out_kind = out_kind; a.out_scales = (uint8_t*)out_scales;
    a.scales = w->scales;
    a.M = m; a.N = n; a.blocks = (int)blocks; a.weight_tiles = w->tiles;
    a.out_blocks = mx_blocks(n); a.out_padded_rows = (int)rows4;
    a.activation = activation; a.act_param = act_param; a.softcap = softcap;
    a.wait_cycles = rdl_wait_cycles_for(RDL_FAULT_MX_MANY); a.test_extra_tx = rdl_test_extra_tx_for(RDL_FAULT_MX_MANY);
    a.status = status;
    const int out_bn = w->gated ? BN / 2 : BN;
    const long long tiles = (long long)((n + out_bn - 1) / out_bn) * ((m + BM - 1) / BM);
    RDL_REQUIRE(tiles <= 0x3fffffffLL, "mx_many_rows: %lld tiles are too many", tiles);
    const int grid = tiles < rdl_sm_count() ? (int)tiles : rdl_sm_count();
    cudaStream_t st = (cudaStream_t)stream;
    if (w->gated) {
        RDL_CUDA(rdl_allow_shared<mx_many_rows_kernel<true>>(SMEM_BYTES), "mx_many_rows");
        RDL_CHECK_EX(rdl_launch(mx_many_rows_kernel<true>, dim3(grid), dim3(THREADS), (size_t)SMEM_BYTES, st, mx, mxs, w->codes_map, a), "mx_many_rows");
    } else {
        RDL_CUDA(rdl_allow_shared<mx_many_rows_kernel<false>>(SMEM_BYTES), "mx_many_rows");
        RDL_CHECK_EX(rdl_launch(mx_many_rows_kernel<false>, dim3(grid), dim3(THREADS), (size_t)SMEM_BYTES, st, mx, mxs, w->codes_map, a), "mx_many_rows");
    }
    return 0;
}
