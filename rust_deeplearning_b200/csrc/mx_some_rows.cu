// 17 to 128 rows of 8 bits times a 4-bit weight matrix (formats: microscaling.cuh): short prompts, wide batches.
//
// Bound by the bytes of the weights, as fewer rows are, so the weight tile is the M side of the block-scaled product (mx_tensor.cuh) and
// the rows, all of them, its N side of 128: every weight byte is read once, and a matrix makes as many tiles as it has 128
// rows, however few rows there are.  With the rows as the M side (mx_many_rows.cu) 64 rows of 2,304 x 4,096 kept 16 multiprocessors busy and
// took 10 us.  Rows that are not there arrive as zeros and cost no transfer.
//
// The rows' scales lie in memory row by row; as there, the rows' tensor map brings row 4 l + c to operand row 32 c + l, where
// tcgen05.cp puts its scales, and the epilogue knows that accumulator column 32 c + l is row 4 l + c.
//
// Warp 0 loads (weights before the kernel ahead has ended, the rows after), warp 1 issues scales and products, eight warps take the
// sums out.  A matrix with fewer tiles than multiprocessors: a cluster of up to 8 blocks shares a tile, each with its part of the
// columns; when all are done they send their sums through distributed shared memory, over what was the ring, to the block that adds
// up that part of the outputs, in rank order.  Every wait is bounded.
//
// Measured: 64 rows x 2,304 x 4,096 outputs 7.6 us, x 14,336 x 3,584 12.7 us (27 MB of weights, 2.2 TB/s); 128 rows 10.5 and 15.7 us.
#include <atomic>

#include "activations.cuh"
#include "api.h"
#include "launch.cuh"
#include "mx_tensor.cuh"

namespace {

constexpr int THREADS = 320, EPI = 256, MAX_STAGES = 6, SCALE_BUFS = 4, ROWS = 128;
constexpr int STAGE_BYTES = 2 * MX_TILE_BYTES + 2 * MX_SCALE_BYTES;                   // codes | rows | scales of both
constexpr int STAGE_TX = MX_TILE_TX + MX_TILE_BYTES + 2 * MX_SCALE_BYTES;
// Tensor memory: two accumulators of 128 columns, then scales; in a cluster, where a block has one tile, one accumulator (the reason stands in mx_tensor.cuh)
constexpr int TMEM_COLS = 512, CLUSTER_TMEM_COLS = 256, CLUSTER_STAGES = 3;
static_assert(2 * ROWS + SCALE_BUFS * 8 <= TMEM_COLS && ROWS + SCALE_BUFS * 8 <= CLUSTER_TMEM_COLS && 2 * CLUSTER_TMEM_COLS <= 512, "columns of tensor memory");
static_assert(3 * (CLUSTER_STAGES * STAGE_BYTES + 1024) > 228 * 1024, "no three blocks of clusters on a multiprocessor");
constexpr int OUTS_MOST = MX_ROWS + 16;                                               // weight rows of a tile over all blocks of a cluster, rounded up
// floats from a weight row's sums to the next one's: 16 bytes beyond whole lines, so that neighbouring lanes use different banks
__host__ __device__ constexpr int sums_pitch(int m) { return (m + 31) / 32 * 32 + 4; }

struct SomeArgs {
    void* out; int out_dtype;
    int M, N, blocks;                            // rows, outputs, blocks of 128 columns
    int tiles, split, slice_blocks, stages, share;
    int gated, activation; float act_param, softcap;
    long long wait_cycles; int test_extra_tx;
    int* status;
};

__device__ __forceinline__ void load_rows(uint32_t dst, const CUtensorMap* map, int x, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(0), "r"(0), "r"(bar) : "memory");
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
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {          // as bits; there after mx_tmem_wait_ld
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

__device__ __forceinline__ float finish(const SomeArgs& a, float y, float up) {
    if (a.gated) y = a.out_dtype == RDL_F32 ? rdl_gated(y, up, a.activation, a.act_param) : rdl_gated_near(y, up, a.activation, a.act_param);
    else if (a.activation >= 16) y = rdl_unary(y, a.activation);
    if (a.softcap > 0.f) y = a.softcap * tanhf(y / a.softcap);
    return y;
}

__global__ void __launch_bounds__(THREADS, 1) mx_some_rows_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_xs,
                                                                  const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_ws,
                                                                  const __grid_constant__ SomeArgs a) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) unsigned long long full_bar[MAX_STAGES], empty_bar[MAX_STAGES], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up;
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;      // the compiler may know it uniform
    const int rank = a.split > 1 ? (int)(blockIdx.x % a.split) : 0;
    const int first_tile = blockIdx.x / a.split, tile_step = gridDim.x / a.split;
    const int b0 = min(rank * a.slice_blocks, a.blocks), b1 = min(b0 + a.slice_blocks, a.blocks);
    const uint32_t tmem_cols = a.split > 1 ? CLUSTER_TMEM_COLS : TMEM_COLS, scales_at = a.split > 1 ? ROWS : 2 * ROWS;
    // shared memory: of each stage codes and rows | of each stage the scales of both
    const uint32_t ring_s = mx_smem(smem), scales_s = ring_s + (uint32_t)(a.stages * 2 * MX_TILE_BYTES);
    {
        const int t = threadIdx.x;
        if (t < MAX_STAGES) { mx_bar_init(mx_smem(&full_bar[t]), 1); mx_bar_init(mx_smem(&empty_bar[t]), 1); }
        else if (t < MAX_STAGES + 2) { mx_bar_init(mx_smem(&acc_full[t - MAX_STAGES]), 1); mx_bar_init(mx_smem(&acc_empty[t - MAX_STAGES]), EPI / 32); }
        else if (t == MAX_STAGES + 2) gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(mx_smem(&tmem_slot)), "r"(tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    mx_fence_before();
    __syncthreads();
    mx_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
    volatile int* gave_up_v = &gave_up;
    bool ok = true;

    if (warp == 0) {
        // ---- loader ----
        auto weights = [&](int s, int tile, int kb, uint32_t extra) {
            const uint32_t full = mx_smem(&full_bar[s]), at = ring_s + (uint32_t)(s * 2 * MX_TILE_BYTES);
            mx_bar_expect(full, STAGE_TX + extra);
            mx_tma_2d(at, &map_w, 0, (tile * a.blocks + kb) * MX_ROWS, full);
            mx_tma_2d(scales_s + (uint32_t)(s * 2 * MX_SCALE_BYTES), &map_ws, 0, tile * a.blocks + kb, full);
        };
        auto rows = [&](int s, int kb) {
            const uint32_t full = mx_smem(&full_bar[s]), at = ring_s + (uint32_t)(s * 2 * MX_TILE_BYTES);
            load_rows(at + MX_TILE_BYTES, &map_x, kb * MX_BLOCK, full);
            mx_tma_2d(scales_s + (uint32_t)(s * 2 * MX_SCALE_BYTES + MX_SCALE_BYTES), &map_xs, 0, kb, full);
        };
        const int early = first_tile < a.tiles ? min(a.stages, b1 - b0) : 0;             // blocks whose weights need not wait for the rows
        for (int i = 0; i < early; ++i) {
            if (mx_elect()) weights(i, first_tile, b0 + i, i == 0 ? (uint32_t)a.test_extra_tx : 0u);
            __syncwarp();
        }
        rdl_grid_wait();
        rdl_grid_launch_dependents();
        for (int i = 0; i < early; ++i) {
            if (mx_elect()) rows(i, b0 + i);
            __syncwarp();
        }
        int s = early == a.stages ? 0 : early;
        uint32_t parity = early == a.stages ? 0 : 1;         // places that were never used are free
        for (int tile = first_tile; tile < a.tiles && ok; tile += tile_step) {
            for (int kb = tile == first_tile ? b0 + early : b0; kb < b1; ++kb) {
                if (!mx_warp_wait(mx_smem(&empty_bar[s]), parity, a.wait_cycles, gave_up_v)) { ok = false; break; }
                if (mx_elect()) { weights(s, tile, kb, 0); rows(s, kb); }
                __syncwarp();
                if (++s == a.stages) { s = 0; parity ^= 1; }
            }
        }
    } else if (warp == 1) {
        // ---- scales to tensor memory, and the products ----
        rdl_grid_wait();                                     // as the rows do: the waits here count from then on
        int s = 0, lt = 0, scale_buf = 0;
        uint32_t parity = 0;
        for (int tile = first_tile; tile < a.tiles && ok; tile += tile_step, ++lt) {
            const int buf = lt & 1;
            if (!mx_warp_wait(mx_smem(&acc_empty[buf]), ((lt >> 1) & 1) ^ 1, a.wait_cycles, gave_up_v)) { ok = false; break; }
            mx_fence_after();
            for (int kb = b0; kb < b1; ++kb) {
                if (!mx_warp_wait(mx_smem(&full_bar[s]), parity, a.wait_cycles, gave_up_v)) { ok = false; break; }
                mx_fence_after();
                if (mx_elect()) {
                    const uint32_t sa = tmem + scales_at + (uint32_t)scale_buf * 8, sb = sa + 4, at = ring_s + (uint32_t)(s * 2 * MX_TILE_BYTES);
                    const uint64_t sc = mx_scale_desc(scales_s + (uint32_t)(s * 2 * MX_SCALE_BYTES));
                    copy_scales(sa, sc);
                    copy_scales(sb, sc + (MX_SCALE_BYTES >> 4));
                    const uint64_t ad = mx_operand_desc(at), bd = ad + (MX_TILE_BYTES >> 4);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_mx(tmem + buf * ROWS, ad + (uint32_t)(k * 2), bd + (uint32_t)(k * 2), mx_idesc(MX_E2M1, MX_E4M3, MX_ROWS, ROWS, k), sa, sb, kb != b0 || k != 0);
                    commit(mx_smem(&empty_bar[s]));
                }
                __syncwarp();
                scale_buf = (scale_buf + 1) & (SCALE_BUFS - 1);
                if (++s == a.stages) { s = 0; parity ^= 1; }
            }
            if (ok && mx_elect()) commit(mx_smem(&acc_full[buf]));
            __syncwarp();
        }
    } else {
        // ---- the sums: warp q of four has weight rows 32 q + lane of a tile; two warps share them, 64 of the rows each ----
        rdl_grid_wait();
        const int q = warp & 3, half = (warp - 2) >> 2, pitch = sums_pitch(a.M);
        int lt = 0;
        for (int tile = first_tile; tile < a.tiles; tile += tile_step, ++lt) {
            const int buf = lt & 1;
            if (!mx_bar_wait(mx_smem(&acc_full[buf]), (lt >> 1) & 1, a.wait_cycles, gave_up_v)) ok = false;
            mx_fence_after();
            // where this lane's sums go: of a cluster, to the block that adds up its output
            const int r = 32 * q + lane, o = a.gated ? (r >> 5) * 16 + (r & 15) : r, owner = o / a.share;
            const int outs = a.gated ? 2 * a.share : a.share, at = a.gated ? (o - owner * a.share) * 2 + ((r >> 4) & 1) : o - owner * a.share;
            uint32_t to = 0;
            if (a.split > 1) {
                cluster_arrive();
                cluster_wait();                              // every block's products are done: what was its ring is free
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(ring_s), "r"(owner));
                to += (uint32_t)((rank * outs + at) * pitch) * 4;
            }
            const int n = a.gated ? tile * (MX_ROWS / 2) + 16 * q + lane : tile * MX_ROWS + r;
            for (int l0 = 8 * half; l0 < 32 && 4 * l0 < a.M; l0 += 16) {
                uint32_t v[4][8];                            // row 4 (l0 + j) + c
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld8(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * ROWS + 32 * c + l0), v[c]);
                mx_tmem_wait_ld();
                if (b0 >= b1) {                              // no columns here: no product has written the accumulator
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[c][j] = 0u;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int m = 4 * (l0 + j);
                    if (m >= a.M) break;
                    if (a.split > 1) {
                        asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + (uint32_t)m * 4), "r"(v[0][j]), "r"(v[1][j]), "r"(v[2][j]), "r"(v[3][j]) : "memory");
                    } else {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const float y = __uint_as_float(v[c][j]), up = a.gated ? __shfl_down_sync(0xffffffffu, y, 16) : 0.f;
                            if (m + c < a.M && n < a.N && (!a.gated || lane < 16)) rdl_store(a.out, (long long)(m + c) * a.N + n, a.out_dtype, finish(a, y, up));
                        }
                    }
                }
            }
            mx_fence_before();
            __syncwarp();
            if (lane == 0) mx_bar_arrive(mx_smem(&acc_empty[buf]));
        }
    }
    if (!ok && a.status) atomicExch(a.status, RDL_FAULT_MX_SOME);
    if (a.split > 1) {
        __syncwarp();
        if (warp < 2) {                                      // the barrier the others have behind them
            cluster_arrive();
            cluster_wait();
        }
        cluster_arrive();
        cluster_wait();                                      // every block's sums are where they are added up
        if (warp >= 2) {
            const int tid = threadIdx.x - 64, per_tile = a.gated ? MX_ROWS / 2 : MX_ROWS, outs = a.gated ? 2 * a.share : a.share;
            const int pitch = sums_pitch(a.M), mine = min(a.share, per_tile - rank * a.share);      // outputs this block adds up (none: negative)
            const float* y = reinterpret_cast<const float*>(smem);
            // a thread adds up four neighbouring rows of one output; neighbouring threads have neighbouring outputs
            for (int idx = tid; idx < (a.M + 3) / 4 * a.share; idx += EPI) {
                const int m = idx / a.share * 4, o = idx % a.share, n = first_tile * per_tile + rank * a.share + o;
                if (o >= mine || n >= a.N) continue;
                const float4* ys = reinterpret_cast<const float4*>(y + (a.gated ? 2 * o : o) * pitch + m);
                const int step = outs * pitch / 4;
                float4 sum = make_float4(0.f, 0.f, 0.f, 0.f), up = sum;
#pragma unroll
                for (int s = 0; s < 8; ++s) {
                    if (s >= a.split) break;
                    const float4 v = ys[s * step];
                    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
                    if (a.gated) {
                        const float4 u = ys[s * step + pitch / 4];
                        up.x += u.x; up.y += u.y; up.z += u.z; up.w += u.w;
                    }
                }
                const float v[4] = {sum.x, sum.y, sum.z, sum.w}, u[4] = {up.x, up.y, up.z, up.w};
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (m + c < a.M) rdl_store(a.out, (long long)(m + c) * a.N + n, a.out_dtype, finish(a, v[c], u[c]));
            }
        }
    }
    mx_fence_before();
    __syncthreads();
    if (*gave_up_v) {                    // behind the barrier: whichever warp gave up, the loader has asked for its last copies by now
        rdl_drain_copies();
        __syncwarp();
    }
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols) : "memory");
}

}  // namespace

extern "C" int rdl_mx_some_rows(void* out, int out_dtype, const void* x, const void* row_scales, const void* weight, int m,
                                int activation, float act_param, float softcap, int* status, void* stream) {
    const Mx4Matrix* w = (const Mx4Matrix*)weight;
    RDL_REQUIRE(w && w->codes, "mx_some_rows: missing weight");
    RDL_REQUIRE(m >= 0 && m <= ROWS, "mx_some_rows: %d rows, at most %d are supported", m, ROWS);
    if (m == 0) return 0;
    RDL_REQUIRE(out && x && row_scales, "mx_some_rows: missing operand");
    RDL_REQUIRE(rdl_valid_dtype(out_dtype), "mx_some_rows: bad output dtype %d", out_dtype);
    RDL_REQUIRE((uintptr_t)x % 16 == 0 && (uintptr_t)row_scales % 16 == 0, "mx_some_rows: the rows must start on 16-byte boundaries");
    RDL_REQUIRE(!w->gated || rdl_gated_known(activation), "mx_some_rows: unknown activation %d", activation);
    RDL_REQUIRE(softcap >= 0.f, "mx_some_rows: soft-cap must not be negative");
    const long long blocks = w->blocks, rows4 = (m + 3LL) / 4 * 4;
    MxRowsMaps maps;
    if (int e = mx_rows_maps(&maps, x, row_scales, blocks, rows4)) return e;
    SomeArgs a{};
    a.out = out; a.out_dtype = out_dtype;
    a.M = m; a.N = w->gated ? w->rows / 2 : w->rows; a.blocks = w->blocks; a.tiles = w->tiles;
    a.gated = w->gated; a.activation = activation; a.act_param = act_param; a.softcap = softcap;
    a.wait_cycles = rdl_wait_cycles_for(RDL_FAULT_MX_SOME); a.test_extra_tx = rdl_test_extra_tx_for(RDL_FAULT_MX_SOME);
    a.status = status;
    const int sms = rdl_sm_count();
    a.split = mx_split(a.tiles, a.blocks, sms);
    a.share = ((a.gated ? MX_ROWS / 2 : MX_ROWS) + a.split - 1) / a.split;
    a.slice_blocks = (a.blocks + a.split - 1) / a.split;
    // no deeper than the block's work, but room for a cluster's sums: what shared memory is left lets the next kernel's blocks begin
    const int turns = a.split > 1 ? 1 : (a.tiles + sms - 1) / sms, sums = a.split > 1 ? OUTS_MOST * sums_pitch(m) * 4 : 0;
    a.stages = (long long)turns * a.slice_blocks < MAX_STAGES ? turns * a.slice_blocks : MAX_STAGES;
    if (a.stages * STAGE_BYTES < sums) a.stages = (sums + STAGE_BYTES - 1) / STAGE_BYTES;
    if (a.split > 1 && a.stages < CLUSTER_STAGES) a.stages = CLUSTER_STAGES;
    const int smem = 1024 + a.stages * STAGE_BYTES;
    cudaStream_t st = (cudaStream_t)stream;
    RDL_CUDA(rdl_allow_shared<mx_some_rows_kernel>(smem), "mx_some_rows");
    const int grid = a.split > 1 ? a.tiles * a.split : (a.tiles < sms ? a.tiles : sms);
    RDL_CHECK_EX(rdl_launch_cluster(mx_some_rows_kernel, dim3(grid), dim3(THREADS), a.split, (size_t)smem, st, maps.values, maps.scales, w->codes_map, w->scales_map, a), "mx_some_rows");
    return 0;
}
