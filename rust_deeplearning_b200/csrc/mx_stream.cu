// Few rows times a 4-bit weight matrix (microscaling.cuh):  out[m, n] = epilogue(sum_k x[m, k] w[n, k]),  m <= 16.
//
// Decode: bound by the bytes of the weights, 4.25 bits each, which are read once.  Eight warps multiply and a ninth copies
// (cp.async.bulk, a ring of tiles behind mbarriers; it reads weights only, so it starts while the kernel before is
// still running).  A unit of work is 16 weight rows (the gated form: 16 gate rows and the 16 up rows of the same outputs) times the
// block's slice of the columns; a warp takes every eighth group of 32 columns of it.
//
// One ldmatrix hands a lane eight codes (a 32-bit word) of a row of a group, where the four lanes of a row share the
// group's 16 bytes; cvt turns them into four pairs of f16, which are the operands of two mma.m16n8k16 with the columns taken in the same
// order on both sides.  The two products of a group are summed on their own and join the warp's sum times the group's scale
// in float, so a scale costs one multiply-add a result and codes enter the tensor core as they are: exactly.
//
// The rows enter as f16 with one power of two a row and slice that brings its largest value below 2^15.  A bfloat16 or e4m3 value has
// at most 8 bits, so it is exact above 2^-29 of the row's largest and off by at most 2^-40 of that below: far less than the
// rounding of a float sum.  A float32 value enters as two f16 (the second holds what the first leaves, times 2^11): 22 bits.
//
// The columns are cut into slices where the rows of a slice do not fit shared memory; a slice's sums go to scratch in float and
// a second kernel adds them up, slice by slice in order.
#include <cuda_fp16.h>

#include "activations.cuh"
#include "api.h"
#include "launch.cuh"
#include "microscaling.cuh"

namespace {

constexpr int WARPS = 8, THREADS = (WARPS + 1) * 32;
constexpr int X_BYTES = 80 * 1024;               // most shared memory the rows of a slice take
constexpr int MAX_STAGES = 8;
constexpr int TILE_BLOCKS = 10;                  // most blocks of 128 columns of a tile

struct StreamArgs {
    const void* x; int x_kind;                   // RDL_F32, RDL_BF16, or RDL_MX8: values and row_scales
    const uint8_t* row_scales;
    const uint8_t* codes; const uint8_t* scales;
    void* out; int out_dtype;
    float* partial;                              // [slices][M][weight rows]; NULL: one slice
    int M, N, K;                                 // N: outputs (gated: of each half)
    int blocks, padded_rows;                     // blocks of 128 columns; the rows' padded count (RDL_MX8)
    int half_padded;                             // gated: weight row where the up rows begin
    int slices, slice_blocks, tile_blocks, stages;
    int activation; float act_param, softcap;
    long long wait_cycles; int test_extra_tx;
    int* status;
};

__device__ __forceinline__ void bar_init(uint32_t bar, int count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// false if the phase did not complete in time, or if another warp of the block has given up
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, long long limit, volatile int* gave_up) {
    if (*gave_up) return false;
    if (bar_try(bar, parity)) return true;
    const long long t0 = clock64();
    while (!bar_try(bar, parity)) {
        if (*gave_up) return false;
        if (clock64() - t0 > limit) { *gave_up = 1; return false; }
    }
    return true;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar, unsigned long long policy) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar), "l"(policy) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A tile in shared memory: 16 MT rows of codes, each tile_blocks * 64 bytes and 16 more apart (eight rows' 16-byte pieces then lie in
// eight different groups of banks), then their scales, 64 bytes a block and 16 rows.
__host__ __device__ constexpr int row_pitch(int tile_blocks) { return tile_blocks * 64 + 16; }
__host__ __device__ constexpr int tile_bytes(int mt, int tile_blocks) { return (16 * mt * row_pitch(tile_blocks) + mt * tile_blocks * 64 + 127) / 128 * 128; }
// The rows in shared memory: f16, 64 bytes more than the slice's columns apart (neighbouring rows' 64-byte pieces lie in different banks)
__host__ __device__ constexpr int x_pitch(int slice_blocks) { return slice_blocks * MX_BLOCK * 2 + 64; }

// NT: 8 rows each; GATED: 16 gate and 16 up rows a unit, else 16 rows; PARTS: f16 numbers a value enters as
template <int NT, bool GATED, int PARTS>
__global__ void __launch_bounds__(THREADS, 2) mx_stream_kernel(const __grid_constant__ StreamArgs a) {
    constexpr int MT = GATED ? 2 : 1;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(8) unsigned long long full_bar[MAX_STAGES], empty_bar[MAX_STAGES];
    __shared__ float partial[WARPS][MT][NT][16 * 8];
    __shared__ float row_factor[NT * 8];
    __shared__ int gave_up;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int slice = blockIdx.x % a.slices, first_unit = blockIdx.x / a.slices, unit_step = gridDim.x / a.slices;
    const int n_units = (a.N + MX_UNIT - 1) / MX_UNIT;
    const int b0 = slice * a.slice_blocks, b1 = min(b0 + a.slice_blocks, a.blocks);
    const int pitch = row_pitch(a.tile_blocks), stage_bytes = tile_bytes(MT, a.tile_blocks), xp = x_pitch(a.slice_blocks);
    const uint32_t x_s = (uint32_t)__cvta_generic_to_shared(smem), tiles_s = x_s + (uint32_t)(NT * 8 * PARTS * xp);
    const uint32_t full_s = (uint32_t)__cvta_generic_to_shared(full_bar), empty_s = (uint32_t)__cvta_generic_to_shared(empty_bar);
    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int s = 0; s < a.stages; ++s) {
            bar_init(full_s + 8 * s, 1);
            bar_init(empty_s + 8 * s, WARPS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    volatile int* gave_up_v = &gave_up;

    if (warp == WARPS) {
        // ---- the copying warp: lane r brings row r of a tile, and lanes 0 (and 1) the scales of 16 rows ----
        int s = 0;
        uint32_t round = 0;
        bool first_copy = true;
        unsigned long long policy;                        // read once a step: first to leave L2
        asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
        for (int unit = first_unit; unit < n_units && !*gave_up_v; unit += unit_step) {
            const long long row0 = (long long)unit * MX_UNIT;
            for (int b = b0; b < b1; b += a.tile_blocks) {
                if (round > 0 && !bar_wait(empty_s + 8 * s, (round & 1) ^ 1, a.wait_cycles, gave_up_v)) break;
                const int nb = min(a.tile_blocks, b1 - b);
                const uint32_t bytes = (uint32_t)nb * 64u, tile = tiles_s + (uint32_t)(s * stage_bytes);
                if (lane == 0) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    bar_expect(full_s + 8 * s, bytes * (uint32_t)(17 * MT) + (first_copy ? (uint32_t)a.test_extra_tx : 0u));
                }
                __syncwarp();
                if (lane < 16 * MT) {
                    const long long row = (lane < 16 ? row0 : a.half_padded + row0 - 16) + lane;
                    bulk_load(tile + (uint32_t)(lane * pitch), a.codes + (row * a.blocks + b) * 64, bytes, full_s + 8 * s, policy);
                }
                if (lane < MT) {
                    const long long u = lane == 0 ? unit : a.half_padded / MX_UNIT + unit;
                    bulk_load(tile + (uint32_t)(16 * MT * pitch + lane * a.tile_blocks * 64), a.scales + (u * a.blocks + b) * 64, bytes, full_s + 8 * s, policy);
                }
                first_copy = false;
                if (++s == a.stages) { s = 0; ++round; }
            }
        }
    } else {
        // ---- the multiplying warps; first the rows of the slice, a warp a row ----
        rdl_grid_wait();
        rdl_grid_launch_dependents();
        const int c0 = b0 * MX_BLOCK, cols = (b1 - b0) * MX_BLOCK;
        for (int m = warp; m < NT * 8; m += WARPS) {
            const bool on = m < a.M;
            auto load = [&](int c, float (&v)[4]) {       // four columns from column c of the slice
                const int k = c0 + c;
                if (!on) { v[0] = v[1] = v[2] = v[3] = 0.f; return; }
                if (a.x_kind == RDL_MX8) {
                    const uint32_t raw = *reinterpret_cast<const uint32_t*>((const uint8_t*)a.x + (long long)m * a.blocks * MX_BLOCK + k);
                    const float sc = mx_scale(a.row_scales[((long long)(k / MX_BLOCK) * a.padded_rows + m) * 4 + k % MX_BLOCK / MX_GROUP]);
                    const uint32_t lo = mx_from_e4m3(raw & 0xffffu), hi = mx_from_e4m3(raw >> 16);
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&lo)), g = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                    v[0] = f.x * sc; v[1] = f.y * sc; v[2] = g.x * sc; v[3] = g.y * sc;
                } else {
                    const long long base = (long long)m * a.K;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = k + i < a.K ? rdl_load(a.x, base + k + i, a.x_kind) : 0.f;
                }
            };
            uint32_t top = 0;                             // the largest finite magnitude, as bits
            for (int c = lane * 4; c < cols; c += 128) {
                float v[4];
                load(c, v);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t bits = __float_as_uint(v[i]) & 0x7fffffffu;
                    if (bits < 0x7f800000u) top = max(top, bits);
                }
            }
            top = __reduce_max_sync(0xffffffffu, top);
            const int up = min(14 - ((int)(top >> 23) - 127), 127);       // x 2^up is below 2^15
            const float factor = ldexpf(1.f, up);
            if (lane == 0) row_factor[m] = ldexpf(1.f, -up);
            unsigned char* xrow = smem + m * xp;
            for (int c = lane * 4; c < cols; c += 128) {
                float v[4];
                load(c, v);
                __half h[4], l[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float y = v[i] * factor;
                    h[i] = __float2half_rn(y);
                    if (PARTS == 2) l[i] = isfinite(y) ? __float2half_rn((y - __half2float(h[i])) * 2048.f) : __float2half_rn(0.f);
                }
                *reinterpret_cast<uint2*>(xrow + c * 2) = *reinterpret_cast<const uint2*>(h);
                if (PARTS == 2) *reinterpret_cast<uint2*>(xrow + NT * 8 * xp + c * 2) = *reinterpret_cast<const uint2*>(l);
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory");

        const int g = lane >> 2, t = lane & 3, tid = threadIdx.x;
        // ldmatrix: lanes 0 to 15 give the rows of the first group's 16 bytes, lanes 16 to 31 those of the second
        const uint32_t lane_row = (uint32_t)((lane & 15) * pitch + (lane >> 4) * 16);
        int s = 0;
        uint32_t round = 0;
        for (int unit = first_unit; unit < n_units; unit += unit_step) {
            float acc[MT][NT][4];
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.f;
            for (int b = b0; b < b1; b += a.tile_blocks) {
                bar_wait(full_s + 8 * s, round & 1, a.wait_cycles, gave_up_v);
                const int pairs = min(a.tile_blocks, b1 - b) * 2;           // of groups
                const uint32_t tile = tiles_s + (uint32_t)(s * stage_bytes);
                for (int p = warp; p < pairs; p += WARPS) {
                    uint32_t w[MT][4];                                      // (row g, first group), (row g + 8), (row g, second), (row g + 8)
                    uint32_t sc[MT][2];                                     // scale codes of both groups: rows g and g + 8
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                                     : "=r"(w[i][0]), "=r"(w[i][1]), "=r"(w[i][2]), "=r"(w[i][3]) : "r"(tile + (uint32_t)(i * 16 * pitch + p * 32) + lane_row));
                        const uint32_t sa = tile + (uint32_t)(16 * MT * pitch + i * a.tile_blocks * 64 + (p >> 1) * 64 + g * 4 + (p & 1) * 2);
                        uint16_t s0, s1;
                        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(s0) : "r"(sa));
                        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(s1) : "r"(sa + 32));
                        sc[i][0] = s0; sc[i][1] = s1;
                    }
                    const uint32_t xa = x_s + (uint32_t)(((b - b0) * MX_BLOCK + p * 64 + t * 8) * 2 + g * xp);
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        uint4 xb[PARTS][NT];
#pragma unroll
                        for (int e = 0; e < PARTS; ++e)
#pragma unroll
                            for (int j = 0; j < NT; ++j)
                                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(xb[e][j].x), "=r"(xb[e][j].y), "=r"(xb[e][j].z), "=r"(xb[e][j].w)
                                             : "r"(xa + (uint32_t)(q * 64 + (e * NT * 8 + j * 8) * xp)));
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            uint32_t lo[4], hi[4];
                            mx_from_e2m1(w[i][2 * q], lo);
                            mx_from_e2m1(w[i][2 * q + 1], hi);
                            const uint32_t f0[4] = {lo[0], hi[0], lo[1], hi[1]}, f1[4] = {lo[2], hi[2], lo[3], hi[3]};
                            const float s0 = mx_scale(q ? sc[i][0] >> 8 : sc[i][0] & 255u), s1 = mx_scale(q ? sc[i][1] >> 8 : sc[i][1] & 255u);
#pragma unroll
                            for (int j = 0; j < NT; ++j) {
                                float d[4] = {0.f, 0.f, 0.f, 0.f};
                                mma_f16(d, f0, xb[0][j].x, xb[0][j].y);
                                mma_f16(d, f1, xb[0][j].z, xb[0][j].w);
                                if (PARTS == 2) {
                                    float l[4] = {0.f, 0.f, 0.f, 0.f};
                                    mma_f16(l, f0, xb[PARTS - 1][j].x, xb[PARTS - 1][j].y);
                                    mma_f16(l, f1, xb[PARTS - 1][j].z, xb[PARTS - 1][j].w);
#pragma unroll
                                    for (int v = 0; v < 4; ++v) d[v] = fmaf(l[v], 1.f / 2048.f, d[v]);
                                }
                                acc[i][j][0] = fmaf(d[0], s0, acc[i][j][0]);
                                acc[i][j][1] = fmaf(d[1], s0, acc[i][j][1]);
                                acc[i][j][2] = fmaf(d[2], s1, acc[i][j][2]);
                                acc[i][j][3] = fmaf(d[3], s1, acc[i][j][3]);
                            }
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) bar_arrive(empty_s + 8 * s);
                if (++s == a.stages) { s = 0; ++round; }
            }
            // element v of a lane: weight row g + 8 (v >> 1), activation row 2 t + (v & 1)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int v = 0; v < 4; ++v) partial[warp][i][j][(2 * t + (v & 1)) * 16 + g + 8 * (v >> 1)] = acc[i][j][v];
            asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory");
            for (int idx = tid; idx < NT * 8 * 16; idx += WARPS * 32) {
                const int m = idx >> 4, r = idx & 15, n = unit * MX_UNIT + r;
                if (m >= a.M || n >= a.N) continue;
                float y[MT];
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    y[i] = 0.f;
#pragma unroll
                    for (int w = 0; w < WARPS; ++w) y[i] += partial[w][i][m >> 3][(m & 7) * 16 + r];
                    y[i] *= row_factor[m];
                }
                if (a.partial) {
#pragma unroll
                    for (int i = 0; i < MT; ++i) a.partial[((long long)slice * a.M + m) * (MT * a.N) + i * a.N + n] = y[i];
                    continue;
                }
                float v = GATED ? rdl_gated(y[0], y[MT - 1], a.activation, a.act_param) : y[0];
                if (!GATED && a.activation >= 16) v = rdl_unary(v, a.activation);
                if (a.softcap > 0.f) v = a.softcap * tanhf(v / a.softcap);
                rdl_store(a.out, (long long)m * a.N + n, a.out_dtype, v);
            }
            asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory");      // the partial sums are free again
        }
    }
    if (*gave_up_v) {
        if (a.status && lane == 0) atomicExch(a.status, RDL_FAULT_MX_STREAM);
        if (warp == WARPS)                                // copies that are on their way still write to this block's shared memory
            for (const long long t0 = clock64(); clock64() - t0 < RDL_COPY_DRAIN_CYCLES;) {}
    }
}

// the slices' sums in order, and the epilogue
template <bool GATED>
__global__ void __launch_bounds__(256) mx_stream_finish_kernel(const __grid_constant__ StreamArgs a) {
    constexpr int MT = GATED ? 2 : 1;
    rdl_grid_wait();
    rdl_grid_launch_dependents();
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x, total = (long long)a.M * a.N;
    if (i >= total) return;
    const int m = (int)(i / a.N), n = (int)(i - (long long)m * a.N);
    float y[MT];
#pragma unroll
    for (int h = 0; h < MT; ++h) {
        y[h] = 0.f;
        for (int s = 0; s < a.slices; ++s) y[h] += a.partial[((long long)s * a.M + m) * (MT * a.N) + h * a.N + n];
    }
    float v = GATED ? rdl_gated(y[0], y[MT - 1], a.activation, a.act_param) : y[0];
    if (!GATED && a.activation >= 16) v = rdl_unary(v, a.activation);
    if (a.softcap > 0.f) v = a.softcap * tanhf(v / a.softcap);
    rdl_store(a.out, i, a.out_dtype, v);
}

int rows_of(int m) { return m <= 8 ? 1 : 2; }
int slice_limit(int m, int x_kind) { return X_BYTES / (rows_of(m) * 8 * (x_kind == RDL_F32 ? 2 : 1) * MX_BLOCK * 2); }

template <int NT, bool GATED, int PARTS>
cudaError_t launch(StreamArgs a, cudaStream_t st) {
    constexpr int MT = GATED ? 2 : 1;
    const int x_bytes = NT * 8 * PARTS * x_pitch(a.slice_blocks);
    // tiles of a slice, of one size and about 10 to 20 KB
    const int most = GATED ? TILE_BLOCKS / 2 : TILE_BLOCKS;
    const int tiles = (a.slice_blocks + most - 1) / most;
    a.tile_blocks = (a.slice_blocks + tiles - 1) / tiles;
    const int stage = tile_bytes(MT, a.tile_blocks);
    // two blocks a multiprocessor where each has room for three tiles beside its rows, else one with twice the ring
    const int fixed = 2048 + WARPS * MT * NT * 512;      // static shared memory and what the system takes
    const int units = (a.N + MX_UNIT - 1) / MX_UNIT, sms = rdl_sm_count();
    int per_sm = x_bytes + 3 * stage + fixed <= 113 * 1024 ? 2 : 1;
    if ((long long)units * a.slices <= sms) per_sm = 1;
    const int room = (per_sm == 2 ? 113 : 225) * 1024 - fixed - x_bytes;
    a.stages = room / stage;
    if (a.stages > MAX_STAGES) a.stages = MAX_STAGES;
    if (a.stages < 2) return cudaErrorInvalidConfiguration;
    const int smem = x_bytes + a.stages * stage;
    cudaError_t e = rdl_allow_shared<mx_stream_kernel<NT, GATED, PARTS>>(smem);
    if (e != cudaSuccess) return e;
    int columns = per_sm * sms / a.slices;                // blocks that share a slice
    if (columns < 1) columns = 1;
    if (columns > units) columns = units;
    e = rdl_launch(mx_stream_kernel<NT, GATED, PARTS>, dim3(columns * a.slices), dim3(THREADS), (size_t)smem, st, a);
    if (e != cudaSuccess || !a.partial) return e;
    return rdl_launch(mx_stream_finish_kernel<GATED>, dim3((unsigned)(((long long)a.M * a.N + 255) / 256)), dim3(256), 0, st, a);
}

}  // namespace

// slices of the columns a call with these sizes is cut into; above 1 it needs scratch of slices * m * (gated ? 2 n : n) floats
extern "C" int rdl_mx_stream_slices(int m, int k, int x_kind) {
    if (m <= 0 || m > 16 || k <= 0) return 1;
    const int limit = slice_limit(m, x_kind), blocks = mx_blocks(k);
    return (blocks + limit - 1) / limit;
}

extern "C" int rdl_mx_stream(void* out, int out_dtype, const void* x, int x_kind, const void* row_scales, const void* codes, const void* scales,
                             int m, int n, int k, int gated, int activation, float act_param, float softcap, float* scratch, long long scratch_floats,
                             int* status, void* stream) {
    RDL_REQUIRE(out && x && codes && scales, "mx_stream: missing operand");
    RDL_REQUIRE(rdl_valid_dtype(out_dtype), "mx_stream: bad output dtype %d", out_dtype);
    RDL_REQUIRE(rdl_valid_dtype(x_kind) || (x_kind == RDL_MX8 && row_scales), "mx_stream: bad rows (kind %d)", x_kind);
    RDL_REQUIRE(m >= 0 && m <= 16, "mx_stream: %d rows, at most 16 are supported", m);
    RDL_REQUIRE(n > 0 && k > 0, "mx_stream: n=%d, k=%d", n, k);
    RDL_REQUIRE((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 16 == 0, "mx_stream: the weight must start on 16-byte boundaries");
    RDL_REQUIRE(x_kind != RDL_MX8 || (uintptr_t)x % 4 == 0, "mx_stream: the rows must start on a 4-byte boundary");
    RDL_REQUIRE(!gated || rdl_gated_known(activation), "mx_stream: unknown activation %d", activation);
    RDL_REQUIRE(softcap >= 0.f, "mx_stream: soft-cap must not be negative");
    if (m == 0) return 0;
    StreamArgs a{};
    a.x = x; a.x_kind = x_kind; a.row_scales = (const uint8_t*)row_scales;
    a.codes = (const uint8_t*)codes; a.scales = (const uint8_t*)scales;
    a.out = out; a.out_dtype = out_dtype;
    a.M = m; a.N = n; a.K = k;
    a.blocks = mx_blocks(k); a.padded_rows = (m + 3) / 4 * 4;
    a.half_padded = gated ? (n + MX_UNIT - 1) / MX_UNIT * MX_UNIT : 0;
    a.slices = rdl_mx_stream_slices(m, k, x_kind);
    a.slice_blocks = (a.blocks + a.slices - 1) / a.slices;
    a.slices = (a.blocks + a.slice_blocks - 1) / a.slice_blocks;          // none is empty
    a.activation = activation; a.act_param = act_param; a.softcap = softcap;
    a.wait_cycles = rdl_wait_cycles_for(RDL_FAULT_MX_STREAM); a.test_extra_tx = rdl_test_extra_tx_for(RDL_FAULT_MX_STREAM);
    a.status = status;
    if (a.slices > 1) {
        RDL_REQUIRE(scratch && scratch_floats >= (long long)a.slices * m * (gated ? 2LL * n : n), "mx_stream: %d slices need scratch of %lld floats",
                    a.slices, (long long)a.slices * m * (gated ? 2LL * n : n));
        a.partial = scratch;
    }
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e;
#define RDL_MX_STREAM(NT, PARTS) (e = gated ? launch<NT, true, PARTS>(a, st) : launch<NT, false, PARTS>(a, st))
    if (rows_of(m) == 1) { if (x_kind == RDL_F32) RDL_MX_STREAM(1, 2); else RDL_MX_STREAM(1, 1); }
    else { if (x_kind == RDL_F32) RDL_MX_STREAM(2, 2); else RDL_MX_STREAM(2, 1); }
#undef RDL_MX_STREAM
    RDL_CHECK_EX(e, "mx_stream");
    return 0;
}
