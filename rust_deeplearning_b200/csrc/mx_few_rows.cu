// Few rows times a 4-bit weight matrix (formats: microscaling.cuh):  out[m, n] = epilogue(sum_k x[m, k] w[n, k]),  m <= 16.
//
// Decode: bound by the bytes of the weights, 4.25 bits each, read once.  Anything a thread does per weight would cost more than the
// weight's transfer, so no thread touches one: TMA brings codes to shared memory in the form the block-scaled tcgen05 product reads
// (mx_tensor.cuh), with 128 weight rows as its M side and the few rows as its N side.
//
// The rows have to be 8-bit values with a power of two a group, too.  Rows that are in that form enter as they are.  A bfloat16 value
// has 8 significant bits and e4m3 has 4: it enters as the sum of two, itself rounded to four bits and the rest, with a scale 2^4
// smaller.  This is exact for values above 2^-13 of the largest of their group (below it, it is off by at most 2^-21 of that
// largest one).  A float32 value enters as six parts, exact above 2^-13 of the largest, off by at most 2^-37 of that below.  The parts are
// columns of the one product and are added up in its epilogue.  Rows that hold an infinity or a NaN, which parts cannot, or nothing
// but numbers so small that a part's scale would fall below 2^-127, are computed again by plain arithmetic.
//
// Warp 0 loads weights: they depend on nothing an earlier kernel of the step writes, so it starts while that kernel is still running.
// Warp 1 issues scales and products.  Sixteen warps turn the rows into parts (once, where a block's columns fit shared memory; else for
// every tile, into slots that are used in turn), a block of columns after another so that the products can begin; eight of them then take
// finished sums out of tensor memory.  A wide matrix: a block takes 128 rows of weights after another.  One with fewer tiles than
// multiprocessors: a cluster of up to 8 blocks shares a tile, each with its part of the columns, and its blocks send their sums through
// distributed shared memory to the one that adds up that part of the outputs, in rank order.  Every wait is bounded.
//
// Up to 8 bfloat16 rows can have a deferred norm on either side (the algebra: DeferredNormArgs in api.h).  The branch's product writes its
// partial sums a block of the cluster at a time.  In the product behind the norm four warps add them up and see to the stream.  Up to 4
// rows: both halves of the operand are rows of the product, and a row's two sums are joined on their way out of tensor memory, so
// that nothing waits for the partial sums.  5 to 8 rows: that would be 16 rows to make parts of; the halves are joined first, x = s2 (ht + s1 at),
// rounded to bfloat16.  Output projection, gated product, down projection and next projection of a layer with the norms between: width
// 2,304 1 row 28.5 us (29.9 with kernels for the norms), 8 rows 32.7 (34.7); width 3,584 40.9 (45.1), 47.2 (51.3); 4,608 74.7 (79.3), 83.4 (87.6).
//
// The loops that make parts and write results are not unrolled.  In a step this kernel's forms alternate with one another and with other
// kernels, and each starts with instructions that are not at hand: with the loops unrolled a pair of forms took 0.5 to 2.2 us more than
// each of them alone, and now 0 to 0.4.
//
// Measured on the device, one bfloat16 row: 256,000 outputs of 2,304 columns (313 MB) 52.1 us, 6.0 TB/s; 28,672 of 3,584, gated, 14.0 us,
// 3.9 TB/s; 4,096 of 2,304 (5 MB) 5.4 us: there what bounds it is the chain of a launch, the first copy, the products of a block's columns
// and the exchange in the cluster.  16 rows: 58.6, 20.2 and 6.9 us (in 8 bits already: 56.7, 16.2 and 6.0; float32: 172, 39.7 and 8.1).
#include <cuda_fp16.h>

#include "activations.cuh"
#include "api.h"
#include "launch.cuh"
#include "mx_tensor.cuh"

namespace {

// A stage of the ring is STEP blocks of columns: a stage costs the issuing thread a wait beside its products, about as long as those of a block.
// Its blocks' places are filled again one by one (1 row x 2,304, 256,000 outputs 53.7 -> 52.4 us; x 3,584, 28,672 gated 15.0 -> 14.6; rows that
// are in 8 bits already 52.7 -> 54.9).
constexpr int WORKERS = 512, THREADS = 64 + WORKERS, MAX_STAGES = 8, STEP = 2, SCALE_BUFS = 4, MAX_SLOTS = 64, AHEAD_L2 = 4;

struct FewArgs {
    const void* x; const uint8_t* row_scales;
    const uint8_t* codes; const uint8_t* scales;
    void* out; int out_dtype;
    int M, N, K;                                 // N: outputs
    int blocks, row_pad;                         // blocks of 128 columns; the rows' padded count (8-bit rows)
    int tiles, split, slice_blocks, slots, stages;   // slots: blocks of the rows that shared memory holds
    int share;                                   // outputs of a tile that a block of a cluster adds up
    int gated, activation; float act_param, softcap;
    bool vec;                                    // rows lie on 16-byte boundaries
    DeferredNormArgs norm; int src_rows;             // one side of a deferred norm; the rows of which sums are wanted (M: rows of the output)
    long long wait_cycles; int test_extra_tx;
    int* status;
};

__device__ __forceinline__ void tma_codes(uint32_t dst, const CUtensorMap* map, int y, uint32_t bar, unsigned long long policy) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3}], [%4], %5;"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(y), "r"(bar), "l"(policy) : "memory");
}
__device__ __forceinline__ void bulk_scales(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar, unsigned long long policy) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar), "l"(policy) : "memory");
}
__device__ __forceinline__ void ask_l2(const void* src, uint32_t bytes) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(bytes) : "memory");
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
// N accumulator columns of the warp's lanes, as bits; there after mx_tmem_wait_ld
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t* r) {
    static_assert(N == 2 || N == 4 || N == 8, "two, four or eight columns");
    if constexpr (N == 2)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(taddr) : "memory");
    else if constexpr (N == 4)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(taddr) : "memory");
    else
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t map_to_block(uint32_t addr, uint32_t rank) {      // the same place in the shared memory of block `rank`
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}

__device__ __forceinline__ float finish(const FewArgs& a, float y, float up) {
    if (a.gated) y = a.out_dtype == RDL_F32 ? rdl_gated(y, up, a.activation, a.act_param) : rdl_gated_near(y, up, a.activation, a.act_param);
    else if (a.activation >= 16) y = rdl_unary(y, a.activation);
    if (a.softcap > 0.f) y = a.softcap * tanhf(y / a.softcap);
    return y;
}

// ---- eight columns of a row, as they lie and in parts; the four lanes of a group hold neighbouring ones ----
template <int PARTS>
struct Chunk {
    uint32_t w[PARTS == 6 ? 8 : (PARTS == 2 ? 4 : 2)];
    uint32_t code;                               // the group's scale, of 8-bit rows
};

template <int PARTS>
__device__ __forceinline__ void load_chunk(const FewArgs& a, int m, int k, Chunk<PARTS>& d) {
    if constexpr (PARTS == 1) {
        const uint2 v = *reinterpret_cast<const uint2*>((const uint8_t*)a.x + (long long)m * a.blocks * MX_BLOCK + k);
        d.w[0] = v.x; d.w[1] = v.y;
        d.code = a.row_scales[((long long)(k / MX_BLOCK) * a.row_pad + m) * 4 + k % MX_BLOCK / MX_GROUP];
    } else {
        const long long base = (long long)m * a.K + k;
#pragma unroll
        for (int i = 0; i < (PARTS == 6 ? 8 : 4); ++i) d.w[i] = 0;
        if (a.vec) {
            if (k < a.K) {
                const uint4* p = reinterpret_cast<const uint4*>((const char*)a.x + base * (PARTS == 2 ? 2 : 4));
#pragma unroll
                for (int i = 0; i < (PARTS == 6 ? 2 : 1); ++i) *reinterpret_cast<uint4*>(&d.w[4 * i]) = p[i];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (k + e >= a.K) continue;
                if (PARTS == 2) d.w[e >> 1] |= (uint32_t)((const unsigned short*)a.x)[base + e] << (16 * (e & 1));
                else d.w[PARTS == 2 ? 0 : e] = ((const uint32_t*)a.x)[base + e];
            }
        }
    }
}

__device__ __forceinline__ uint32_t raw_load(const void* p, long long i, int dtype) {             // bits now, the value when it is needed
    return dtype == RDL_BF16 ? (uint32_t)((const unsigned short*)p)[i] : ((const uint32_t*)p)[i];
}
__device__ __forceinline__ float raw_value(uint32_t bits, int dtype) { return __uint_as_float(dtype == RDL_BF16 ? bits << 16 : bits); }

// The two halves of the operand behind a deferred norm joined: what the rows stand for, rounded to bfloat16 as a norm's result is
__device__ __forceinline__ float join(float h, float b, float2 r) { return r.y * fmaf(r.x, b, h); }
__device__ __forceinline__ uint32_t join_pair(uint32_t h, uint32_t b, float2 r) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(join(__uint_as_float(h << 16), __uint_as_float(b << 16), r),
                                                   join(__uint_as_float(h & 0xffff0000u), __uint_as_float(b & 0xffff0000u), r));
    return *reinterpret_cast<const uint32_t*>(&v);
}
// A kernel's MODE is 0, RDL_NORM_BRANCH, RDL_NORM_DEFERRED (both halves of the operand are rows of the product) or this (they are joined first).
constexpr int NORM_JOINED = 3;
__host__ __device__ constexpr bool behind_norm(int mode) { return mode == RDL_NORM_DEFERRED || mode == NORM_JOINED; }

constexpr int ROW_FINE = 0, ROW_ZERO = 1, ROW_TINY = 2, ROW_BAD = 3;

// The parts of a chunk as e4m3 bytes, and the scale codes of its group; the four lanes of a group come here together.  A part is what the
// parts before it leave, rounded to four bits, which leaves at most a 2^-4 of the largest: so the next one's scale is 2^4 smaller.
// (Cut off instead of rounded, and not converted back, values below 2^-13 lost up to 2^-17 of the largest; 8 rows x 2,304, 18,432 gated
// outputs took 8.65 us, and 8.7 to 8.9 so.)
template <int PARTS>
__device__ __forceinline__ int make_parts(const Chunk<PARTS>& d, uint2 (&bytes)[PARTS], uint32_t (&code)[PARTS]) {
    if constexpr (PARTS == 1) {
        bytes[0] = make_uint2(d.w[0], d.w[1]);
        code[0] = d.code;
        return ROW_ZERO;
    } else {
        uint32_t top = 0;                                    // magnitudes are in order as integers
        if constexpr (PARTS == 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) top = __vmaxu2(top, d.w[i] & 0x7fff7fffu);
            top = max(top & 0xffff0000u, top << 16);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, d.w[i] & 0x7fffffffu);
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const bool bad = top >= 0x7f800000u;
        const uint32_t c = bad ? 0u : mx8_scale_code(__uint_as_float(top));
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(PARTS == 6 ? d.w[PARTS == 6 ? e : 0] : (e & 1 ? d.w[e >> 1] & 0xffff0000u : d.w[e >> 1] << 16));
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            code[part] = c > 4u * part ? c - 4u * part : 0u;
            const float f = mx_inverse_scale(code[part]);
            bytes[part] = make_uint2(mx_to_e4m3(v[0] * f, v[1] * f, v[2] * f, v[3] * f), mx_to_e4m3(v[4] * f, v[5] * f, v[6] * f, v[7] * f));
            if (part + 1 < PARTS) {                          // what this part leaves, exactly
                const float s = mx_scale(code[part]);
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float2 h = mx_from_e4m3((e < 4 ? bytes[part].x : bytes[part].y) >> (8 * (e & 2)));
                    v[e] = fmaf(-h.x, s, v[e]);
                    v[e + 1] = fmaf(-h.y, s, v[e + 1]);
                }
            }
            if (bad) bytes[part] = make_uint2(0, 0);         // the row is computed again: zeros keep its columns quiet
        }
        return bad ? ROW_BAD : (top == 0 ? ROW_ZERO : (c >= 4u * (PARTS - 1) ? ROW_FINE : ROW_TINY));
    }
}

// PARTS: 1 (8-bit rows), 2 (bfloat16), 6 (float32); R: rows the product has place for; MODE: see above
template <int PARTS, int R, int MODE>
__global__ void __launch_bounds__(THREADS, PARTS == 6 ? 1 : 2) mx_few_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ FewArgs a) {
    constexpr int NB = PARTS * R;                            // columns of the product: part p of row m is column p R + m
    constexpr int X_BLOCK = NB * MX_BLOCK;                   // bytes of a block of 128 columns of the rows
    constexpr int TMEM_COLS = 2 * NB + SCALE_BUFS * 8 <= 128 ? 128 : 256;
    constexpr int AHEAD = PARTS == 6 || MODE == NORM_JOINED ? 2 : 4;                // chunks a lane asks for before it works on the first: two rows each
    constexpr int PIECE_ROWS = 2 * AHEAD, PIECES = STEP * (R / PIECE_ROWS);              // pieces of a group of STEP blocks
    // behind a deferred norm four of the workers see to the sums and to the stream; the others make parts (of 18 blocks of 16 rows, three
    // pieces each, as sixteen would)
    constexpr int SIDE = behind_norm(MODE) ? 4 : 0, TAKERS = WORKERS / 32 - SIDE;
    static_assert(NB % 16 == 0 && 2 * NB + SCALE_BUFS * 8 <= TMEM_COLS, "the sums of two tiles and the scales share tensor memory");
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) unsigned long long full_bar[MAX_STAGES], empty_bar[MAX_STAGES * STEP], acc_full[2], acc_empty[2], x_ready[MAX_SLOTS / STEP], x_free[MAX_SLOTS / STEP];
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up;
    // rows with an infinity or a NaN here; rows with a group too small for its last parts; rows with one that is not
    __shared__ unsigned bad_rows, tiny_rows, fine_rows;
    __shared__ float4 norm_part[SIDE ? SIDE : 1][8];         // the branch's partial sums, a warp's share of the units
    __shared__ float2 row_scale[8];                          // a row's two numbers
    // shared memory: rows | ring of codes | the rows' scales | ring of scales | sums of a cluster's blocks
    const uint32_t x_s = mx_smem(smem), ring_s = x_s + (uint32_t)(a.slots * X_BLOCK);
    const uint32_t xs_s = ring_s + (uint32_t)(a.stages * STEP * MX_TILE_BYTES), ws_s = xs_s + (uint32_t)(a.slots * MX_SCALE_BYTES);
    const uint32_t y_off = (uint32_t)(a.slots * (X_BLOCK + MX_SCALE_BYTES) + a.stages * STEP * (MX_TILE_BYTES + MX_SCALE_BYTES));

    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;      // the compiler may know it uniform
    const int rank = a.split > 1 ? (int)(blockIdx.x % a.split) : 0;
    const int first_tile = blockIdx.x / a.split, tile_step = gridDim.x / a.split;
    const int b0 = min(rank * a.slice_blocks, a.blocks), b1 = min(b0 + a.slice_blocks, a.blocks);
    // the rows lie in slots of STEP blocks: all of them once (they stay for every tile), or as many as there is room for, in turn
    const int groups = (b1 - b0 + STEP - 1) / STEP, x_groups = a.slots / STEP;
    const bool resident = groups <= x_groups;
    {   // every barrier by a thread of its own
        const int t = threadIdx.x;
        if (t < MAX_STAGES) {
            mx_bar_init(mx_smem(&full_bar[t]), STEP);
#pragma unroll
            for (int j = 0; j < STEP; ++j) mx_bar_init(mx_smem(&empty_bar[t * STEP + j]), 1);
        }
        else if (t < MAX_STAGES + 2) { mx_bar_init(mx_smem(&acc_full[t - MAX_STAGES]), 1); mx_bar_init(mx_smem(&acc_empty[t - MAX_STAGES]), 8); }
        else if (t == MAX_STAGES + 2) { gave_up = 0; bad_rows = tiny_rows = fine_rows = 0; }
        else if (t >= 64 && t < 64 + MAX_SLOTS / STEP) { mx_bar_init(mx_smem(&x_ready[t - 64]), PIECES); mx_bar_init(mx_smem(&x_free[t - 64]), 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(mx_smem(&tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    mx_fence_before();
    __syncthreads();
    if (a.split > 1) cluster_arrive();                       // "this block runs"; waited for before anything is stored in another one
    mx_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
    volatile int* gave_up_v = &gave_up;
    bool ok = true;

    if (warp == 0) {
        // ---- weights ----
        if (mx_elect()) {
            unsigned long long policy;                       // read once a step: first to leave L2
            asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
            int s = 0, piece = first_tile * a.blocks + b0;   // place in the ring; block of columns over all tiles
            bool behind = false;                             // the kernel ahead has ended
            uint32_t parity = 1, extra = (uint32_t)a.test_extra_tx;      // the first round finds every place free
            // A short ring keeps too few bytes on their way: L2 is asked for what will be loaded up to AHEAD_L2 stages later (16 rows x 3,584,
            // 28,672 gated outputs, two stages: 24.9 -> 21.8 us in the form of that time; with five stages it costs: 1 row x 2,304, 18,432 outputs 7.1 -> 8.1).
            int ask_tile = a.stages < 4 ? first_tile : a.tiles, ask_kb = b0, asked = 0;
            auto ask = [&]() {
                if (ask_tile >= a.tiles || b0 >= b1) return;
                const int n = min(STEP, b1 - ask_kb);
                const long long at = (long long)ask_tile * a.blocks + ask_kb;
                if (asked >= a.stages) {
                    ask_l2(a.codes + at * (MX_ROWS * MX_BLOCK / 2), (uint32_t)n * (MX_ROWS * MX_BLOCK / 2));
                    ask_l2(a.scales + at * MX_SCALE_BYTES, (uint32_t)n * MX_SCALE_BYTES);
                }
                ++asked;
                ask_kb += n;
                if (ask_kb >= b1) { ask_kb = b0; ask_tile += tile_step; }
            };
#pragma unroll 1
            for (int i = 0; i < a.stages + AHEAD_L2; ++i) ask();
            for (int tile = first_tile; tile < a.tiles && ok; tile += tile_step, piece += (tile_step - 1) * a.blocks + (a.blocks - (b1 - b0))) {
                for (int kb = b0; kb < b1;) {
                    const int n = min(STEP, b1 - kb);
                    const uint32_t full = mx_smem(&full_bar[s]);
#pragma unroll
                    for (int j = 0; j < STEP; ++j) {         // a block's place is filled again as soon as its own products are done
                        if (!mx_bar_wait(mx_smem(&empty_bar[s * STEP + j]), parity, a.wait_cycles, gave_up_v)) { ok = false; break; }
                        if (j >= n) { mx_bar_arrive(full); continue; }
                        mx_bar_expect(full, MX_TILE_TX + MX_SCALE_BYTES + extra);
                        extra = 0;
                        tma_codes(ring_s + (uint32_t)((s * STEP + j) * MX_TILE_BYTES), &map_w, (piece + j) * MX_ROWS, full, policy);
                        bulk_scales(ws_s + (uint32_t)((s * STEP + j) * MX_SCALE_BYTES), a.scales + (long long)(piece + j) * MX_SCALE_BYTES, MX_SCALE_BYTES, full, policy);
                    }
                    if (!ok) break;
                    ask();
                    kb += n;
                    piece += n;
                    if (++s == a.stages) {
                        // the ring is full: waits from here on are for products, which wait for the kernel ahead, and its time is not to count
                        if (!behind) { rdl_grid_wait(); behind = true; }
                        s = 0;
                        parity ^= 1;
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---- scales to tensor memory, and the products ----
        if (mx_elect()) {
            rdl_grid_wait();                                 // as the rows do: the waits here count from then on
            int s = 0, lt = 0, scale_buf = 0, g = 0;         // g: the rows' group
            uint32_t parity = 0, x_parity = 0;
            for (int tile = first_tile; tile < a.tiles && ok; tile += tile_step, ++lt) {
                const int buf = lt & 1;
                if (!mx_bar_wait(mx_smem(&acc_empty[buf]), ((lt >> 1) & 1) ^ 1, a.wait_cycles, gave_up_v)) { ok = false; break; }
                if (resident) g = 0;
                for (int kb = b0; kb < b1; kb += STEP) {
                    const int n = min(STEP, b1 - kb);
                    const uint32_t full = mx_smem(&full_bar[s]);
                    const bool fresh = !resident || lt == 0; // the rows are being made ready
                    if (!mx_bar_wait_both(full, parity, fresh ? mx_smem(&x_ready[g]) : full, fresh ? x_parity : parity, a.wait_cycles, gave_up_v)) { ok = false; break; }
                    mx_fence_after();
#pragma unroll
                    for (int j = 0; j < STEP; ++j) {
                        if (j >= n) { commit(mx_smem(&empty_bar[s * STEP + j])); break; }
                        const uint32_t sa = tmem + 2 * NB + (uint32_t)((scale_buf + j) & (SCALE_BUFS - 1)) * 8, sb = sa + 4;
                        copy_scales(sa, mx_scale_desc(ws_s + (uint32_t)((s * STEP + j) * MX_SCALE_BYTES)));
                        copy_scales(sb, mx_scale_desc(xs_s + (uint32_t)((g * STEP + j) * MX_SCALE_BYTES)));
                        const uint64_t ad = mx_operand_desc(ring_s + (uint32_t)((s * STEP + j) * MX_TILE_BYTES)), bd = mx_operand_desc(x_s + (uint32_t)((g * STEP + j) * X_BLOCK));
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            mma_mx(tmem + buf * NB, ad + (uint32_t)(k * 2), bd + (uint32_t)(k * 2), mx_idesc(MX_E2M1, MX_E4M3, MX_ROWS, NB, k), sa, sb, kb + j != b0 || k != 0);
                        commit(mx_smem(&empty_bar[s * STEP + j]));
                    }
                    if (!resident) commit(mx_smem(&x_free[g]));
                    scale_buf = (scale_buf + n) & (SCALE_BUFS - 1);
                    if (++s == a.stages) { s = 0; parity ^= 1; }
                    if (++g == x_groups) { g = 0; x_parity ^= 1; }
                }
                if (resident) x_parity = 0;
                if (ok) commit(mx_smem(&acc_full[buf]));
            }
        }
        __syncwarp();
    } else {
        // ---- rows to parts; then the sums ----
        rdl_grid_wait();
        rdl_grid_launch_dependents();
        const int q = warp & 3, half = (warp - 2) >> 2;      // the first eight of these warps take the sums out
        // a lane's chunk of row 0 (lanes 16 to 31: of row 1) of a block, and its group's scale: the two halves of a warp hold neighbouring rows
        const uint32_t my_place = x_s + (uint32_t)((lane >> 4) * 128 + ((((lane & 15) >> 1) ^ (lane >> 4)) << 4) + (lane & 1) * 8);
        const uint32_t my_scale = xs_s + (uint32_t)((lane >> 4) * 16 + ((lane & 15) >> 2));
        // behind a deferred norm the rows are the operand's: R / 2 of the stream, R / 2 of the branch, the first src_rows of each in use
        auto used_row = [&](int r) { return MODE != RDL_NORM_DEFERRED || (r & (R / 2 - 1)) < a.src_rows; };
        // The rows of tile `turn` of this block: warps take pieces in turn, PIECE_ROWS rows of a block of columns, and hand them over; the
        // products begin with the first STEP blocks.  Where the rows do not stay, a piece waits until its slot has been read.  The pieces
        // are counted on over the tiles, and there are no more warps at it than a round over the slots has pieces: so a warp's next piece
        // is at most one round on, and the phase of its slot's barrier before the one that it waits for is over.
        const int pieces = groups * PIECES, takers = min(TAKERS, x_groups * PIECES);
        auto shift = [](Chunk<PARTS> (&d)[AHEAD]) {
#pragma unroll
            for (int i = 1; i < AHEAD; ++i) d[i - 1] = d[i];
        };
        // the rows' numbers, for the warps that need them: the ones that take sums out, or the ones that join halves
        constexpr int SCALED = (MODE == NORM_JOINED ? TAKERS : 8) * 32;
        auto wait_scales = [&]() { asm volatile("bar.sync 2, %0;" ::"n"(SIDE * 32 + SCALED) : "memory"); };
        bool have_scales = false;
        const int branch_row = a.src_rows <= 4 ? 4 : 8;      // where the operand's second half begins
        auto prepare = [&](int turn) {
            if (warp - 2 >= takers) return;
            const int before = turn * pieces;
            for (int p = before + ((warp - 2 - before % takers + takers) % takers); p < before + pieces; p += takers) {
                const int nth = p / PIECES, piece = p - before, gi = piece / PIECES, round = nth / x_groups, gs = nth - round * x_groups;
                if (round > 0 && !resident && !mx_bar_wait(mx_smem(&x_free[gs]), (round - 1) & 1, a.wait_cycles, gave_up_v)) ok = false;
                const int j = piece % PIECES / (R / PIECE_ROWS), first = piece % (R / PIECE_ROWS) * PIECE_ROWS, block = b0 + gi * STEP + j, slot = gs * STEP + j;
                const int chunks = block < b1 ? min((MODE == RDL_NORM_DEFERRED ? R : a.src_rows) - first, PIECE_ROWS) * (MX_BLOCK / 8) : 0;     // 16 a row
                const uint32_t at = my_place + (uint32_t)(slot * X_BLOCK + first * 128), sc_at = my_scale + (uint32_t)(slot * MX_SCALE_BYTES + first * 16);
                uint32_t seen[4] = {0, 0, 0, 0};         // rows by kind
                Chunk<PARTS> d[AHEAD];
                uint4 branch[MODE == NORM_JOINED ? AHEAD : 1];
                if (chunks > 0) {
#pragma unroll
                    for (int u = 0; u < AHEAD; ++u) {
                        const int i = u * 32 + lane;
#pragma unroll
                        for (int e = 0; e < (int)(sizeof(d[u].w) / 4); ++e) d[u].w[e] = 0;
                        d[u].code = 0;
                        const int k = block * MX_BLOCK + (lane & 15) * 8;
                        if (i < chunks && used_row(first + (i >> 4))) load_chunk<PARTS>(a, first + (i >> 4), k, d[u]);
                        if constexpr (MODE == NORM_JOINED) {
                            branch[u] = make_uint4(0, 0, 0, 0);
                            if (i < chunks && k < a.K) branch[u] = *reinterpret_cast<const uint4*>((const __nv_bfloat16*)a.x + (long long)(branch_row + first + (i >> 4)) * a.K + k);
                        }
                    }
                }
                if (MODE == NORM_JOINED && !have_scales) {           // asked for before the rows' numbers are there
                    wait_scales();
                    have_scales = true;
                }
                if (chunks > 0) {
#pragma unroll 1                                                                     // short code: see the head of the file
                    for (int u = 0; u < AHEAD; ++u) {
                        const int m0 = u * 2;                                        // this lane's row of the piece: m0 or m0 + 1
                        if (u * 32 >= chunks) break;                                 // none of this warp's
                        if (MODE == RDL_NORM_DEFERRED && !used_row(first + m0)) { shift(d); continue; }
                        if constexpr (MODE == NORM_JOINED) {
                            const float2 r = row_scale[(first + m0 + (lane >> 4)) & 7];
                            d[0].w[0] = join_pair(d[0].w[0], branch[0].x, r);
                            d[0].w[1] = join_pair(d[0].w[1], branch[0].y, r);
                            d[0].w[2] = join_pair(d[0].w[2], branch[0].z, r);
                            d[0].w[3] = join_pair(d[0].w[3], branch[0].w, r);
#pragma unroll
                            for (int i = 1; i < AHEAD; ++i) branch[i - 1] = branch[i];
                        }
                        uint2 bytes[PARTS];
                        uint32_t code[PARTS];
                        const int kind = make_parts<PARTS>(d[0], bytes, code);
                        shift(d);
                        if (u * 32 + lane < chunks) {
                            // swizzled by the row: rows r and r + 1, r even, flip the pieces by r & 6 beside what my_place has of the lane's own
                            const uint32_t to = (at ^ (uint32_t)(((first + m0) & 6) << 4)) + (uint32_t)(m0 * 128);
#pragma unroll
                            for (int part = 0; part < PARTS; ++part)
                                asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(to + (uint32_t)(part * R * 128)), "r"(bytes[part].x), "r"(bytes[part].y) : "memory");
                            if ((lane & 3) == 0) {
#pragma unroll
                                for (int part = 0; part < PARTS; ++part)
                                    asm volatile("st.shared.u8 [%0], %1;" ::"r"(sc_at + (uint32_t)(m0 * 16 + (part * R & 31) * 16 + (part * R >> 5) * 4)), "r"(code[part]) : "memory");
                            }
                            if (PARTS > 1) {
#pragma unroll
                                for (int kd = 0; kd < 4; ++kd)
                                    if (kd != ROW_ZERO && kind == kd) seen[kd] |= 1u << (first + m0 + (lane >> 4));
                            }
                        }
                    }
                }
                if (PARTS > 1) {
                    const uint32_t fine = __reduce_or_sync(0xffffffffu, seen[ROW_FINE]), rare = seen[ROW_TINY] | seen[ROW_BAD];
                    if (lane == 0 && fine) atomicOr(&fine_rows, fine);
                    if (rare) { atomicOr(&tiny_rows, seen[ROW_TINY]); atomicOr(&bad_rows, seen[ROW_BAD]); }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");             // the products read what was stored here
                __syncwarp();
                if (lane == 0) mx_bar_arrive(mx_smem(&x_ready[gs]));
            }
        };
        int lt = 0;
        // (a wait in vain ends no loop here: the blocks of a cluster meet again below)
        prepare(0);
        if (MODE == NORM_JOINED && warp < 2 + TAKERS && !have_scales) wait_scales();     // (it had no rows: the barrier counts it)
        if (SIDE > 0 && warp >= 2 + TAKERS) {
            // a row's two numbers, lane & 7 the row, from the branch's partial sums in a fixed order
            const DeferredNormArgs& d = a.norm;
            auto add_lanes = [](float4& v) {                 // over the lanes with the same lane & 7
#pragma unroll
                for (int o = 8; o <= 16; o <<= 1) {
                    v.x += __shfl_xor_sync(0xffffffffu, v.x, o); v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
                    v.z += __shfl_xor_sync(0xffffffffu, v.z, o); v.w += __shfl_xor_sync(0xffffffffu, v.w, o);
                }
            };
            const int me = warp - 2 - TAKERS;
            float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
            if ((lane & 7) < a.src_rows) {
                for (int u0 = me * 4 + (lane >> 3); u0 < d.n_sums; u0 += 8 * SIDE * 4) {
                    float4 v[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int u = u0 + i * SIDE * 4;
                        v[i] = u < d.n_sums ? __ldcg(reinterpret_cast<const float4*>(d.sums) + u * 8 + (lane & 7)) : make_float4(0.f, 0.f, 0.f, 0.f);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) { t.x += v[i].x; t.y += v[i].y; t.z += v[i].z; t.w += v[i].w; }
                }
            }
            add_lanes(t);
            if (lane < 8) norm_part[me][lane] = t;
            asm volatile("bar.sync 1, %0;" ::"n"(SIDE * 32) : "memory");
            static_assert(SIDE == 0 || SIDE == 4, "four shares, one a quarter of the warp");
            t = norm_part[(lane >> 3) & (SIDE ? SIDE - 1 : 0)][lane & 7];
            add_lanes(t);
            const float s1 = rsqrtf(t.x / (float)a.K + d.eps1);
            const float s2 = rsqrtf(fmaxf(t.y + 2.f * s1 * t.z + s1 * s1 * t.w, 0.f) / (float)a.K + d.eps2);     // of the squares of h + s1 a'
            if (me == 0 && lane < 8) row_scale[lane] = make_float2(s1, s2);
            __syncwarp();
            asm volatile("bar.arrive 2, %0;" ::"n"(SIDE * 32 + SCALED) : "memory");
            // this block's slice of the updated stream and of the operand after it
            if (d.residual_out || d.scaled_next) {
                const long long total = (long long)a.src_rows * a.K, per = (total + gridDim.x - 1) / gridDim.x;
                const long long begin = (long long)blockIdx.x * per, end = begin + per < total ? begin + per : total;
                for (long long e0 = begin + me * 32; e0 < end; e0 += SIDE * 32) {
                    const long long e = e0 + lane;
                    const bool in = e < end;
                    const int m = in ? (int)(e / a.K) : 0;
                    const float r1 = __shfl_sync(0xffffffffu, s1, m);
                    if (!in) continue;
                    const float h = fmaf(r1, raw_value(raw_load(d.branch_in, e, RDL_BF16), RDL_BF16), d.residual_in[e]);
                    if (d.residual_out) d.residual_out[e] = h;
                    if (d.scaled_next)
                        ((__nv_bfloat16*)d.scaled_next)[e] = __float2bfloat16_rn(h * (raw_value(raw_load(d.w_next, e - (long long)m * a.K, d.w_next_dtype), d.w_next_dtype) + d.off_next));
                }
            }
        }
        for (int tile = first_tile; tile < a.tiles; tile += tile_step, ++lt) {
            // the next tile's rows before this one's sums: its products then find them (they need the sums before these to be out, which
            // the last turn saw to)
            if (!resident && tile + tile_step < a.tiles) prepare(lt + 1);
            const int buf = lt & 1;
            // Only the warps that take the sums out wait for them: the products of the tile after next need their arrival, so this barrier
            // is never two phases ahead of them.  A warp without a say in that could come two tiles late and wait for a phase that is not to be.
            if (warp < 10 && !mx_bar_wait(mx_smem(&acc_full[buf]), (lt >> 1) & 1, a.wait_cycles, gave_up_v)) ok = false;
            mx_fence_after();
            if (MODE == RDL_NORM_DEFERRED && lt == 0 && warp < 10) wait_scales();
            float* y = reinterpret_cast<float*>(smem + y_off);       // a cluster's sums (one tile each)
            if (warp < 10) {
                // lane l of quarter q: weight row 32 q + l of the tile; this warp takes half of the rows
                constexpr int MINE = R / 2;
                // which row sum[j] is of: half of the rows, or (deferred) of the stream's the same as of the branch's
                auto row_of = [&](int j) { return MODE != RDL_NORM_DEFERRED ? half * MINE + j : (j < MINE / 2 ? 0 : MINE / 2) + half * (MINE / 2) + j; };
                float sum[MINE];
#pragma unroll
                for (int j = 0; j < MINE; ++j) sum[j] = 0.f;
                if (groups > 0) {
                    uint32_t v[PARTS][MINE];
#pragma unroll
                    for (int part = 0; part < PARTS; ++part) {
                        const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * NB + part * R);
                        if constexpr (MODE != RDL_NORM_DEFERRED) tmem_ld<MINE>(at + half * MINE, v[part]);
                        else {
                            tmem_ld<MINE / 2>(at + half * (MINE / 2), v[part]);
                            tmem_ld<MINE / 2>(at + R / 2 + half * (MINE / 2), v[part] + MINE / 2);
                        }
                    }
                    mx_tmem_wait_ld();
#pragma unroll
                    for (int part = PARTS - 1; part >= 0; --part)                            // the smallest first
#pragma unroll
                        for (int j = 0; j < MINE; ++j) sum[j] += __uint_as_float(v[part][j]);
                }
                mx_fence_before();
                __syncwarp();
                if (lane == 0) mx_bar_arrive(mx_smem(&acc_empty[buf]));
                // all of a row too small for its last parts (below 2^-98): they would be lost
                const unsigned bad = *(volatile unsigned*)&bad_rows | (*(volatile unsigned*)&tiny_rows & ~*(volatile unsigned*)&fine_rows);
                if (PARTS > 1 && bad) {                          // plain arithmetic, for what the parts cannot hold
                    const int wr = tile * MX_ROWS + 32 * q + lane;
                    for (int j = 0; j < MINE; ++j) {
                        const int m = row_of(j);
                        if (!(bad >> m & 1)) continue;
                        float y = 0.f;
                        for (int k = b0 * MX_BLOCK; k < min(b1 * MX_BLOCK, a.K); ++k) {
                            const uint32_t code = a.codes[mx_code_at(wr, k, a.blocks)] >> (4 * (k & 1));
                            uint32_t h[4];
                            mx_from_e2m1(code & 15u, h);
                            const float w = __half2float(__ushort_as_half((unsigned short)(h[0] & 0xffffu)))
                                            * mx_scale(a.scales[mx_scale_at(wr, k, a.blocks)]);
                            float x = rdl_load(a.x, (long long)m * a.K + k, PARTS == 2 ? RDL_BF16 : RDL_F32);
                            if constexpr (MODE == NORM_JOINED)
                                x = __bfloat162float(__float2bfloat16_rn(join(x, rdl_load(a.x, (long long)(branch_row + m) * a.K + k, RDL_BF16), row_scale[m])));
                            y = fmaf(x, w, y);
                        }
#pragma unroll
                        for (int i = 0; i < MINE; ++i)
                            if (i == j) sum[i] = y;
                    }
                }
                if constexpr (MODE == RDL_NORM_DEFERRED) {       // both halves joined; sum[j] is row half * MINE / 2 + j of the result
#pragma unroll
                    for (int j = 0; j < MINE / 2; ++j) {
                        const float2 r = row_scale[half * (MINE / 2) + j];
                        sum[j] = r.y * fmaf(r.x, sum[j + MINE / 2], sum[j]);
                    }
                }
                constexpr int OWN = MODE == RDL_NORM_DEFERRED ? MINE / 2 : MINE;
                const int m_first = half * OWN, m_end = min(m_first + OWN, a.src_rows);
                if (a.split == 1) {
                    // neighbouring lanes have neighbouring outputs; gated: 16 gate rows, then their 16 up rows
                    const int n = a.gated ? tile * (MX_ROWS / 2) + 16 * q + lane : tile * MX_ROWS + 32 * q + lane;
#pragma unroll 1
                    for (int m = m_first; m < m_end; ++m) {
                        const float up = a.gated ? __shfl_down_sync(0xffffffffu, sum[0], 16) : 0.f;
                        if (n < a.N && (!a.gated || lane < 16)) {
                            const float y = finish(a, sum[0], up);
                            if (!behind_norm(MODE) || !a.norm.row_index) rdl_store(a.out, (long long)m * a.N + n, a.out_dtype, y);
                            else
                                for (int j = 0; j < a.M; ++j)
                                    if (a.norm.row_index[j] == m) rdl_store(a.out, (long long)j * a.N + n, a.out_dtype, y);
                        }
#pragma unroll
                        for (int i = 1; i < OWN; ++i) sum[i - 1] = sum[i];
                    }
                } else {
                    // each block adds up a part of the outputs: this row's sums go to its block, to this rank's place there
                    const int r = 32 * q + lane, o = a.gated ? (r >> 5) * 16 + (r & 15) : r, owner = o / a.share;
                    const int at = a.gated ? (o - owner * a.share) * 2 + ((r >> 4) & 1) : o - owner * a.share, outs = a.gated ? 2 * a.share : a.share;
                    cluster_wait();                              // every block of the cluster runs
                    const uint32_t to = map_to_block(mx_smem(y), owner) + (uint32_t)(rank * R * outs + at) * 4;
#pragma unroll
                    for (int j = 0; j < OWN; ++j)
                        if (m_first + j < m_end) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + (uint32_t)((m_first + j) * outs) * 4), "f"(sum[j]) : "memory");
                }
            } else if (a.split > 1) {
                cluster_wait();
            }
        }
    }
    if (!ok && a.status) atomicExch(a.status, RDL_FAULT_MX_FEW);
    if (a.split > 1) {
        __syncwarp();
        if (warp < 2) cluster_wait();                        // the first barrier: the workers are past it
        cluster_arrive();
        // the branch of a residual stream: a warp takes a row, and has its elements of the stream and the norms' weights on their way now
        constexpr int PER_LANE = MODE == RDL_NORM_BRANCH ? 2 : 1;                        // of at most 64 outputs
        float stream[PER_LANE];
        uint32_t w1[PER_LANE], w2[PER_LANE];
        if constexpr (MODE == RDL_NORM_BRANCH) {
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i) {
                const int o = lane + 32 * i, of_tile = rank * a.share + o, n = first_tile * MX_ROWS + of_tile, m = warp - 2;
                stream[i] = 0.f; w1[i] = w2[i] = 0;
                if (m < 0 || m >= a.M || o >= a.share || of_tile >= MX_ROWS || n >= a.N) continue;
                stream[i] = a.norm.residual[(long long)m * a.N + n];
                w1[i] = raw_load(a.norm.w1, n, a.norm.w1_dtype);
                w2[i] = raw_load(a.norm.w2, n, a.norm.w2_dtype);
            }
        }
        cluster_wait();                                      // every block's sums are where they are added up
        if constexpr (MODE == RDL_NORM_BRANCH) {
            const int m = warp - 2;
            if (m >= 0 && m < 8) {
                const DeferredNormArgs& d = a.norm;
                const float* ys = reinterpret_cast<const float*>(smem + y_off) + m * a.share;
                float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int i = 0; i < PER_LANE; ++i) {
                    const int o = lane + 32 * i, of_tile = rank * a.share + o, n = first_tile * MX_ROWS + of_tile;
                    if (m >= a.M || o >= a.share || of_tile >= MX_ROWS || n >= a.N) continue;
                    float v[8], y = 0.f;
#pragma unroll
                    for (int s = 0; s < 8; ++s) v[s] = s < a.split ? ys[s * R * a.share + o] : 0.f;
#pragma unroll
                    for (int s = 0; s < 8; ++s) y += v[s];
                    const __nv_bfloat16 b = __float2bfloat16_rn(y * (raw_value(w1[i], d.w1_dtype) + d.off1));
                    const float bv = __bfloat162float(b);    // what the stream will add, s1 times
                    t.x = fmaf(y, y, t.x); t.y = fmaf(stream[i], stream[i], t.y); t.z = fmaf(stream[i], bv, t.z); t.w = fmaf(bv, bv, t.w);
                    ((__nv_bfloat16*)d.branch)[(long long)m * a.N + n] = b;
                    ((__nv_bfloat16*)d.scaled)[(long long)m * a.N + n] = __float2bfloat16_rn(bv * (raw_value(w2[i], d.w2_dtype) + d.off2));
                }
                t.x = warp_sum(t.x); t.y = warp_sum(t.y); t.z = warp_sum(t.z); t.w = warp_sum(t.w);
                if (lane == 0) reinterpret_cast<float4*>(d.sums)[blockIdx.x * 8 + m] = t;        // rows beyond M: zeros
            }
        } else if (warp >= 2) {
            const int tid = threadIdx.x - 64, per_tile = a.gated ? MX_ROWS / 2 : MX_ROWS, outs = a.gated ? 2 * a.share : a.share;
            const float* y = reinterpret_cast<const float*>(smem + y_off);
            for (int idx = tid; idx < a.M * a.share; idx += WORKERS) {
                const int m = idx / a.share, o = idx - m * a.share, of_tile = rank * a.share + o, n = first_tile * per_tile + of_tile;
                const int src = behind_norm(MODE) && a.norm.row_index ? a.norm.row_index[m] : m;
                if (of_tile >= per_tile || n >= a.N || src < 0 || src >= a.src_rows) continue;
                const float* ys = y + src * outs + (a.gated ? 2 * o : o);
                float v[8], u[8];
#pragma unroll
                for (int s = 0; s < 8; ++s) {                // all asked for before the first is used
                    v[s] = s < a.split ? ys[s * R * outs] : 0.f;
                    u[s] = a.gated && s < a.split ? ys[s * R * outs + 1] : 0.f;
                }
                float sum = 0.f, up = 0.f;
#pragma unroll
                for (int s = 0; s < 8; ++s) { sum += v[s]; up += u[s]; }
                rdl_store(a.out, (long long)m * a.N + n, a.out_dtype, finish(a, sum, up));
            }
        }
    }
    mx_fence_before();
    __syncthreads();
    if (*gave_up_v) {                    // behind the barrier: whichever warp gave up, the loader has asked for its last copies by now
        rdl_drain_copies();
        __syncwarp();
    }
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
}

// How a product is divided and what shared memory holds; returns its bytes.
template <int PARTS, int R, int MODE>
int plan(FewArgs& a, const Mx4Matrix& w) {
    constexpr int NB = PARTS * R, PER_BLOCK = NB * MX_BLOCK + MX_SCALE_BYTES, PER_STAGE = STEP * (MX_TILE_BYTES + MX_SCALE_BYTES);
    const int sms = rdl_sm_count();
    a.blocks = w.blocks; a.gated = w.gated;
    a.tiles = w.tiles;
    a.split = mx_split(a.tiles, a.blocks, sms);
    a.share = ((a.gated ? MX_ROWS / 2 : MX_ROWS) + a.split - 1) / a.split;
    a.slice_blocks = (a.blocks + a.split - 1) / a.split;
    const int sums = a.split > 1 ? R * (MX_ROWS + 16) * 4 : 0, most = 226 * 1024 - 1024 - (behind_norm(MODE) ? 2048 : 1024) - sums;    // alignment, static shared memory
    // The rows of all of a block's columns, if a ring of two stages fits beside them (in the form of that time float32, 8 rows x 2,304, 256,000 outputs: 71 us so
    // and 94 with the rows brought anew for every tile; bfloat16, 16 x 3,584, 28,672 gated: 20.5 and 23.0; now 62.7 and 20.2); else as many as fit beside four.
    a.slots = (a.slice_blocks + STEP - 1) / STEP * STEP;
    if (a.slots * PER_BLOCK + 2 * PER_STAGE > most) a.slots = (most - 4 * PER_STAGE) / PER_BLOCK / STEP * STEP;
    if (a.slots > MAX_SLOTS) a.slots = MAX_SLOTS;
    a.stages = (most - a.slots * PER_BLOCK) / PER_STAGE;
    if (a.stages > MAX_STAGES) a.stages = MAX_STAGES;
    // no deeper than the block's work: what shared memory is left lets the next kernel's blocks begin
    const int turns = a.split > 1 ? 1 : (a.tiles + sms - 1) / sms;
    const int steps = (a.slice_blocks + STEP - 1) / STEP;
    if ((long long)a.stages > (long long)turns * steps) a.stages = turns * steps;
    return 1024 + a.slots * PER_BLOCK + a.stages * PER_STAGE + sums;
}
// the rows of a block are made ready once, not again for every tile
bool once(const FewArgs& a) { return a.slots >= a.slice_blocks || a.split > 1 || a.tiles <= rdl_sm_count(); }

template <int PARTS, int R, int MODE = 0>
int launch(FewArgs a, const Mx4Matrix& w, cudaStream_t st) {
    a.codes = w.codes; a.scales = w.scales;
    a.N = w.gated ? w.rows / 2 : w.rows; a.K = w.columns;
    a.wait_cycles = rdl_wait_cycles_for(RDL_FAULT_MX_FEW); a.test_extra_tx = rdl_test_extra_tx_for(RDL_FAULT_MX_FEW);
    const int smem = plan<PARTS, R, MODE>(a, w), sms = rdl_sm_count();
    RDL_CUDA((rdl_allow_shared<mx_few_rows_kernel<PARTS, R, MODE>>(smem)), "mx_few_rows");
    const int grid = a.split > 1 ? a.tiles * a.split : (a.tiles < sms ? a.tiles : sms);
    RDL_CHECK_EX(rdl_launch_cluster(mx_few_rows_kernel<PARTS, R, MODE>, dim3(grid), dim3(THREADS), a.split, (size_t)smem, st, w.codes_map, a), "mx_few_rows");
    return 0;
}

}  // namespace

extern "C" int rdl_mx_few_rows(void* out, int out_dtype, const void* x, int x_kind, const void* row_scales, const void* weight, int m,
                               int activation, float act_param, float softcap, int* status, void* stream) {
    const Mx4Matrix* w = (const Mx4Matrix*)weight;
    RDL_REQUIRE(w && w->codes, "mx_few_rows: missing weight");
    RDL_REQUIRE(m >= 0 && m <= 16, "mx_few_rows: %d rows, at most 16 are supported", m);
    if (m == 0) return 0;
    RDL_REQUIRE(out && x, "mx_few_rows: missing operand");
    RDL_REQUIRE(rdl_valid_dtype(out_dtype), "mx_few_rows: bad output dtype %d", out_dtype);
    RDL_REQUIRE(rdl_valid_dtype(x_kind) || (x_kind == RDL_MX8 && row_scales && (uintptr_t)x % 8 == 0), "mx_few_rows: bad rows (kind %d)", x_kind);
    RDL_REQUIRE(!w->gated || rdl_gated_known(activation), "mx_few_rows: unknown activation %d", activation);
    RDL_REQUIRE(softcap >= 0.f, "mx_few_rows: soft-cap must not be negative");
    FewArgs a{};
    a.x = x; a.row_scales = (const uint8_t*)row_scales;
    a.out = out; a.out_dtype = out_dtype;
    a.M = a.src_rows = m; a.row_pad = (m + 3) / 4 * 4;
    a.activation = activation; a.act_param = act_param; a.softcap = softcap;
    a.vec = w->columns % 8 == 0 && (uintptr_t)x % 16 == 0;
    a.status = status;
    cudaStream_t st = (cudaStream_t)stream;
    if (x_kind == RDL_MX8) return launch<1, 16>(a, *w, st);
    if (x_kind == RDL_BF16) return m <= 8 ? launch<2, 8>(a, *w, st) : launch<2, 16>(a, *w, st);
    return m <= 8 ? launch<6, 8>(a, *w, st) : launch<6, 16>(a, *w, st);
}

// The partial sums a branch's product writes for each of its rows: one a block; 0: the matrix is not shared by clusters, no such form
extern "C" int rdl_mx_branch_units(const void* weight) {
    const Mx4Matrix* w = (const Mx4Matrix*)weight;
    if (!w || !w->codes || w->gated) return 0;
    const int split = mx_split(w->tiles, w->blocks, rdl_sm_count());
    return split > 1 ? w->tiles * split : 0;
}

// Up to how many rows the product behind a deferred norm pays: none where its rows are made ready again for every tile
extern "C" int rdl_mx_deferred_rows(const void* weight) {
    const Mx4Matrix* w = (const Mx4Matrix*)weight;
    if (!w || !w->codes) return 0;
    FewArgs a{};
    plan<2, 8, NORM_JOINED>(a, *w);
    return once(a) ? 8 : 0;
}

extern "C" int rdl_mx_few_rows_norm(void* out, int out_dtype, const void* x, const void* weight, int m, int activation, float act_param,
                                    float softcap, const DeferredNormArgs* norm, int* status, void* stream) {
    const Mx4Matrix* w = (const Mx4Matrix*)weight;
    RDL_REQUIRE(w && w->codes && x && norm, "mx_few_rows_norm: missing operand");
    RDL_REQUIRE(m > 0 && m <= 8, "mx_few_rows_norm: %d rows, 1 to 8 are supported", m);
    RDL_REQUIRE(norm->sums && (uintptr_t)norm->sums % 16 == 0, "mx_few_rows_norm: the partial sums must lie on a 16-byte boundary");
    FewArgs a{};
    a.x = x; a.norm = *norm; a.status = status;
    a.activation = activation; a.act_param = act_param; a.softcap = softcap;
    a.M = a.src_rows = m;
    a.vec = w->columns % 8 == 0 && (uintptr_t)x % 16 == 0;
    if (norm->mode == RDL_NORM_BRANCH) {
        RDL_REQUIRE(!w->gated && activation == 0 && softcap == 0.f, "mx_few_rows_norm: a branch's product has the plain epilogue");
        RDL_REQUIRE(norm->residual && norm->w1 && norm->w2 && norm->branch && norm->scaled, "mx_few_rows_norm: a branch needs the stream, both norms' weights and its two outputs");
        RDL_REQUIRE(rdl_valid_dtype(norm->w1_dtype) && rdl_valid_dtype(norm->w2_dtype), "mx_few_rows_norm: bad dtype of a norm's weight");
        const int units = rdl_mx_branch_units(weight);
        RDL_REQUIRE(units > 0 && norm->n_sums == units, "mx_few_rows_norm: place for %d units of sums, the matrix has %d", norm->n_sums, units);
        return launch<2, 8, RDL_NORM_BRANCH>(a, *w, (cudaStream_t)stream);
    }
    RDL_REQUIRE(norm->mode == RDL_NORM_DEFERRED, "mx_few_rows_norm: unknown mode %d", norm->mode);
    RDL_REQUIRE(out && rdl_valid_dtype(out_dtype), "mx_few_rows_norm: missing output or bad output dtype %d", out_dtype);
    RDL_REQUIRE(!w->gated || rdl_gated_known(activation), "mx_few_rows_norm: unknown activation %d", activation);
    RDL_REQUIRE(softcap >= 0.f, "mx_few_rows_norm: soft-cap must not be negative");
    RDL_REQUIRE(a.vec, "mx_few_rows_norm: the operand needs a multiple of 8 columns and a 16-byte boundary");
    RDL_REQUIRE(norm->n_sums > 0 && norm->n_out > 0 && norm->n_out <= 8 && (norm->row_index || norm->n_out == m), "mx_few_rows_norm: %d units of sums, %d output rows of %d", norm->n_sums, norm->n_out, m);
    const bool side = norm->residual_out || norm->scaled_next;
    RDL_REQUIRE(!side || (norm->branch_in && norm->residual_in), "mx_few_rows_norm: the stream's update needs the branch and the stream");
    // other blocks still read the old one
    RDL_REQUIRE(!norm->residual_out || norm->residual_out != norm->residual_in, "mx_few_rows_norm: the updated stream needs a buffer of its own");
    RDL_REQUIRE(!norm->scaled_next || (norm->w_next && rdl_valid_dtype(norm->w_next_dtype)), "mx_few_rows_norm: the next operand needs the next norm's weight");
    a.out = out; a.out_dtype = out_dtype;
    a.M = norm->n_out;
    // 4 rows, 2,304 wide, gated 18,432 and 4,096 outputs: 8.7 and 6.8 us as halves, 9.9 and 6.9 joined; 8 rows: 11.1 and 7.1, 9.7 and 6.6
    return m <= 4 ? launch<2, 8, RDL_NORM_DEFERRED>(a, *w, (cudaStream_t)stream) : launch<2, 8, NORM_JOINED>(a, *w, (cudaStream_t)stream);
}
