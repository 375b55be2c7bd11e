// Log probabilities, entropy and alternatives by the logits  z = scale * cap tanh(x W^T / cap)  of bfloat16 rows x behind an output head W
// [vocab, k], without logits in memory: the product runs on the fifth-generation tensor cores, and what takes a tile of it out
// of tensor memory keeps each row's statistics and list (logprobs.cuh) instead of storing it.
//
// A tile is 128 CTAS rows x 256 tokens.  CTAS 2 (more than 128 rows): a pair of blocks on two multiprocessors (cta_group::2); each holds 128 of
// the rows and 128 of the tile's weight rows, and the products, issued by a thread of block 0, read both halves.  CTAS 1: up to 128
// rows, where reading the weights is what takes the time.  Two accumulators: the products of a tile run while the tile before it is
// taken out.
//
// Persistent: a group (a pair, or a block) walks along the vocabulary for one block of rows, so that a row's statistics stay in one
// thread's registers.  Groups of all row blocks walk side by side over the same part of it (a slice), and their weight tiles come from
// memory once.  With B row blocks and P groups there are P / B slices; the P mod B groups over share the end of the vocabulary, all row blocks in
// turn, so that every group has as many tiles.  Each (row block, range) leaves partial results, which a second kernel joins.
//
// Warp 0 loads (TMA, a ring of stages of 64 k), warp 1 issues the products, eight warps take the accumulator out: two a quarter of
// tensor memory, half of the columns each, a row a thread.  A row's logits beyond its list's last place are put aside in shared memory, and put
// into the list when some lane has five of them: all lanes of a warp then do so together, which a logit by itself would not.
//
// Every wait is bounded; a block that gives up sets `status` and every path ends in the common tear-down.  A block takes all of a
// multiprocessor's shared memory (see "Tensor memory" in mx_tensor.cuh: nothing that holds tensor memory fits beside it).
#include "api.h"
#include "launch.cuh"
#include "logprobs.cuh"
#include "mx_tensor.cuh"

namespace {

constexpr int BM = 128, BN = 256, BK = 64, EPI_WARPS = 8, EPI_THREADS = EPI_WARPS * 32, THREADS = 64 + EPI_THREADS;
constexpr int ASIDE = 8, AT_ONCE = 4;                     // logits a thread puts aside; that are looked at between two looks at how full that is
constexpr int TMEM_COLS = 2 * BN, MOST_STAGES = 6;
constexpr int SMEM_BYTES = 232448 - 1024;                 // a block's limit less the static variables
__host__ __device__ constexpr int stage_bytes(int ctas) { return BM * BK * 2 + BN / ctas * BK * 2; }

struct HeadArgs {
    int M, N, kblocks;
    int row_blocks, tiles_n;                              // of 128 CTAS rows, of 256 tokens
    int groups, slices, main_tiles;                       // slices share the first main_tiles tiles of every row block
    int stages, top;
    float cap, inv_cap, scale;
    const int* targets; float* target_logit;              // [M]
    float4* stats;                                        // [slot][column half][row of the block]: m, s, t
    LpKey* keys;                                          // [slot][column half][top][row of the block]
    long long wait_cycles; int test_extra_tx;
    int* status;
};

// The (row block, tiles) pieces of a group, one after another.
struct Pieces {
    int block, t0, t1, slot;
    long long at, end;                                    // of what is left: of the end of the vocabulary, row block by row block
    bool main_left;

    __host__ __device__ Pieces(const HeadArgs& a, int group) {
        const int mains = a.row_blocks * a.slices;
        main_left = group < mains;
        at = end = 0;
        if (main_left) {
            block = group % a.row_blocks;
            const int slice = group / a.row_blocks;
            t0 = (int)((long long)a.main_tiles * slice / a.slices);
            t1 = (int)((long long)a.main_tiles * (slice + 1) / a.slices);
            slot = block * a.slices + slice;
        } else {
            const long long total = (long long)a.row_blocks * (a.tiles_n - a.main_tiles), n = a.groups - mains, x = group - mains;
            at = total * x / n;
            end = total * (x + 1) / n;
            slot = mains + (int)x;
        }
    }
    // the next piece, or false
    __host__ __device__ bool next(const HeadArgs& a, int& b, int& first, int& last, int& place) {
        if (main_left) {
            main_left = false;
            b = block, first = t0, last = t1, place = slot;
            return first < last;
        }
        if (at >= end) return false;
        const int tiles = a.tiles_n - a.main_tiles, t = (int)(at % tiles);
        b = (int)(at / tiles);
        first = a.main_tiles + t;
        last = (int)(end - at < tiles - t ? first + (end - at) : a.tiles_n);
        place = slot + b;                                 // along the pieces either the group or the row block goes up: a number of its own
        at += last - first;
        return true;
    }
};

template <int CTAS>
__device__ __forceinline__ void load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if constexpr (CTAS == 1)
        mx_tma_2d(dst, map, x, y, bar);
    else
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar) : "memory");
}
// kind::f16: float accumulator, bfloat16 operands, both K-major
__host__ __device__ constexpr uint32_t head_idesc(int m) { return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }
template <int CTAS>
__device__ __forceinline__ void product(uint32_t d, uint64_t a, uint64_t b, uint32_t accumulate) {
    if constexpr (CTAS == 1)
        asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
                     ::"r"(d), "l"(a), "l"(b), "r"(head_idesc(BM)), "r"(accumulate) : "memory");
    else
        asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}"
                     ::"r"(d), "l"(a), "l"(b), "r"(head_idesc(2 * BM)), "r"(accumulate) : "memory");
}
// arrives at `bar` when the products so far are done; of a pair in both blocks
template <int CTAS>
__device__ __forceinline__ void commit(uint32_t bar) {
    if constexpr (CTAS == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((unsigned short)3) : "memory");
}
__device__ __forceinline__ uint32_t map_to_block(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// relaxed: what it orders, this warp's reads of tensor memory, has completed before
__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) { asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory"); }
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
                   "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
                   "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr) : "memory");
    mx_tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// A thread's `n` logits put aside, into its sorted list of `top` places (both in shared memory, a thread's keys EPI_THREADS apart).  Returns
// what a logit must exceed to enter: NaN while anything does.
__device__ __noinline__ float put_away(LpKey* list, const LpKey* aside, int n, int top) {
    LpKey last = list[(top - 1) * EPI_THREADS];
    for (int i = 0; i < n; ++i) {
        const LpKey k = aside[i * EPI_THREADS];
        if (k <= last) continue;
        int p = top - 1;
        for (; p > 0; --p) {
            const LpKey above = list[(p - 1) * EPI_THREADS];
            if (above > k) break;
            list[p * EPI_THREADS] = above;
        }
        list[p * EPI_THREADS] = k;
        last = list[(top - 1) * EPI_THREADS];
    }
    return (last >> 32) == 0 ? NAN : lp_key_logit(last);
}

template <int CTAS, bool TOP>
__global__ void __launch_bounds__(THREADS, 1) head_logprobs_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                                                                   const __grid_constant__ HeadArgs a) {
    constexpr int STAGE = stage_bytes(CTAS), A_BYTES = BM * BK * 2, ROWS = BM * CTAS;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) unsigned long long full_bar[MOST_STAGES], empty_bar[MOST_STAGES], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up;
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = CTAS == 1 ? 0 : (int)(blockIdx.x & 1), group = blockIdx.x / CTAS;
    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int s = 0; s < MOST_STAGES; ++s) {
            mx_bar_init(mx_smem(&full_bar[s]), 1);
            mx_bar_init(mx_smem(&empty_bar[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mx_bar_init(mx_smem(&acc_full[b]), 1);
            mx_bar_init(mx_smem(&acc_empty[b]), EPI_WARPS * CTAS);       // of a pair: used in block 0
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if constexpr (CTAS == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(mx_smem(&tmem_slot)), "r"(TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(mx_smem(&tmem_slot)), "r"(TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
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
    Pieces pieces(a, group);
    int block, t0, t1, slot;

    if (warp == 0) {
        // ---- loader, in every block: its rows and its part of the weight tile; of a pair all report to block 0 ----
        int s = 0;
        uint32_t parity = 1, extra = (uint32_t)a.test_extra_tx;      // the first round finds every stage free
        while (ok && pieces.next(a, block, t0, t1, slot)) {
            const int m0 = block * ROWS + rank * BM;
            for (int t = t0; t < t1 && ok; ++t) {
                const int n0 = t * BN + rank * (BN / CTAS);
                for (int kb = 0; kb < a.kblocks; ++kb) {
                    if (!mx_warp_wait(mx_smem(&empty_bar[s]), parity, a.wait_cycles, gave_up_v)) { ok = false; break; }
                    if (mx_elect()) {
                        const uint32_t own = mx_smem(&full_bar[s]), full = CTAS == 1 ? own : map_to_block(own, 0), st = mx_smem(smem + (size_t)s * STAGE);
                        if (rank == 0) mx_bar_expect(own, CTAS * STAGE + extra);
                        load<CTAS>(st, &map_x, kb * BK, m0, full);
                        load<CTAS>(st + A_BYTES, &map_w, kb * BK, n0, full);
                    }
                    __syncwarp();
                    extra = 0;
                    if (++s == a.stages) { s = 0; parity ^= 1; }
                }
            }
        }
    } else if (warp == 1) {
        // ---- the products: one thread, of a pair in block 0 ----
        int s = 0, lt = 0;
        uint32_t parity = 0;
        while (rank == 0 && ok && pieces.next(a, block, t0, t1, slot)) {
            for (int t = t0; t < t1 && ok; ++t, ++lt) {
                const int buf = lt & 1;
                if (!mx_warp_wait(mx_smem(&acc_empty[buf]), ((lt >> 1) & 1) ^ 1, a.wait_cycles, gave_up_v)) { ok = false; break; }
                mx_fence_after();
                for (int kb = 0; kb < a.kblocks; ++kb) {
                    if (!mx_warp_wait(mx_smem(&full_bar[s]), parity, a.wait_cycles, gave_up_v)) { ok = false; break; }
                    mx_fence_after();
                    if (mx_elect()) {
                        const uint32_t st = mx_smem(smem + (size_t)s * STAGE);
                        const uint64_t ad = mx_operand_desc(st), bd = mx_operand_desc(st + A_BYTES);
#pragma unroll
                        for (int k = 0; k < BK / 16; ++k) product<CTAS>(tmem + (uint32_t)(buf * BN), ad + (uint32_t)(k * 2), bd + (uint32_t)(k * 2), (kb | k) != 0);
                        commit<CTAS>(mx_smem(&empty_bar[s]));
                    }
                    __syncwarp();
                    if (++s == a.stages) { s = 0; parity ^= 1; }
                }
                if (ok && mx_elect()) commit<CTAS>(mx_smem(&acc_full[buf]));
                __syncwarp();
            }
        }
    } else {
        // ---- statistics and lists: warp q of four has the lanes of rows 32 q + lane, and of two such warps each has half of the columns ----
        const int q = warp & 3, half = (warp - 2) >> 2, own_row = rank * BM + q * 32 + lane, id = (int)threadIdx.x - 64;
        LpKey* list = reinterpret_cast<LpKey*>(smem + (size_t)a.stages * STAGE) + id;
        LpKey* aside = list + (TOP ? a.top : 0) * EPI_THREADS;
        const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(half * (BN / 2));
        const uint32_t to_issuer = CTAS == 1 ? mx_smem(&acc_empty[0]) : map_to_block(mx_smem(&acc_empty[0]), 0);
        int lt = 0;
        while (ok && pieces.next(a, block, t0, t1, slot)) {
            const int row = block * ROWS + own_row;
            const bool any_row = block * ROWS + rank * BM + q * 32 < a.M, mine = row < a.M;      // of the warp; of the lane
            const int target = mine && a.targets ? a.targets[row] : -1;
            LpStats st = lp_empty();
            float s_low = 0.f, t_low = 0.f;               // what the sums have lost to rounding: thousands of tiles may come
            float least = mine ? NAN : INFINITY;          // what a logit must exceed to enter the list (NaN: nothing)
            int n_aside = 0;
            if (TOP)
                for (int i = 0; i < a.top; ++i) list[i * EPI_THREADS] = 0;
            for (int t = t0; t < t1; ++t, ++lt) {
                const int buf = lt & 1;
                if (!mx_warp_wait(mx_smem(&acc_full[buf]), (lt >> 1) & 1, a.wait_cycles, gave_up_v)) { ok = false; break; }
                mx_fence_after();
                const int n0 = t * BN + half * (BN / 2);
#pragma unroll 1
                for (int c = 0; c < BN / 2; c += 32) {
                    const int n = n0 + c, there = a.N - n;                 // columns from here on
                    float v[32];
                    if (any_row && there > 0) tmem_ld32(lanes + (uint32_t)(buf * BN + c), v);
                    if (c == BN / 2 - 32) {                                // the last columns are in registers: the accumulator is free
                        mx_fence_before();
                        __syncwarp();
                        if (lane == 0) arrive_at(to_issuer + (uint32_t)(buf * 8));
                    }
                    if (!any_row || there <= 0) continue;
                    if (a.cap > 0.f && mine) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = a.cap * tanhf(v[i] * a.inv_cap);
                    }
                    if (a.scale != 1.f) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] *= a.scale;
                    }
                    if (there < 32) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = i < there ? v[i] : -INFINITY;
                    }
                    if ((unsigned)(target - n) < 32u) {
                        float z = v[0];
#pragma unroll
                        for (int i = 1; i < 32; ++i) z = target - n == i ? v[i] : z;
                        if (target < a.N) a.target_logit[row] = z;
                    }
                    float most = v[0];
#pragma unroll
                    for (int i = 1; i < 32; ++i) most = fmaxf(most, v[i]);
                    if (most > st.m) {
                        const float d = fmaxf(st.m - most, -1e30f), f = lp_exp2(d * LP_LOG2E);
                        t_low = f * fmaf(s_low, d, t_low);
                        s_low *= f;
                        lp_move(st, most);
                    }
                    LpStats more = {st.m, 0.f, 0.f};
                    lp_add(more, v);
                    const float ys = more.s + s_low, ns = st.s + ys, yt = more.t + t_low, nt = st.t + yt;
                    s_low = ys - (ns - st.s);
                    t_low = yt - (nt - st.t);
                    st.s = ns;
                    st.t = nt;
                    if (TOP && __any_sync(0xffffffffu, !(most <= least))) {
#pragma unroll
                        for (int g = 0; g < 32; g += AT_ONCE) {
                            if (__any_sync(0xffffffffu, n_aside > ASIDE - AT_ONCE)) {
                                if (mine) least = put_away(list, aside, n_aside, a.top);
                                n_aside = 0;
                            }
#pragma unroll
                            for (int i = g; i < g + AT_ONCE; ++i)
                                if (!(v[i] <= least) && i < there) {
                                    aside[n_aside * EPI_THREADS] = lp_key(v[i], (unsigned)(n + i));
                                    ++n_aside;
                                }
                        }
                    }
                }
            }
            if (!ok) break;
            if (mine) {
                const long long place = 2LL * slot + half;
                a.stats[place * ROWS + own_row] = make_float4(st.m, st.s + s_low, st.t + t_low, 0.f);
                if (TOP) {
                    put_away(list, aside, n_aside, a.top);
                    for (int i = 0; i < a.top; ++i) a.keys[(place * a.top + i) * ROWS + own_row] = list[i * EPI_THREADS];
                }
            }
        }
    }
    if (!ok && a.status) atomicExch(a.status, RDL_FAULT_LOGPROBS_HEAD);
    if (*gave_up_v && threadIdx.x == 0) mx_drain();
    // ---- tear-down, reached by every thread ----
    mx_fence_before();
    __syncthreads();
    if (CTAS == 2) cluster_sync();       // neither block leaves while the other may still read its shared memory or report to its barriers
    if (warp == 1) {
        if constexpr (CTAS == 1)
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// ---- the partial results of a row, joined: a block a row ----

struct JoinOut { float* logprobs; float* entropy; float* top_logprobs; int* top_ids; };

template <int WARPS>
__global__ void __launch_bounds__(WARPS * 32) head_join_kernel(const __grid_constant__ HeadArgs a, int rows_a_block, JoinOut o) {
    __shared__ LpStats part[WARPS];
    __shared__ LpKey lists[WARPS][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = blockIdx.x, block = row / rows_a_block, own_row = row - block * rows_a_block;
    // groups that share the vocabulary's end: those whose range meets this row block's
    const int mains = a.row_blocks * a.slices, tail = a.tiles_n - a.main_tiles, extras = a.groups - mains;
    const long long total = (long long)a.row_blocks * tail;
    int x0 = 0, x1 = 0;
    if (total > 0) {
        while (total * (x0 + 1) / extras <= (long long)block * tail) ++x0;
        x1 = x0;
        while (x1 < extras && total * x1 / extras < (long long)(block + 1) * tail) ++x1;
    }
    rdl_grid_wait();
    rdl_grid_launch_dependents();
    LpStats st = lp_empty();
    LpKey keys = 0;
    const int n = a.slices + x1 - x0;
    for (int p = warp; p < 2 * n; p += WARPS) {
        const int i = p >> 1;
        if (i >= a.slices && total * (x0 + i - a.slices) / extras == total * (x0 + i - a.slices + 1) / extras) continue;
        const long long place = 2LL * (i < a.slices ? block * a.slices + i : mains + (x0 + i - a.slices) + block) + (p & 1);
        const float4 s = a.stats[place * rows_a_block + own_row];
        lp_join(st, LpStats{s.x, s.y, s.z});
        if (a.top > 0) {
            const LpKey k = lane < a.top ? a.keys[(place * a.top + lane) * rows_a_block + own_row] : 0;
            keys = lp_merge(keys, k, lane);
        }
    }
    if (lane == 0) part[warp] = st;
    lists[warp][lane] = keys;
    __syncthreads();
    if (warp != 0) return;
    for (int w = 1; w < WARPS; ++w) {
        lp_join(st, part[w]);
        if (a.top > 0) keys = lp_merge(keys, lists[w][lane], lane);
    }
    const float log_s = logf(st.s);
    if (lane == 0) {
        o.entropy[row] = log_s - st.t / st.s;
        if (o.logprobs) {
            const int id = a.targets[row];
            const bool known = id < a.N;
            if (!known && a.status) atomicExch(a.status, RDL_FAULT_TARGET_ID);
            o.logprobs[row] = id < 0 ? 0.f : known ? (a.target_logit[row] - st.m) - log_s : NAN;
        }
    }
    if (lane < a.top) {
        o.top_ids[(long long)row * a.top + lane] = (int)lp_key_id(keys);
        o.top_logprobs[(long long)row * a.top + lane] = (keys >> 32) == 0 ? NAN : (lp_key_logit(keys) - st.m) - log_s;
    }
}

// how `rows` rows (as many as there are row blocks for) and the vocabulary are shared out
void plan(HeadArgs& a, int rows, int vocab, int ctas) {
    const int sms = rdl_sm_count(), at_once = sms / ctas > 0 ? sms / ctas : 1;
    a.M = rows;
    a.N = vocab;
    a.row_blocks = (int)(((long long)rows + BM * ctas - 1) / (BM * ctas));
    a.tiles_n = (int)(((long long)vocab + BN - 1) / BN);
    const long long tiles = (long long)a.row_blocks * a.tiles_n;
    a.groups = tiles < at_once ? (int)tiles : at_once;
    a.slices = a.groups / a.row_blocks;
    const int mains = a.slices * a.row_blocks;
    a.main_tiles = mains == a.groups ? a.tiles_n : (int)((long long)a.tiles_n * mains / a.groups);
}
int rows_at_once(int ctas) { return (rdl_sm_count() / ctas > 0 ? rdl_sm_count() / ctas : 1) * BM * ctas; }
int ctas_for(int rows) { return rows <= BM ? 1 : 2; }
// the rows of a launch: all, or equal parts where there are more row blocks than groups
int rows_a_launch(int rows, int ctas) {
    const long long most = rows_at_once(ctas), launches = (rows + most - 1) / most, blocks = ((long long)rows + BM * ctas - 1) / (BM * ctas);
    return launches <= 1 ? rows : (int)((blocks + launches - 1) / launches * BM * ctas);
}
struct Work { long long stats, keys, targets, bytes; };
Work work_of(const HeadArgs& a, int ctas, int top) {
    const long long slots = (long long)a.groups + a.row_blocks, places = slots * 2 * BM * ctas;
    Work w;
    w.stats = 0;
    w.keys = w.stats + places * (long long)sizeof(float4);
    w.targets = w.keys + places * top * (long long)sizeof(LpKey);
    w.bytes = w.targets + ((long long)a.M * 4 + 15) / 16 * 16;
    return w;
}

template <int CTAS, bool TOP>
int run(const CUtensorMap& mx, const CUtensorMap& mw, const HeadArgs& a, cudaStream_t st) {
    RDL_CUDA((rdl_allow_shared<head_logprobs_kernel<CTAS, TOP>>(SMEM_BYTES)), "linear_logprobs");
    RDL_CHECK_EX(rdl_launch_cluster(head_logprobs_kernel<CTAS, TOP>, dim3((unsigned)(a.groups * CTAS)), dim3(THREADS), CTAS, (size_t)SMEM_BYTES, st, mx, mw, a),
                 "linear_logprobs");
    return 0;
}

int bf16_map(CUtensorMap* map, const void* p, long long rows, long long cols, int box_rows, const char* what) {
    return mx_make_map(map, p, {CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, {(cuuint64_t)cols, (cuuint64_t)rows}, {(cuuint64_t)cols * 2}, {BK, (cuuint32_t)box_rows},
                                CU_TENSOR_MAP_SWIZZLE_128B}, what);
}

}  // namespace

extern "C" long long rdl_linear_logprobs_work_bytes(int rows, int vocab, int top) {
    if (rows <= 0 || vocab <= 0 || top < 0) return 0;
    HeadArgs a{};
    const int ctas = ctas_for(rows);
    plan(a, rows_a_launch(rows, ctas), vocab, ctas);
    return work_of(a, ctas, top).bytes;
}

extern "C" int rdl_linear_logprobs(const void* x, const void* w, int rows, int vocab, int k, const int* targets, int top, float softcap, float scale,
                                   float* logprobs, float* entropy, float* top_logprobs, int* top_ids, void* work, long long work_bytes, int* status,
                                   void* stream) {
    RDL_REQUIRE(rows >= 0 && vocab > 0 && k > 0 && k % 8 == 0, "linear_logprobs: rows=%d vocab=%d k=%d; k must be a multiple of 8", rows, vocab, k);
    RDL_REQUIRE(top >= 0 && top <= RDL_LOGPROBS_MAX_TOP && top <= vocab, "linear_logprobs: %d alternatives of %d tokens (%d at most)", top, vocab, RDL_LOGPROBS_MAX_TOP);
    RDL_REQUIRE(softcap >= 0.f, "linear_logprobs: soft-cap must not be negative");
    if (rows == 0) return 0;
    RDL_REQUIRE(x && w && entropy && (!targets || logprobs) && (top == 0 || (top_logprobs && top_ids)), "linear_logprobs: missing operand");
    RDL_REQUIRE((uintptr_t)x % 16 == 0 && (uintptr_t)w % 16 == 0, "linear_logprobs: operands must start on 16-byte boundaries");
    RDL_REQUIRE(work && (uintptr_t)work % 16 == 0 && work_bytes >= rdl_linear_logprobs_work_bytes(rows, vocab, top), "linear_logprobs: work space of %lld bytes is too small", work_bytes);
    const int ctas = ctas_for(rows), step = rows_a_launch(rows, ctas);
    CUtensorMap mw;
    if (int e = bf16_map(&mw, w, vocab, k, BN / ctas, "an output head")) return e;
    cudaStream_t st = (cudaStream_t)stream;
    for (long long r = 0; r < rows; r += step) {
        HeadArgs a{};
        plan(a, rows - r < step ? (int)(rows - r) : step, vocab, ctas);
        const Work space = work_of(a, ctas, top);
        a.kblocks = (k + BK - 1) / BK;
        a.top = top;
        const int lists = top ? (top + ASIDE) * EPI_THREADS * (int)sizeof(LpKey) : 0, fit = (SMEM_BYTES - 1024 - lists) / stage_bytes(ctas);
        a.stages = fit < MOST_STAGES ? fit : MOST_STAGES;
        a.cap = softcap;
        a.inv_cap = softcap > 0.f ? 1.f / softcap : 0.f;
        a.scale = scale;
        a.targets = targets ? targets + r : nullptr;
        a.stats = (float4*)((char*)work + space.stats);
        a.keys = (LpKey*)((char*)work + space.keys);
        a.target_logit = (float*)((char*)work + space.targets);
        a.wait_cycles = rdl_wait_cycles_for(RDL_FAULT_LOGPROBS_HEAD);
        a.test_extra_tx = rdl_test_extra_tx_for(RDL_FAULT_LOGPROBS_HEAD);
        a.status = status;
        CUtensorMap mx;
        if (int e = bf16_map(&mx, (const char*)x + r * k * 2, a.M, k, BM, "the rows")) return e;
        const int e = ctas == 1 ? (top ? run<1, true>(mx, mw, a, st) : run<1, false>(mx, mw, a, st)) : (top ? run<2, true>(mx, mw, a, st) : run<2, false>(mx, mw, a, st));
        if (e) return e;
        const JoinOut o{targets ? logprobs + r : nullptr, entropy + r, top ? top_logprobs + r * top : nullptr, top ? top_ids + r * top : nullptr};
        // a row has few partial results where there are many rows, and the other way round
        auto join = a.slices >= 16 ? head_join_kernel<16> : (a.slices >= 4 ? head_join_kernel<4> : head_join_kernel<1>);
        RDL_CHECK_EX(rdl_launch(join, dim3((unsigned)a.M), dim3(a.slices >= 16 ? 512u : a.slices >= 4 ? 128u : 32u), 0, st, a, BM * ctas, o), "linear_logprobs");
    }
    return 0;
}
