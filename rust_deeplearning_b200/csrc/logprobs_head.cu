// Log probabilities, entropy and alternatives by the logits  z = scale * cap tanh(x W^T / cap)  of bfloat16 rows x behind an output head W
// [vocab, k], without logits in memory: the product runs on the fifth-generation tensor cores, and what takes a tile of it out
// of tensor memory keeps each row's statistics (logprobs.cuh) instead of storing it.
//
// A tile is 128 CTAS rows x 256 tokens.  CTAS 2 (many rows): a pair of blocks on two multiprocessors (cta_group::2); each holds 128 of
// the rows and 128 of the tile's weight rows, and the products, issued by a thread of block 0, read both halves.  CTAS 1: up to 128
// rows, where reading the weights is what takes the time, and where pairs would leave too much of their tiles empty.  Two accumulators:
// the products of a tile run while the tile before it is taken out.
//
// Persistent: a group (a pair, or a block) walks along the vocabulary for one block of rows, so that a row's statistics stay in one
// thread's registers.  Groups of all row blocks walk side by side over the same part of it (a slice), and their weight tiles come from
// memory once.  With B row blocks and P groups there are P / B slices; the P mod B groups over share the end of the vocabulary, all row blocks in
// turn, so that every group has as many tiles.  Each (row block, range) leaves partial results, which a second kernel joins.
//
// Warp 0 loads (TMA, a ring of stages of 64 k), warp 1 issues the products, eight warps take the accumulator out: two a quarter of
// tensor memory, half of the columns each, a row a thread.  Logits that may be among a row's largest are put aside in memory (`seen` below
// says which), and the second kernel looks among them.
//
// Measured, 256,000 tokens, k 2,304, soft-cap, calls in a graph, replayed once a while and (behind the stroke) for seconds: 8,192 rows and five alternatives
// 5.5 / 6.3 ms, 1.75 / 1.54 PFLOP/s; 2,048 rows, none, 1.37 / 1.58 ms, 1.76 / 1.53 PFLOP/s.  Over seconds the power limit leaves 1.43 to 1.49 GHz
// (sampled), at which a tile takes 20,600 to 21,700 cycles, its products 18,432.  What is done with a tile takes 5,000 cycles (9,000 with a soft-cap, up to
// 15,000 with alternatives) beside them.  64 rows: 187 us, 202 with 20 alternatives (a kernel more, a longer second kernel), 6.3 and 5.9 TB/s of weights.
// With alternatives a thread would like more than its 168 registers (three warps on a scheduler): 160 bytes a thread go to memory and back.
//
// Every wait is bounded; a block that gives up sets `status` and every path ends in the common tear-down.  A block takes all of a
// multiprocessor's shared memory (see "Tensor memory" in mx_tensor.cuh: nothing that holds tensor memory fits beside it).
#include "api.h"
#include "launch.cuh"
#include "logprobs.cuh"
#include "mx_tensor.cuh"

namespace {

constexpr int BM = 128, BN = 256, BK = 64, EPI_WARPS = 8, EPI_THREADS = EPI_WARPS * 32, THREADS = 64 + EPI_THREADS;
constexpr int AT_ONCE = 8;                                // logits of a row that are looked at together
constexpr int TMEM_COLS = 2 * BN;
constexpr int SMEM_BYTES = 232448 - 1024;                 // a block's limit less the static variables
__host__ __device__ constexpr int stage_bytes(int ctas) { return BM * BK * 2 + BN / ctas * BK * 2; }
__host__ __device__ constexpr int stages(int ctas) { return (SMEM_BYTES - 1024) / stage_bytes(ctas); }      // 7 of a pair, 4

struct HeadArgs {
    int M, N, kblocks;
    int row_blocks, tiles_n;                              // of 128 CTAS rows, of 256 tokens
    int groups, slices, main_tiles;                       // slices share the first main_tiles tiles of every row block
    int top, places;                                      // alternatives; logits a thread can put aside
    float cap, inv_cap, scale;
    const int* targets; float* target_logit;              // [M]
    float4* stats;                                        // [slot][column half][row of the block]: m, s, t, how many are put aside
    float2* aside;                                        // [slot][column half][row of the block][places]: a logit and its token
    LpKey* keys;                                          // [slot][column half][top][row of the block]: lists, where there are any
    unsigned* seen;                                       // [32][M]: what groups of a row's columns were seen to hold at most (order-preserving bits)
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

// ---- a row's largest logits, as one thread sees them ----

__device__ __forceinline__ void exchange(LpKey& a, LpKey& b) {      // the larger one first
    const LpKey x = a, y = b;
    a = x > y ? x : y;
    b = x > y ? y : x;
}
// 16 keys into descending order, from a sequence that falls and then rises
__device__ __forceinline__ void fall16(LpKey (&k)[16]) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if ((i & o) == 0) exchange(k[i], k[i + o]);
}

// Logits that may be among a row's largest are put aside in memory with their tokens, and the second kernel looks among them.  Should a thread
// have put aside as many as there is place for (its logits rise along the vocabulary or are equal, say), it makes them a sorted list there: `n` of
// them at `aside`, into `top` places `stride` keys apart, which `empty` says hold nothing yet.  Returns the last place's logit (NaN where there is none
// yet), which later ones must exceed: a thread comes to larger and larger tokens, so that equal ones are of no use.  (Without that every logit of
// a row of equal ones was put away: 2,048 x 2,304 x 32,000, five alternatives 1,400 us, not 230.)  Called, not inlined, and in loops: it is hardly ever needed, and what lies between
// the instructions that are makes those wait for theirs.
__device__ __noinline__ float put_away(LpKey* list, long long stride, const float2* aside, int n, int top, bool empty) {
#pragma unroll 1
    for (int done = 0; done < n; done += 16) {
        LpKey fresh[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) fresh[i] = done + i < n ? lp_key(aside[done + i].x, __float_as_uint(aside[done + i].y)) : 0;
#pragma unroll 1
        for (int r = 0; r < 8; ++r) {                      // neighbours against each other, 16 rounds in all
#pragma unroll
            for (int i = 0; i < 16; i += 2) exchange(fresh[i], fresh[i + 1]);
#pragma unroll
            for (int i = 1; i < 15; i += 2) exchange(fresh[i], fresh[i + 1]);
        }
#pragma unroll 1
        for (int first = 0; first < top; first += 16) {    // 16 places at a time: they keep the largest, the rest goes on
            LpKey held[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) held[i] = first + i < top && !(empty && done == 0) ? list[(first + i) * stride] : 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const LpKey a = held[i], b = fresh[15 - i];
                held[i] = a > b ? a : b;
                fresh[15 - i] = a > b ? b : a;
            }
            fall16(held);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (first + i < top) list[(first + i) * stride] = held[i];
            if (first + 16 < top) fall16(fresh);
        }
    }
    const LpKey last = list[(top - 1) * stride];
    return (last >> 32) == 0 ? NAN : lp_key_logit(last);
}

// A logit that is not below or equal to `least` (a NaN on either side passes), and its token, to `at`, which moves on; one lane as the
// other without a branch
__device__ __forceinline__ void put_aside(float2*& at, float v, float least, int token) {
    asm volatile("{\n.reg .pred p;\nsetp.gtu.f32 p, %1, %2;\n@p st.global.v2.b32 [%0], {%1, %3};\n@p add.s64 %0, %0, 8;\n}"
                 : "+l"(at) : "f"(v), "f"(least), "r"(token) : "memory");
}

__device__ __forceinline__ unsigned ordered(float z) {
    const unsigned u = __float_as_uint(z);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(unsigned o) { return o == 0 ? -INFINITY : __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }

// `least` rises to `now` where that is known and higher
__device__ __forceinline__ void begin_with(float& least, float now) {
    if (!(now < least) && now == now) least = now;
}
template <int N>
__device__ __forceinline__ float bound_among(float (&v)[N], int top) {
#pragma unroll 1
    for (int r = 0; r < N / 2; ++r) {                      // neighbours against each other, N rounds in all
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float hi = fmaxf(v[i], v[i + 1]);
            v[i + 1] = fminf(v[i], v[i + 1]);
            v[i] = hi;
        }
#pragma unroll
        for (int i = 1; i < N - 1; i += 2) {
            const float hi = fmaxf(v[i], v[i + 1]);
            v[i + 1] = fminf(v[i], v[i + 1]);
            v[i] = hi;
        }
    }
    float b = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) b = top - 1 == i ? v[i] : b;
    if (b == -INFINITY) return NAN;
    if (b == 0.f) return -__uint_as_float(1);
    return __uint_as_float(b > 0.f ? __float_as_uint(b) - 1 : __float_as_uint(b) + 1);
}
// What a logit must exceed.  A row's columns form 32 groups (by column mod 16, and by the half of the tile they lie in), and `seen` holds the largest logit that any block has seen of each
// so far.  At least `top` logits are not below the top-th of these 32, so that a logit below it is none of the row's `top` largest,
// whatever else comes.  When another block's numbers arrive does not change a result, only what is put aside.
//
// A thread keeps the maxima of what it has seen in registers, puts them in and takes the bound of all after its first tile (which it goes
// through a second time for what exceeds that), after its second and whenever its tiles are four times as many.  Of N logits in no order about 1.5 top / N of the next
// exceed the bound.  Measured instead, 2,048 rows and 20 alternatives: a sorted list a thread in shared memory (a call that merges 16 logits
// waits 10,000 cycles for its instructions) 1.8 ms, its logits alone in registers (2,000 instructions a piece of 32 columns) 4.1 ms.
//
// NaN where nothing is known; the number under the top-th value keeps logits that equal it.
__device__ __noinline__ float bound_of(const unsigned* seen, int rows, int top) {
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = from_ordered(__ldcg(seen + (long long)i * rows));
    if (top > 8) return bound_among(v, top);
    float w[16];                                           // few alternatives: 16 groups tell as much
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = fmaxf(v[i], v[i + 16]);
    return bound_among(w, top);
}

// Logits from their sums of products v: cap tanh(y), y = v / cap.  From |y| = 1/2 on cap - 2 cap / (e^(2 y) + 1), by the hardware's power and
// reciprocal (2^-22 and 2^-23 of themselves).  That form cancels around zero, so below it is v + v u P(u), u = y^2, with the cubic P whose largest
// relative error on that range is least (fitted to tanh(y) / y in long double: 2^-26).  Off by at most 4.5 * 2^-22 of the logit wherever it lies and
// whatever the cap (2.8 * 2^-22 where it is positive), so that small logits keep their order.  (The first form alone loses them, 2^-21 of the cap, and was no
// faster: 4,000 x 256 x 30,000 131 us, 512 x 2,304 x 256,000 with 20 alternatives 440 to 540 either way.  tanhf took 796 there.)
constexpr float TANH_SERIES = 0.5f, TANH_P0 = -0.33333144f, TANH_P1 = 0.13325879f, TANH_P2 = -0.05304549f, TANH_P3 = 0.01724149f;
__device__ __forceinline__ void logits_of(const HeadArgs& a, float (&v)[32]) {
    if (a.cap > 0.f) {
        const float c2 = -2.f * a.cap;
        const unsigned long long inv = lp_pair(a.inv_cap, a.inv_cap), two_log2e = lp_pair(2.f * LP_LOG2E, 2.f * LP_LOG2E), one = lp_pair(1.f, 1.f);
        const unsigned long long p0 = lp_pair(TANH_P0, TANH_P0), p1 = lp_pair(TANH_P1, TANH_P1), p2 = lp_pair(TANH_P2, TANH_P2), p3 = lp_pair(TANH_P3, TANH_P3);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            const unsigned long long w = lp_pair(v[i], v[i + 1]), y = lp_mul2(w, inv), u = lp_mul2(y, y);
            const unsigned long long near = lp_fma2(w, lp_mul2(u, lp_fma2(lp_fma2(lp_fma2(p3, u, p2), u, p1), u, p0)), w);
            float y0, y1, n0, n1, x0, x1, e0, e1, r0, r1;
            lp_unpair(y, y0, y1);
            lp_unpair(near, n0, n1);
            lp_unpair(lp_mul2(y, two_log2e), x0, x1);
            lp_unpair(lp_add2(lp_pair(lp_exp2(x0), lp_exp2(x1)), one), e0, e1);
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(e0));
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r1) : "f"(e1));
            v[i] = fabsf(y0) < TANH_SERIES ? n0 : fmaf(c2, r0, a.cap);
            v[i + 1] = fabsf(y1) < TANH_SERIES ? n1 : fmaf(c2, r1, a.cap);
        }
    }
    if (a.scale != 1.f) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] *= a.scale;
    }
}

template <int CTAS, bool TOP>
__global__ void __launch_bounds__(THREADS, 1) head_logprobs_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                                                                   const __grid_constant__ HeadArgs a) {
    constexpr int STAGE = stage_bytes(CTAS), STAGES = stages(CTAS), A_BYTES = BM * BK * 2, ROWS = BM * CTAS;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) unsigned long long full_bar[STAGES], empty_bar[STAGES], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up;
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = CTAS == 1 ? 0 : (int)(blockIdx.x & 1), group = blockIdx.x / CTAS;
    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int s = 0; s < STAGES; ++s) {
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
                    if (++s == STAGES) { s = 0; parity ^= 1; }
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
                    if (++s == STAGES) { s = 0; parity ^= 1; }
                }
                if (ok && mx_elect()) commit<CTAS>(mx_smem(&acc_full[buf]));
                __syncwarp();
            }
        }
    } else {
        // ---- statistics and lists: warp q of four has the lanes of rows 32 q + lane, and of two such warps each has half of the columns ----
        const int q = warp & 3, half = (warp - 2) >> 2, own_row = rank * BM + q * 32 + lane;
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
            const long long place = 2LL * slot + half;
            float2* const aside = a.aside + (TOP ? (place * ROWS + own_row) * a.places : 0);
            float2* at = aside;                           // where the next logit is put aside
            bool listed = false;                          // whether some have been put into a list
            float groups[TOP ? 16 : 1];                   // the largest of every group of this column half
            if (TOP)
#pragma unroll
                for (int j = 0; j < 16; ++j) groups[j] = -INFINITY;
            auto put_in = [&] {
#pragma unroll
                for (int j = 0; j < 16; ++j) atomicMax(a.seen + (long long)(half * 16 + j) * a.M + row, ordered(groups[j]));
            };
            for (int t = t0; t < t1; ++t, ++lt) {
                const int buf = lt & 1;
                if (!mx_warp_wait(mx_smem(&acc_full[buf]), (lt >> 1) & 1, a.wait_cycles, gave_up_v)) { ok = false; break; }
                mx_fence_after();
                const int n0 = t * BN + half * (BN / 2);
                const int since = t - t0;
                const bool two = TOP && since == 0;
                if (TOP && (since & 0x55555555) != 0 && (since & (since - 1)) == 0 && mine) {      // 1, 4, 16, ..
                    if (since > 1) put_in();
                    begin_with(least, bound_of(a.seen + row, a.M, a.top));
                }
#pragma unroll 1
                for (int i = two ? -4 : 0; i < 4; ++i) {
                    const int c = (i & 3) * 32, n = n0 + c, there = a.N - n;                 // columns from here on
                    if (two && i == 0 && mine) {
                        put_in();
                        begin_with(least, bound_of(a.seen + row, a.M, a.top));
                    }
                    float v[32];
                    if (any_row && there > 0) tmem_ld32(lanes + (uint32_t)(buf * BN + c), v);
                    if (i == 3) {                                // the last columns are in registers: the accumulator is free
                        mx_fence_before();
                        __syncwarp();
                        if (lane == 0) arrive_at(to_issuer + (uint32_t)(buf * 8));
                    }
                    if (!any_row || there <= 0) continue;
                    if (mine) logits_of(a, v);
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
                    float of[32 / AT_ONCE], most = -INFINITY;             // the largest of every few
#pragma unroll
                    for (int g = 0; g < 32 / AT_ONCE; ++g) {
                        of[g] = fmaxf(v[g * AT_ONCE], v[g * AT_ONCE + 1]);
#pragma unroll
                        for (int i = 2; i < AT_ONCE; i += 2) of[g] = lp_max3(of[g], v[g * AT_ONCE + i], v[g * AT_ONCE + i + 1]);
                        most = fmaxf(most, of[g]);
                    }
                    if (!two || i < 0) {
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
                        if (TOP)
#pragma unroll
                            for (int j = 0; j < 16; ++j) groups[j] = lp_max3(groups[j], v[j], v[j + 16]);
                    }
                    if (TOP && i >= 0 && __any_sync(0xffffffffu, !(most <= least))) {
#pragma unroll
                        for (int g = 0; g < 32; g += AT_ONCE) {
                            if (!__any_sync(0xffffffffu, !(of[g / AT_ONCE] <= least))) continue;
                            if (__any_sync(0xffffffffu, at > aside + (a.places - AT_ONCE))) {
                                if (mine && at > aside) {                  // a lane that has put nothing aside has no list either
                                    begin_with(least, put_away(a.keys + place * a.top * ROWS + own_row, ROWS, aside, (int)(at - aside), a.top, !listed));
                                    listed = true;
                                }
                                at = aside;
                            }
                            if (there >= 32) {
#pragma unroll
                                for (int j = g; j < g + AT_ONCE; ++j) put_aside(at, v[j], least, n + j);
                            } else {
#pragma unroll
                                for (int j = g; j < g + AT_ONCE; ++j)
                                    if (j < there) put_aside(at, v[j], least, n + j);
                            }
                        }
                    }
                    // The first 32 columns brought as many as there are alternatives, all above `least` (no NaN among them: s would be one): the lowest number
                    // above it is of no use to larger tokens.  That ends rows of equal logits at once.
                    if (two && i == 0 && mine && at - aside >= a.top && st.s == st.s && least < INFINITY) least = from_ordered(ordered(least) + 1);
                }
            }
            if (!ok) break;
            // with the statistics: how many logits have been put aside, one's complement where there is a list as well
            if (mine) a.stats[place * ROWS + own_row] = make_float4(st.m, st.s + s_low, st.t + t_low, __int_as_float(listed ? ~(int)(at - aside) : (int)(at - aside)));
        }
    }
    if (!ok && a.status) atomicExch(a.status, RDL_FAULT_LOGPROBS_HEAD);
    // ---- tear-down, reached by every thread ----
    mx_fence_before();
    __syncthreads();
    if (*gave_up_v) {                    // behind the barrier: whichever warp gave up, the loader has asked for its last copies by now
        rdl_drain_copies();
        __syncwarp();
    }
    if (CTAS == 2) cluster_sync();       // neither block leaves while the other may still read its shared memory or report to its barriers
    if (warp == 1) {
        if constexpr (CTAS == 1)
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// Nothing has been seen yet.
__global__ void __launch_bounds__(256) head_clear_kernel(unsigned* seen, long long n) {
    rdl_grid_wait();
    rdl_grid_launch_dependents();
    const long long i = blockIdx.x * 256LL + threadIdx.x;
    if (i < n) seen[i] = 0;
}

// ---- the partial results of a row, joined: a block a row ----

struct JoinOut { float* logprobs; float* entropy; float* top_logprobs; int* top_ids; };

// Partial results are shared out to the warps, a lane one.  What they have put aside is looked at 32 logits at a time, no matter whose they are.
template <int WARPS>
__global__ void __launch_bounds__(WARPS * 32) head_join_kernel(const __grid_constant__ HeadArgs a, int rows_a_block, JoinOut o) {
    __shared__ LpStats part[WARPS];
    __shared__ LpKey lists[WARPS][32], buffer[WARPS][64];
    __shared__ __align__(16) unsigned seen[WARPS][32];
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
    LpKey keys = 0, least = 0;
    const int n = 2 * (a.slices + x1 - x0);
    if (a.top > 0) {
        const unsigned own = a.seen[(long long)lane * a.M + row];      // what the 32 groups held in the end
        seen[warp][lane] = own;
        __syncwarp();
        least = lp_floor(lp_bound(seen[warp], own, a.top));
    }
    int aside = 0;                                         // keys above the bound that are not in the list yet
    auto take = [&](int count) {
        keys = lp_take(keys, buffer[warp], count, aside, lane);
        aside -= count;
        const LpKey last = __shfl_sync(0xffffffffu, keys, a.top - 1);
        least = last > least ? last : least;
    };
    auto offer = [&](LpKey key) {                          // a key a lane, or 0
        const bool in = key > least;
        const unsigned mask = __ballot_sync(0xffffffffu, in);
        if (mask == 0) return;
        if (in) buffer[warp][aside + __popc(mask & ((1u << lane) - 1))] = key;
        aside += __popc(mask);
        if (aside >= 32) take(32);
    };
    for (int first = warp * 32; first < n; first += WARPS * 32) {
        const int p = first + lane, i = p >> 1, x = x0 + i - a.slices;
        const bool there = p < n && (i < a.slices || total * x / extras != total * (x + 1) / extras);
        const long long place = (2LL * (i < a.slices ? block * a.slices + i : mains + x + block) + (p & 1)) * rows_a_block + own_row;
        int count = 0;
        if (there) {
            const float4 s = a.stats[place];
            lp_join(st, LpStats{s.x, s.y, s.z});
            count = __float_as_int(s.w);
        }
        if (a.top == 0) continue;
        const bool listed = count < 0;
        if (listed) count = ~count;
        count = min(count, a.places);                      // of a block that gave up there is anything here
        int upto = count;                                  // logits put aside by this lane's and the lanes before
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += v;
        }
        const int all = __shfl_sync(0xffffffffu, upto, 31);
        for (int e = 0; e < all; e += 32) {
            // whose is number e + lane: the first lane whose count reaches beyond it
            const int mine = e + lane;
            int owner = 0;
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) owner += __shfl_sync(0xffffffffu, upto, owner + d - 1) <= mine ? d : 0;
            const long long at = __shfl_sync(0xffffffffu, place, owner & 31);
            const int before = __shfl_sync(0xffffffffu, upto - count, owner & 31);
            LpKey key = 0;
            if (mine < all) {
                const float2 v = a.aside[at * a.places + (mine - before)];
                key = lp_key(v.x, __float_as_uint(v.y));
            }
            offer(key);
        }
        if (__any_sync(0xffffffffu, listed)) {
            const long long list = place - own_row;        // rows of the places before
            for (int k = 0; k < a.top; ++k) offer(listed ? a.keys[list * a.top + (long long)k * rows_a_block + own_row] : 0);
        }
    }
    if (aside > 0) take(aside);
    st = lp_warp_join(st);
    if (lane == 0) part[warp] = st;
    lists[warp][lane] = keys;
    __syncthreads();
#pragma unroll 1
    for (int w = WARPS / 2; w > 0; w >>= 1) {
        if (warp < w && a.top > 0) lists[warp][lane] = lp_merge(lists[warp][lane], lists[warp + w][lane], lane);
        if (WARPS > 1) __syncthreads();
    }
    if (warp != 0) return;
    keys = lists[0][lane];
    st = lp_warp_join(lane < WARPS ? part[lane] : lp_empty());
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
// Pairs from 129 rows on, but for three blocks of 128: as two of 256 a quarter of the products are for nobody (300 rows by pairs and without, 2,304 x
// 256,000: 382 and 342 us, 2,304 x 32,000 55 and 53, 256 x 30,000 20 and 18, 256 x 3,000 10.5 and 8.9; 384 rows within 0.3 us of each other at the
// smallest).  Blocks without a partner fetch half as much again (129 rows, 2,304 x 256,000: 218 us by pairs, 245 without; 200 rows, 256 x 30,000 with 20
// alternatives, where products are the least of it, 37 and 34; 2,048 rows 1.8 ms by pairs and 2.0 without).
int ctas_for(int rows) { return rows <= BM || (rows > 2 * BM && rows <= 3 * BM) ? 1 : 2; }
// the rows of a launch: all, or equal parts where there are more row blocks than groups
int rows_a_launch(int rows, int ctas) {
    const long long most = rows_at_once(ctas), launches = (rows + most - 1) / most, blocks = ((long long)rows + BM * ctas - 1) / (BM * ctas);
    return launches <= 1 ? rows : (int)((blocks + launches - 1) / launches * BM * ctas);
}
// About 1.5 top ln(tiles) are put aside where logits come in no order.
int places_for(int top) { return top ? 16 + 12 * top : 0; }
struct Work { long long stats, keys, aside, targets, seen, bytes; };
Work work_of(const HeadArgs& a, int ctas, int top) {
    const long long slots = (long long)a.groups + a.row_blocks, places = slots * 2 * BM * ctas;
    Work w;
    w.stats = 0;
    w.keys = w.stats + places * (long long)sizeof(float4);
    w.aside = w.keys + places * top * (long long)sizeof(LpKey);
    w.targets = w.aside + places * places_for(top) * (long long)sizeof(float2);
    w.seen = w.targets + ((long long)a.M * 4 + 15) / 16 * 16;
    w.bytes = w.seen + (top ? 32LL * a.M * 4 : 0);
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
        a.places = places_for(top);
        a.cap = softcap;
        a.inv_cap = softcap > 0.f ? 1.f / softcap : 0.f;
        a.scale = scale;
        a.targets = targets ? targets + r : nullptr;
        a.stats = (float4*)((char*)work + space.stats);
        a.keys = (LpKey*)((char*)work + space.keys);
        a.target_logit = (float*)((char*)work + space.targets);
        a.aside = (float2*)((char*)work + space.aside);
        a.seen = (unsigned*)((char*)work + space.seen);
        a.wait_cycles = rdl_wait_cycles_for(RDL_FAULT_LOGPROBS_HEAD);
        a.test_extra_tx = rdl_test_extra_tx_for(RDL_FAULT_LOGPROBS_HEAD);
        a.status = status;
        CUtensorMap mx;
        if (int e = bf16_map(&mx, (const char*)x + r * k * 2, a.M, k, BM, "the rows")) return e;
        if (top) RDL_CHECK_EX(rdl_launch(head_clear_kernel, dim3((unsigned)((32LL * a.M + 255) / 256)), dim3(256), 0, st, a.seen, 32LL * a.M), "linear_logprobs");
        const int e = ctas == 1 ? (top ? run<1, true>(mx, mw, a, st) : run<1, false>(mx, mw, a, st)) : (top ? run<2, true>(mx, mw, a, st) : run<2, false>(mx, mw, a, st));
        if (e) return e;
        const JoinOut o{targets ? logprobs + r : nullptr, entropy + r, top ? top_logprobs + r * top : nullptr, top ? top_ids + r * top : nullptr};
        // a row has few partial results where there are many rows, and the other way round
        const int warps = a.slices > 64 ? 16 : a.slices > 16 ? 4 : 1;
        auto join = warps == 16 ? head_join_kernel<16> : warps == 4 ? head_join_kernel<4> : head_join_kernel<1>;
        RDL_CHECK_EX(rdl_launch(join, dim3((unsigned)a.M), dim3(warps * 32u), 0, st, a, BM * ctas, o), "linear_logprobs");
    }
    return 0;
}
