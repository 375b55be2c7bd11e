// Log probabilities of given tokens, entropy and the largest logits of rows of logits, in one pass over the row.
//
// Memory bounds many rows (2,048 rows of 256,000 float32 logits: 2.1 GB), latency few of them.  A row belongs to a block, or to a cluster of 2, 4
// or 8 where there are fewer rows than the device has room for blocks.  A thread copies what it looks at into shared memory of its own,
// LP_RING batches ahead (cp.async), so that memory is kept busy while lists are sorted, and no thread waits for another's copy.
//
// Measured, calls in a graph, replayed once a while and (behind the stroke) for seconds, at the clock then sampled: 2,048 rows of 256,000, float32 303 / 302 us
// without alternatives (6.9 TB/s; 1.60 GHz), 314 / 322 with five (1.69), 323 / 345 with 20 (1.74; a logit takes 12 to 16 instructions, so that the
// multiprocessors are busy three quarters of the time); bfloat16 215 / 207, 240 / 229 and 322 / 309, at 1.85 to 1.97 GHz: those instructions.  8,192 rows of
// 32,000, float32 154, 173 and 231 us; of 1,000 10, 20 and 29 us.  One row of 32,000 3.9 us, with five alternatives 6.3; eight of 256,000 6.2 us, with 20 12:
// latency, of the lists at last.
#include "api.h"
#include "launch.cuh"
#include "logprobs.cuh"

namespace {

constexpr int LP_MAX_THREADS = 512, LP_MAX_WARPS = LP_MAX_THREADS / 32;
constexpr int LP_BATCH = 4, LP_RING = 3;                             // 16-byte vectors of a thread in a batch; batches on their way or looked at
constexpr int LP_THREAD_BYTES = LP_RING * LP_BATCH * 16;             // of the ring
constexpr int LP_LIST_BYTES = 64 / 32 * 8;                           // of its warp's list
constexpr int LP_MAX_CLUSTER = 8;

struct LpArgs {
    const void* z;
    long long row_stride;          // elements
    int rows, vocab, top;
    const int* targets;
    float* logprobs; float* entropy; float* top_logprobs; int* top_ids;
    int* status;
};

// 16 bytes of a row as floats
__device__ __forceinline__ void lp_widen(const uint4 v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void lp_widen(const uint4 v, float (&f)[8]) {
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void lp_copy16(unsigned to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void lp_copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void lp_copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// ---- the largest logits ----
//
// What a warp takes of its logits for the list.  A row's logits form 32 groups, by the lane that sees them; `seen` holds the largest
// one of each that the block's warps have put in.  At least `top` logits are not below the top-th of these, so that one below it is none of
// the row's largest.  A warp puts in what its lanes hold and takes the bound of all after its first batch and after every doubling of
// them; what is not below it is put aside, and one warp looks among it in the end.
// (Bounds that rose only with a warp's own sorted list let one or two logits of every 512 through, each of which costs its warp 200
// instructions: 393 us for five alternatives.)  Where a warp has put 32 aside it merges them into a list of its own.  A warp comes to larger
// and larger tokens, so that behind such a list equal logits are of no use either: rows of few allowed tokens, or of one value, would put every
// logit aside (2,048 rows of 256,000 with 10 allowed tokens 4,140 us, not 330).  What the list says is looked at once a vector: the lanes'
// tokens interleave within one, and after each of its logits it took longer (1,024 rows of 256,000 in bfloat16, 20 alternatives 184 us, not 166).
struct LpList {
    LpKey keys;                    // lane: its place's key
    float least;                   // what a logit must reach
    int aside;                     // how many are put aside
    LpKey* buffer;                 // 64
    unsigned* seen;                // 32, order-preserving bits
    int top, lane;
    int listed;                    // how often 32 have been merged into `keys`

    __device__ __forceinline__ void take(int n) {
        keys = lp_take(keys, buffer, n, aside, lane);
        aside -= n;
        ++listed;
    }
    // what follows are larger tokens than the list's
    __device__ __forceinline__ void beyond() { least = fmaxf(least, lp_key_beyond(__shfl_sync(0xffffffffu, keys, top - 1))); }
    // one logit a lane (or none)
    __device__ __forceinline__ void offer(float z, unsigned id, bool valid) {
        const bool in = valid && !(z < least);
        const unsigned mask = __ballot_sync(0xffffffffu, in);
        if (mask == 0) return;
        if (in) buffer[aside + __popc(mask & ((1u << lane) - 1))] = lp_key(z, id);
        aside += __popc(mask);
        if (aside >= 32) take(32);
    }
    // most: the largest logit that the lane has seen
    __device__ __forceinline__ void look(float most) {
        atomicMax(seen + lane, (unsigned)(lp_key(most, 0) >> 32));
        __syncwarp();
        const unsigned own = *(volatile unsigned*)(seen + lane);
        least = fmaxf(least, lp_key_logit((LpKey)lp_bound(seen, own, top) << 32));
    }
};

__device__ __forceinline__ unsigned lp_cluster_rank() {
    unsigned r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ unsigned lp_cluster_size() {
    unsigned r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void lp_cluster_sync() { asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory"); }
// a 32-bit word of the shared memory of the cluster's block `rank`
__device__ __forceinline__ unsigned lp_remote(const void* p, unsigned rank) {
    unsigned a, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((unsigned)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(LP_MAX_THREADS, 2) token_logprobs_kernel(LpArgs a) {
    constexpr int V = 16 / (int)sizeof(T);
    // [LP_RING][LP_BATCH][thread], then lists [warp][64]: no more than the block's warps need, since it bounds how many small blocks there are at once
    extern __shared__ uint4 ring[];
    __shared__ LpStats part[LP_MAX_WARPS];
    __shared__ __align__(16) unsigned seen[32];
    __shared__ int counts[LP_MAX_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, threads = blockDim.x, warps = threads >> 5;
    const unsigned rank = lp_cluster_rank(), size = lp_cluster_size();
    const long long row = blockIdx.x / size;
    LpKey (*lists)[64] = (LpKey (*)[64])(ring + threads * LP_RING * LP_BATCH);
    if (threadIdx.x < 32) seen[threadIdx.x] = 0;
    rdl_grid_wait();
    rdl_grid_launch_dependents();
    __syncthreads();
    const T* z = (const T*)a.z + row * a.row_stride;
    // columns before the first 16-byte boundary, whole vectors, columns behind the last; a block of a cluster has its part of the vectors
    const int head = min(a.vocab, (int)(((16 - ((uintptr_t)z & 15)) & 15) / sizeof(T)));
    const int all = (a.vocab - head) / V, tail = head + all * V;
    const int from = (int)((long long)all * rank / size), vectors = (int)((long long)all * (rank + 1) / size) - from;
    const T* body = z + head + (long long)from * V;
    const int body_id = head + from * V;

    const unsigned own = (unsigned)__cvta_generic_to_shared(ring + threadIdx.x);
    // a warp's vectors of a batch lie side by side (2 KB; with a block's threads side by side and a warp's vectors 8 KB apart 2,048 rows of 256,000
    // bfloat16 logits took 204 us, not 195)
    const int step = threads * LP_BATCH, mine = warp * 32 * LP_BATCH + lane;
    auto ask = [&](int first, int place) {
#pragma unroll
        for (int j = 0; j < LP_BATCH; ++j) {
            const int at = first + j * 32 + mine;
            if (at < vectors) lp_copy16(own + (unsigned)((place * LP_BATCH + j) * threads * 16), body + (long long)at * V);
        }
        lp_copies_end();
    };
#pragma unroll
    for (int r = 0; r < LP_RING - 1; ++r) ask(r * step, r);

    LpStats st = lp_empty();
    LpList list;
    if (TOP) list = {0, -INFINITY, 0, lists[warp], seen, a.top, lane, 0};
    int place = 0, batches = 0;
    for (int first = 0; first < vectors; first += step) {
        ask(first + (LP_RING - 1) * step, place == 0 ? LP_RING - 1 : place - 1);
        lp_copies_wait<LP_RING - 1>();
        float v[LP_BATCH][V];
        float most = -INFINITY;
#pragma unroll
        for (int j = 0; j < LP_BATCH; ++j) {
            if (first + j * 32 + mine < vectors) {
                lp_widen(ring[(place * LP_BATCH + j) * threads + threadIdx.x], v[j]);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) v[j][i] = -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < V; i += 2) most = lp_max3(most, v[j][i], v[j][i + 1]);
        }
        if (++place == LP_RING) place = 0;
        if (most > st.m) lp_move(st, most);
#pragma unroll
        for (int j = 0; j < LP_BATCH; ++j) lp_add(st, v[j]);
        if (TOP) {
            if ((batches & (batches - 1)) == 0) list.look(st.m > -FLT_MAX ? st.m : -INFINITY);
            ++batches;
            if (__any_sync(0xffffffffu, !(most < list.least))) {
#pragma unroll
                for (int j = 0; j < LP_BATCH; ++j) {
                    float of_vector = -INFINITY;             // few vectors of a batch have one (8,192 rows of 32,000 in bfloat16: 236 -> 214 us)
#pragma unroll
                    for (int i = 0; i < V; i += 2) of_vector = lp_max3(of_vector, v[j][i], v[j][i + 1]);
                    if (!__any_sync(0xffffffffu, !(of_vector < list.least))) continue;
                    const int at = first + j * 32 + mine;
                    const int listed = list.listed;
#pragma unroll
                    for (int i = 0; i < V; ++i) list.offer(v[j][i], body_id + at * V + i, at < vectors);
                    if (list.listed != listed) list.beyond();
                }
            }
        }
    }
    if (warp == 0 && rank == 0) {                                    // fewer than 8 columns at either end
        const int i = lane < 16 ? lane : tail + lane - 16;
        const bool valid = lane < 16 ? lane < head : i < a.vocab;
        const float v = valid ? to_float<T>(z[i]) : -INFINITY;
        if (v > st.m) lp_move(st, v);
        const float one[2] = {v, -INFINITY};
        if (valid) lp_add(st, one);
        if (TOP) {
            if (list.listed) list.least = -INFINITY;                 // smaller tokens than the list's among them
            list.offer(v, i, valid);
        }
    }
    if (TOP) {
        if (list.listed) {
            if (list.aside > 0) list.take(list.aside);
            __syncwarp();
            lists[warp][lane] = list.keys;
            list.aside = 32;
        }
        if (lane == 0) counts[warp] = list.aside;
    }
    st = lp_warp_join(st);
    if (lane == 0) part[warp] = st;
    __syncthreads();
    if (warp == 0) {
        st = lp_warp_join(lane < warps ? part[lane] : lp_empty());
        if (lane == 0) part[0] = st;
        if (TOP) {
            // what the warps have put aside, 32 keys at a time, no matter whose they are
            int upto = lane < warps ? counts[lane] : 0;
            const int count = upto;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= d) upto += v;
            }
            const int all_keys = __shfl_sync(0xffffffffu, upto, 31);
            LpKey keys = 0, least = 0;
#pragma unroll 1
            for (int e = 0; e < all_keys; e += 32) {
                const int mine = e + lane;
                int owner = 0;
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) owner += __shfl_sync(0xffffffffu, upto, owner + d - 1) <= mine ? d : 0;
                const int before = __shfl_sync(0xffffffffu, upto - count, owner & 31);
                const LpKey key = mine < all_keys ? lists[owner][mine - before] : 0;
                if (!__any_sync(0xffffffffu, key > least)) continue;
                keys = lp_merge(keys, lp_sort(key, lane), lane);
                least = __shfl_sync(0xffffffffu, keys, a.top - 1);
            }
            __syncwarp();
            lists[0][lane] = keys;
            __syncwarp();
        }
    }
    if (size > 1) {                                                  // the cluster's blocks, a warp of the first for each
        lp_cluster_sync();
        if (rank == 0 && warp > 0 && warp < (int)size) {
            if (TOP) {
                const LpKey lo = lp_remote((const unsigned*)&lists[0][lane], warp), hi = lp_remote((const unsigned*)&lists[0][lane] + 1, warp);
                lists[warp][lane] = hi << 32 | lo;
            }
            if (lane < 3) ((unsigned*)&part[warp])[lane] = lp_remote((const unsigned*)&part[0] + lane, warp);
        }
        __syncthreads();
        if (TOP && rank == 0) {
#pragma unroll 1
            for (int n = (int)size / 2; n > 0; n >>= 1) {
                if (warp < n) lists[warp][lane] = lp_merge(lists[warp][lane], lists[warp + n][lane], lane);
                __syncthreads();
            }
        }
        lp_cluster_sync();                                           // no block leaves while its memory may be read
        if (rank != 0) return;
        if (warp == 0) st = lp_warp_join(lane < (int)size ? part[lane] : lp_empty());
    }
    if (warp != 0) return;
    const float log_s = logf(st.s);
    if (lane == 0) {
        a.entropy[row] = log_s - st.t / st.s;
        if (a.targets) {
            const int id = a.targets[row];
            const bool known = id < a.vocab;
            if (!known && a.status) atomicExch(a.status, RDL_FAULT_TARGET_ID);
            a.logprobs[row] = id < 0 ? 0.f : known ? (to_float<T>(z[id]) - st.m) - log_s : NAN;
        }
    }
    if (TOP && lane < a.top) {
        const LpKey k = lists[0][lane];
        a.top_ids[row * a.top + lane] = (int)lp_key_id(k);
        a.top_logprobs[row * a.top + lane] = (k >> 32) == 0 ? NAN : (lp_key_logit(k) - st.m) - log_s;
    }
}

template <typename T, bool TOP>
int lp_run(const LpArgs& a, int cluster, int threads, cudaStream_t st) {
    constexpr int BYTES = LP_THREAD_BYTES + (TOP ? LP_LIST_BYTES : 0);
    RDL_CUDA((rdl_allow_shared<token_logprobs_kernel<T, TOP>>(LP_MAX_THREADS * BYTES)), "token_logprobs");
    RDL_CHECK_EX(rdl_launch_cluster(token_logprobs_kernel<T, TOP>, dim3((unsigned)a.rows * cluster), dim3(threads), cluster, (size_t)threads * BYTES, st, a),
                 "token_logprobs");
    return 0;
}

}  // namespace

extern "C" int rdl_token_logprobs(const void* logits, int dtype, long long row_stride, int rows, int vocab, const int* targets, int top, float* logprobs,
                                  float* entropy, float* top_logprobs, int* top_ids, int* status, void* stream) {
    RDL_REQUIRE(rdl_valid_dtype(dtype), "token_logprobs: bad dtype %d", dtype);
    RDL_REQUIRE(rows >= 0 && vocab > 0 && row_stride >= 0, "token_logprobs: %d rows of %d logits", rows, vocab);
    RDL_REQUIRE(top >= 0 && top <= RDL_LOGPROBS_MAX_TOP && top <= vocab, "token_logprobs: %d alternatives of %d tokens (%d at most)", top, vocab, RDL_LOGPROBS_MAX_TOP);
    if (rows == 0) return 0;
    RDL_REQUIRE(logits && entropy && (!targets || logprobs) && (top == 0 || (top_logprobs && top_ids)), "token_logprobs: missing operand");
    RDL_REQUIRE((uintptr_t)logits % rdl_dtype_size(dtype) == 0, "token_logprobs: logits that are not on an element's boundary");
    const LpArgs a{logits, row_stride, rows, vocab, top, targets, logprobs, entropy, top_logprobs, top_ids, status};
    // Few rows: as many blocks share a row as there is room for at once (two on a multiprocessor), each thread with a batch where the row has one.
    // More: as many threads a row as keep the device about full, or as leave each 16 batches (8 without alternatives), since what a warp
    // does once for a row takes as long as one or two of them (five alternatives: 600 rows of 32,000 22 us with 256 threads, 25 with 64, 35 with 32;
    // 4,000 rows 94 us with 64, 104 with 256).
    const long long vectors = (long long)vocab * (long long)rdl_dtype_size(dtype) / 16;
    const long long room = (long long)rdl_sm_count() * 2 * LP_MAX_THREADS;
    int threads = 32, cluster = 1;
    while (threads < LP_MAX_THREADS && vectors >= threads * 2LL * LP_BATCH
           && (3LL * rows * threads <= 2 * room || vectors >= threads * 2LL * LP_BATCH * (top ? 16 : 8))) threads *= 2;
    while (cluster < LP_MAX_CLUSTER && (long long)rows * cluster * 2 <= 2 * rdl_sm_count() && vectors >= cluster * 2LL * LP_MAX_THREADS) cluster *= 2;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == RDL_BF16) return top ? lp_run<__nv_bfloat16, true>(a, cluster, threads, st) : lp_run<__nv_bfloat16, false>(a, cluster, threads, st);
    return top ? lp_run<float, true>(a, cluster, threads, st) : lp_run<float, false>(a, cluster, threads, st);
}
