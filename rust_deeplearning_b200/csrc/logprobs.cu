// Log probabilities of given tokens, entropy and the largest logits of rows of logits, in one pass over the row.
#include "api.h"
#include "launch.cuh"
#include "logprobs.cuh"

namespace {

constexpr int LP_THREADS = 512, LP_WARPS = LP_THREADS / 32, LP_BATCH = 4;      // vectors a thread asks for before it uses the first

struct LpArgs {
    const void* z;
    long long row_stride;          // elements
    int rows, vocab, top;
    const int* targets;
    float* logprobs; float* entropy; float* top_logprobs; int* top_ids;
    int* status;
};

// 16 bytes of a row as floats
__device__ __forceinline__ void lp_load16(const float* p, float (&f)[4]) {
    const float4 v = __ldcs(reinterpret_cast<const float4*>(p));
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
}
__device__ __forceinline__ void lp_load16(const __nv_bfloat16* p, float (&f)[8]) {
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

// A warp's list of largest logits while a row passes by.  Logits not below `least` are put aside in shared memory; when there are 32
// of them they are sorted and merged into the list, whose last wanted place raises `least`: for itself, and through `shared_least` for
// the block's other warps, whose lists cannot hold less than that either.
// (called, not inlined: its 20 exchanges between lanes stand once in the kernel and not behind every logit of a batch)
__device__ __noinline__ LpKey lp_take(LpKey keys, LpKey* buffer, int n, int aside, int lane) {
    __syncwarp();
    const LpKey k = lane < n ? buffer[lane] : 0;
    const LpKey rest = lane < aside - n ? buffer[n + lane] : 0;
    __syncwarp();
    if (lane < aside - n) buffer[lane] = rest;
    return lp_merge(keys, lp_sort(k, lane), lane);
}

struct LpList {
    LpKey keys;                    // lane: its place's key
    float least;
    int aside;                     // how many are put aside
    LpKey* buffer;                 // 64
    unsigned* shared_least;        // order-preserving bits
    int top, lane;

    __device__ __forceinline__ void take(int n) {
        keys = lp_take(keys, buffer, n, aside, lane);
        aside -= n;
        const LpKey last = __shfl_sync(0xffffffffu, keys, top - 1);
        if (lane == 0) atomicMax(shared_least, (unsigned)(last >> 32));
        least = fmaxf(least, lp_key_logit(last));
    }
    // one logit a lane (or none)
    __device__ __forceinline__ void offer(float z, unsigned id, bool valid) {
        const bool in = valid && !(z < least);
        const unsigned mask = __ballot_sync(0xffffffffu, in);
        if (mask == 0) return;
        if (in) buffer[aside + __popc(mask & ((1u << lane) - 1))] = lp_key(z, id);
        aside += __popc(mask);
        if (aside >= 32) take(32);
    }
    __device__ __forceinline__ void look() {                      // what the block's other warps have found
        least = fmaxf(least, lp_key_logit((LpKey)(*(volatile unsigned*)shared_least) << 32));
    }
};

template <typename T, bool TOP>
__global__ void __launch_bounds__(LP_THREADS, 2) token_logprobs_kernel(LpArgs a) {
    constexpr int V = 16 / (int)sizeof(T);
    __shared__ LpStats part[LP_WARPS];
    __shared__ LpKey lists[TOP ? LP_WARPS : 1][TOP ? 64 : 1];
    __shared__ unsigned shared_least;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long row = blockIdx.x;
    if (threadIdx.x == 0) shared_least = 0;
    rdl_grid_wait();
    rdl_grid_launch_dependents();
    __syncthreads();
    const T* z = (const T*)a.z + row * a.row_stride;
    // columns before the first 16-byte boundary, whole vectors, columns behind the last
    const int head = min(a.vocab, (int)(((16 - ((uintptr_t)z & 15)) & 15) / sizeof(T)));
    const int vectors = (a.vocab - head) / V, tail = head + vectors * V;

    LpStats st = lp_empty();
    LpList list;
    if (TOP) list = {0, -INFINITY, 0, lists[warp], &shared_least, a.top, lane};
    if (warp == 0) {                                                 // fewer than 8 columns at either end
        const int i = lane < 16 ? lane : tail + lane - 16;
        const bool valid = lane < 16 ? lane < head : i < a.vocab;
        const float v = valid ? to_float<T>(z[i]) : -INFINITY;
        if (v > st.m) lp_move(st, v);
        const float one[1] = {v};
        if (valid) lp_add(st, one);
        if (TOP) list.offer(v, i, valid);
    }
    for (int first = 0; first < vectors; first += LP_THREADS * LP_BATCH) {
        float v[LP_BATCH][V];
#pragma unroll
        for (int j = 0; j < LP_BATCH; ++j) {
            const int at = first + j * LP_THREADS + (int)threadIdx.x;
            if (at < vectors) {
                lp_load16(z + head + (long long)at * V, v[j]);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) v[j][i] = -INFINITY;
            }
        }
        float most = v[0][0];
#pragma unroll
        for (int j = 0; j < LP_BATCH; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) most = fmaxf(most, v[j][i]);
        if (most > st.m) lp_move(st, most);
#pragma unroll
        for (int j = 0; j < LP_BATCH; ++j) lp_add(st, v[j]);
        if (TOP) {
            list.look();
            if (__any_sync(0xffffffffu, !(most < list.least))) {
#pragma unroll
                for (int j = 0; j < LP_BATCH; ++j) {
                    const int at = first + j * LP_THREADS + (int)threadIdx.x;
#pragma unroll
                    for (int i = 0; i < V; ++i) list.offer(v[j][i], head + at * V + i, at < vectors);
                }
            }
        }
    }
    if (TOP) {
        if (list.aside > 0) list.take(list.aside);
        __syncwarp();
        lists[warp][lane] = list.keys;
    }
    st = lp_warp_join(st);
    if (lane == 0) part[warp] = st;
    __syncthreads();
    if (TOP) {
#pragma unroll 1
        for (int n = LP_WARPS / 2; n > 0; n >>= 1) {
            if (warp < n) lists[warp][lane] = lp_merge(lists[warp][lane], lists[warp + n][lane], lane);
            __syncthreads();
        }
    }
    if (warp != 0) return;
    st = lp_warp_join(lane < LP_WARPS ? part[lane] : lp_empty());
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
    auto kernel = dtype == RDL_BF16 ? (top ? token_logprobs_kernel<__nv_bfloat16, true> : token_logprobs_kernel<__nv_bfloat16, false>)
                                    : (top ? token_logprobs_kernel<float, true> : token_logprobs_kernel<float, false>);
    RDL_CHECK_EX(rdl_launch(kernel, dim3((unsigned)rows), dim3(LP_THREADS), 0, (cudaStream_t)stream, a), "token_logprobs");
    return 0;
}
