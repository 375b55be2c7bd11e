// What the kernels that turn logits into log probabilities share: the running statistics of a row, and the list of its
// largest logits.
//
// Of logits z with largest value m:  s = sum exp(z - m),  t = sum (z - m) exp(z - m);  the log probability of token i is
// z_i - m - ln s and the entropy ln s - t / s (every term relative to m, so that nothing cancels).  Two parts of a row with statistics of
// their own join by moving both to the larger m:  exp(z - M) = exp(z - m) exp(m - M),  (z - M) = (z - m) + (m - M).
// A logit of minus infinity (a forbidden token) adds nothing; a NaN or plus infinity makes s NaN, and a row of nothing but minus
// infinities has s = 0 and gives NaN as well: there is no distribution.  m starts at the lowest finite value, so that a row
// masked with that value is uniform.
//
// A logit and its id are one 64-bit key whose order is the order of the alternatives: larger logits first, of equal logits the lowest id
// first, NaN behind everything.  Keys of a row are distinct; 0 is no key.
#pragma once

#include <float.h>

#include "common.cuh"

#define RDL_LOGPROBS_MAX_TOP 32       // alternatives: a key a lane

namespace {

constexpr float LP_LOG2E = 1.4426950408889634f;

struct LpStats { float m, s, t; };

__device__ __forceinline__ LpStats lp_empty() { return {-FLT_MAX, 0.f, 0.f}; }

// 2^x: two units in the last place (the hardware's), 0 below 2^-126 (numbers that are not normal would take four instructions instead of one,
// and none of them counts beside the 1 of a row's largest logit)
__device__ __forceinline__ float lp_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// the statistics seen from a larger maximum; the lower bound keeps 0 * infinity out (what it cuts off is multiplied by 2^-huge = 0)
__device__ __forceinline__ void lp_move(LpStats& a, float m) {
    const float d = fmaxf(a.m - m, -1e30f), c = lp_exp2(d * LP_LOG2E);
    a.t = c * fmaf(a.s, d, a.t);
    a.s *= c;
    a.m = m;
}

__device__ __forceinline__ void lp_join(LpStats& a, LpStats b) {
    const float m = fmaxf(a.m, b.m);
    lp_move(a, m);
    lp_move(b, m);
    a.s += b.s;
    a.t += b.t;
}

// two floats in a register pair, and arithmetic on both at once
__device__ __forceinline__ unsigned long long lp_pair(float a, float b) {
    unsigned long long p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ void lp_unpair(unsigned long long p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ unsigned long long lp_add2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long lp_mul2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long lp_fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// the largest of three (a NaN is passed over, as by fmaxf)
__device__ __forceinline__ float lp_max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// N logits more, an even number of them; m is not below any
template <int N>
__device__ __forceinline__ void lp_add(LpStats& a, const float (&z)[N]) {
    const unsigned long long less = lp_pair(-a.m, -a.m), log2e = lp_pair(LP_LOG2E, LP_LOG2E);
    unsigned long long s = 0, t = 0;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const unsigned long long d = lp_add2(lp_pair(z[i], z[i + 1]), less);
        float d0, d1, x0, x1;
        lp_unpair(d, d0, d1);
        lp_unpair(lp_mul2(d, log2e), x0, x1);
        const unsigned long long e = lp_pair(lp_exp2(x0), lp_exp2(x1));
        s = lp_add2(s, e);
        t = lp_fma2(e, lp_pair(fmaxf(d0, -1e30f), fmaxf(d1, -1e30f)), t);
    }
    float s0, s1, t0, t1;
    lp_unpair(s, s0, s1);
    lp_unpair(t, t0, t1);
    a.s += s0 + s1;
    a.t += t0 + t1;
}

__device__ __forceinline__ LpStats lp_warp_join(LpStats a) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const LpStats b = {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.t, o)};
        lp_join(a, b);
    }
    return a;
}

typedef unsigned long long LpKey;

__device__ __forceinline__ LpKey lp_key(float z, unsigned id) {
    const unsigned u = __float_as_uint(z + 0.0f);               // -0 and +0 are one value
    const unsigned o = z != z ? 0u : (u & 0x80000000u ? ~u : u | 0x80000000u);
    return (LpKey)o << 32 | (unsigned)~id;
}
// the logit of a key (minus infinity for no key and for a NaN's)
__device__ __forceinline__ float lp_key_logit(LpKey k) {
    const unsigned o = (unsigned)(k >> 32);
    return o == 0 ? -INFINITY : __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ unsigned lp_key_id(LpKey k) { return ~(unsigned)k; }
// the least logit that comes before a key's at any larger id (minus infinity for no key and for a NaN's: every number does)
__device__ __forceinline__ float lp_key_beyond(LpKey k) {
    const unsigned o = (unsigned)(k >> 32);
    return o == 0 ? -INFINITY : o >= 0xff800000u ? INFINITY : lp_key_logit(k + (1ull << 32));
}

// A warp's list: 32 keys, a lane each, largest in lane 0.

// descending order over the lanes of a sequence that first falls and then rises, or the other way round (bitonic)
__device__ __forceinline__ LpKey lp_bitonic(LpKey k, int lane) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const LpKey other = __shfl_xor_sync(0xffffffffu, k, o);
        const bool first = (lane & o) == 0;                     // the place that gets the larger one
        k = (k > other) == first ? k : other;
    }
    return k;
}
// any 32 keys, 0 for none; keys may not repeat but for 0
__device__ __forceinline__ LpKey lp_sort(LpKey k, int lane) {
#pragma unroll
    for (int n = 2; n <= 32; n <<= 1) {
#pragma unroll
        for (int o = n >> 1; o > 0; o >>= 1) {
            const LpKey other = __shfl_xor_sync(0xffffffffu, k, o);
            const bool larger = ((lane & o) == 0) == ((lane & n) == 0 || n == 32);
            k = (k > other) == larger ? k : other;
        }
    }
    return k;
}
// the 32 largest of two sorted lists
__device__ __forceinline__ LpKey lp_merge(LpKey a, LpKey b, int lane) {
    const LpKey r = __shfl_sync(0xffffffffu, b, 31 - lane);
    return lp_bitonic(a > r ? a : r, lane);
}

// Keys put aside, the first n <= 32 of them, into a warp's list; what is left of `aside` < 64 moves to the front.  (Called, not inlined: the 20
// exchanges between lanes stand once in a kernel and not behind every place that puts something aside.)
__device__ __noinline__ LpKey lp_take(LpKey keys, LpKey* buffer, int n, int aside, int lane) {
    __syncwarp();
    const LpKey k = lane < n ? buffer[lane] : 0;
    const LpKey rest = lane < aside - n ? buffer[n + lane] : 0;
    __syncwarp();
    if (lane < aside - n) buffer[lane] = rest;
    return lp_merge(keys, lp_sort(k, lane), lane);
}

// The largest of 32 values (16-byte aligned in shared memory, order-preserving bits, own: the lane's) that at least `top` of them are not below,
// by counting: 8 reads and 32 comparisons a lane, where a sort of them is 15 exchanges, one after another.
__device__ __forceinline__ unsigned lp_bound(const unsigned* seen, unsigned own, int top) {
    const unsigned at = (unsigned)__cvta_generic_to_shared(seen);
    int n = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        unsigned v[4];
        asm volatile("ld.volatile.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at + 16 * i) : "memory");
#pragma unroll
        for (int j = 0; j < 4; ++j) n += v[j] >= own;
    }
    return __reduce_max_sync(0xffffffffu, n >= top ? own : 0u);
}
// the key that the largest ones of 32 groups with that bound are above
__device__ __forceinline__ LpKey lp_floor(unsigned bound) {
    return bound > (unsigned)(lp_key(-INFINITY, 0) >> 32) ? ((LpKey)bound << 32) - 1 : 0;
}

}  // namespace
