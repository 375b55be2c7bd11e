// Rows and weights into the microscaling formats (microscaling.cuh), and weights back.
//
// rdl_norm_mx8: what stands before a product of 8-bit rows, in one pass over the row:
//     t = first ? rms_norm(x; first) : x;  h = residual + t (written to residual_out);  y = second ? rms_norm(h; second) : h
//     y -> e4m3 with a scale a group
// Bound by memory: x is read once, the residual read and written once, a byte a column is written.  A block takes a row, held in
// registers between its passes (rows of up to 8,192 columns; wider ones are read again).  A thread holds four neighbouring columns, so
// a group is eight lanes of a warp and a block of 128 columns one warp: the largest magnitude is three shuffles away and the four
// scale codes of a block leave as one word.  The threads a row gets depend on its width alone, so its result does
// not depend on how many rows a step has.
// Measured: 8,192 float32 rows of 4,608 (492 MB) 75.6 us, 6.5 TB/s; 2,048 bfloat16 rows of 2,304 with both norms (52 MB) 11.2 us; 17 rows 3.5 us.
//
// rdl_pack_mx4: a matrix to 4 bits, padding and all.  Memory bound: 36,864 x 4,608 bfloat16 (430 MB) 76 us, 5.7 TB/s.
// rdl_lay_mx4, rdl_lay_mx8: a matrix or rows that came in these formats, to the products' layout: 36,864 x 4,608 codes
// (180 MB) 52 us, 3.5 TB/s; 8,192 rows of 4,608 in 8 bits (78 MB) 15.6 us, 5.0 TB/s.
// rdl_expand_mx4: the values the codes stand for; exact in bfloat16 for scales from 2^-125 up to 2^125.  The same matrix 71 us, 6.1 TB/s.
#include <cuda_fp16.h>

#include "api.h"
#include "launch.cuh"
#include "microscaling.cuh"
#include "mx_tensor.cuh"
#include "row_vec.cuh"

namespace {

struct NormMxArgs {
    const void* x; int x_dtype;
    const void* w1; int w1_dtype; float eps1, off1;
    const float* res; float* res_out;
    const void* w2; int w2_dtype; float eps2, off2;
    uint8_t* values; uint8_t* scales;
    int rows, width, blocks, padded_rows;
};

// 1 / sqrt(sum over the block / n + eps) for every thread; `part` holds a float a warp and is used for this sum alone, so that one barrier
// is enough.  The order of additions depends on the block's size alone.  The hardware's reciprocal root and one Newton step: an
// error of this factor would move every value of the row the same way, and 8-bit codes with them.
__device__ __forceinline__ float row_factor(float v, float* part, int n, float eps) {
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    const int warps = blockDim.x >> 5;
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w)
        if (w < warps) t += part[w];
    const float a = t / (float)n + eps, r = rsqrtf(a);
    const float step = 0.5f * r * fmaf(-(a * r), r, 1.0f);
    return a > 0.f && isfinite(a) && isfinite(r) ? r + step : r;      // nothing to mend of an infinity or a NaN
}

// four consecutive columns from column c of a row that starts at element `base`; zeros beyond the width
template <bool VEC>
__device__ __forceinline__ void load_columns(const void* p, long long base, int c, int width, int dtype, float (&v)[4]) {
    if (VEC) {
        if (c < width) rn_load4(p, base + c, dtype, v);
        else v[0] = v[1] = v[2] = v[3] = 0.f;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = c + k < width ? rdl_load(p, base + c + k, dtype) : 0.f;
    }
}

// a warp's 128 columns of one row, four a lane: codes and the block's four scale codes
__device__ __forceinline__ void store_block(const float (&v)[4], uint8_t* values, uint8_t* scales, int lane) {
    float m = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) m = mx_larger(m, v[k]);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) m = mx_larger(m, __shfl_xor_sync(0xffffffffu, m, o));
    const uint32_t c = mx8_scale_code(m);
    const float inv = mx_inverse_scale(c);
    *reinterpret_cast<uint32_t*>(values + lane * 4) = mx_to_e4m3(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
    uint32_t word = c << (lane & 24);                       // the group's byte of the word
    word |= __shfl_xor_sync(0xffffffffu, word, 8);
    word |= __shfl_xor_sync(0xffffffffu, word, 16);
    if (lane == 0) *reinterpret_cast<uint32_t*>(scales) = word;
}

// HALF: bfloat16 rows, kept as they are between the passes: two registers a group of four columns, which lets one block more run.
template <int ITER, bool VEC, bool HALF>
__global__ void __launch_bounds__(256, ITER <= 4 ? 5 : (ITER <= 6 ? 4 : 3)) norm_mx8_kernel(const __grid_constant__ NormMxArgs a) {
    static_assert(VEC || !HALF, "rows of any width are read value by value");
    __shared__ float part[2][8];
    rdl_grid_wait();
    rdl_grid_launch_dependents();
    const int r = blockIdx.x, lane = threadIdx.x & 31;
    const long long base = (long long)r * a.width;
    uint2 raw[HALF ? ITER : 1];
    float v[ITER][4];                                       // HALF: the residual, then the sum; else x, then the sum
    float h[HALF ? 1 : ITER][4];                            // the residual
    auto column = [&](int i) { return (i * (int)blockDim.x + (int)threadIdx.x) * 4; };
    auto value = [&](int i, float (&x)[4]) {                // x as float
        if (HALF) {
            const uint2 w = raw[HALF ? i : 0];
            x[0] = __uint_as_float(w.x << 16); x[1] = __uint_as_float(w.x & 0xffff0000u); x[2] = __uint_as_float(w.y << 16); x[3] = __uint_as_float(w.y & 0xffff0000u);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = v[i][k];
        }
    };
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int c = column(i);
        if (HALF) raw[HALF ? i : 0] = c < a.width ? *reinterpret_cast<const uint2*>((const __nv_bfloat16*)a.x + base + c) : make_uint2(0, 0);
        else load_columns<VEC>(a.x, base, c, a.width, a.x_dtype, v[i]);
        float (&res)[4] = HALF ? v[i] : h[HALF ? 0 : i];
        if (a.res) load_columns<VEC>(a.res, base, c, a.width, RDL_F32, res);
        else res[0] = res[1] = res[2] = res[3] = 0.f;
    }
    float inv = 1.f;
    if (a.w1) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            float x[4];
            value(i, x);
#pragma unroll
            for (int k = 0; k < 4; ++k) ss = fmaf(x[k], x[k], ss);
        }
        inv = row_factor(ss, part[0], a.width, a.eps1);
    }
    float s2 = 0.f;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int c = column(i);
        float x[4];
        value(i, x);
        if (a.w1) {
            float w[4];
            load_columns<VEC>(a.w1, 0, c, a.width, a.w1_dtype, w);
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = x[k] * inv * (w[k] + a.off1);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[i][k] = a.res ? (HALF ? v[i][k] : h[HALF ? 0 : i][k]) + x[k] : x[k];
            s2 = fmaf(v[i][k], v[i][k], s2);
        }
        if (a.res_out) {
            if (VEC) {
                if (c < a.width) rn_store4(a.res_out + base + c, v[i]);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (c + k < a.width) a.res_out[base + c + k] = v[i][k];
            }
        }
    }
    const float inv2 = a.w2 ? row_factor(s2, part[1], a.width, a.eps2) : 1.f;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int c = column(i);
        const int block = c / MX_BLOCK;                     // one for the whole warp
        if (block >= a.blocks) break;
        if (a.w2) {
            float w[4];
            load_columns<VEC>(a.w2, 0, c, a.width, a.w2_dtype, w);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[i][k] = c + k < a.width ? v[i][k] * inv2 * (w[k] + a.off2) : 0.f;
        }
        store_block(v[i], a.values + (long long)r * a.blocks * MX_BLOCK + block * MX_BLOCK,
                    a.scales + ((long long)block * a.padded_rows + r) * 4, lane);
    }
}

// Rows wider than the registers of a block: the row is read once a pass.
template <bool VEC>
__global__ void __launch_bounds__(256) norm_mx8_wide_kernel(const __grid_constant__ NormMxArgs a) {
    __shared__ float part[2][8];
    rdl_grid_wait();
    rdl_grid_launch_dependents();
    const int r = blockIdx.x, lane = threadIdx.x & 31, step = blockDim.x * 4;
    const long long base = (long long)r * a.width;
    float inv = 1.f;
    if (a.w1) {
        float ss = 0.f;
        for (int c = threadIdx.x * 4; c < a.width; c += step) {
            float v[4];
            load_columns<VEC>(a.x, base, c, a.width, a.x_dtype, v);
#pragma unroll
            for (int k = 0; k < 4; ++k) ss = fmaf(v[k], v[k], ss);
        }
        inv = row_factor(ss, part[0], a.width, a.eps1);
    }
    // h of four columns: the sum of x's norm and the residual
    auto sum_at = [&](int c, float (&v)[4]) {
        load_columns<VEC>(a.x, base, c, a.width, a.x_dtype, v);
        if (a.w1) {
            float w[4];
            load_columns<VEC>(a.w1, 0, c, a.width, a.w1_dtype, w);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = v[k] * inv * (w[k] + a.off1);
        }
        if (a.res) {
            float h[4];
            load_columns<VEC>(a.res, base, c, a.width, RDL_F32, h);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = h[k] + v[k];
        }
    };
    float s2 = 0.f;
    if (a.w2 || a.res_out) {
        for (int c = threadIdx.x * 4; c < a.width; c += step) {
            float v[4];
            sum_at(c, v);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                s2 = fmaf(v[k], v[k], s2);
                if (a.res_out && c + k < a.width) a.res_out[base + c + k] = v[k];
            }
        }
    }
    float inv2 = 1.f;
    if (a.w2) inv2 = row_factor(s2, part[1], a.width, a.eps2);
    for (int c = threadIdx.x * 4; c < a.blocks * MX_BLOCK; c += step) {      // whole warps: both sides are multiples of 128
        float v[4];
        // the sum may have replaced the residual it was formed from: this thread reads what it wrote itself
        if (a.res_out) load_columns<VEC>(a.res_out, base, c, a.width, RDL_F32, v);
        else sum_at(c, v);
        if (a.w2) {
            float w[4];
            load_columns<VEC>(a.w2, 0, c, a.width, a.w2_dtype, w);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = c + k < a.width ? v[k] * inv2 * (w[k] + a.off2) : 0.f;
        }
        const int block = c / MX_BLOCK;
        store_block(v, a.values + (long long)r * a.blocks * MX_BLOCK + block * MX_BLOCK,
                    a.scales + ((long long)block * a.padded_rows + r) * 4, lane);
    }
}

// Packing and expanding: a block takes a tile of 128 x 128, 8 warps two rows at a time, a lane eight columns of one: 256 bytes of bfloat16
// and 64 bytes of codes of a row in one piece, four rows of a lane in flight.
constexpr int TILE_AHEAD = 4;

struct PackArgs {
    const void* w; int dtype;
    uint8_t* codes; uint8_t* scales;
    int rows, columns, blocks, half;                        // half: outputs of a [gate; up] matrix, 0: not one
};

// VEC 2: bfloat16 rows of whole 16-byte pieces; 1: rows of whole groups of four columns; 0: any
template <int VEC>
__global__ void __launch_bounds__(256) pack_mx4_kernel(const __grid_constant__ PackArgs a) {
    rdl_grid_wait();
    rdl_grid_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int tile = blockIdx.x / a.blocks, block = blockIdx.x - tile * a.blocks, c = block * MX_BLOCK + (lane & 15) * 8;
    uint8_t* codes = a.codes + (long long)blockIdx.x * (MX_ROWS * MX_BLOCK / 2);
    uint8_t* scales = a.scales + (long long)blockIdx.x * (MX_ROWS * 4);
#pragma unroll
    for (int r0 = 0; r0 < MX_ROWS; r0 += 16 * TILE_AHEAD) {
        float v[TILE_AHEAD][8];
        uint4 raw[TILE_AHEAD];
#pragma unroll
        for (int i = 0; i < TILE_AHEAD; ++i) {
            const int src = mx_row_at(tile * MX_ROWS + r0 + i * 16 + warp * 2 + (lane >> 4), a.rows, a.half);
            const int width = src < 0 ? 0 : a.columns;      // padding: nothing of the row is there
            const long long base = (long long)src * a.columns;
            if (VEC == 2) {
                raw[i] = c < width ? *reinterpret_cast<const uint4*>((const __nv_bfloat16*)a.w + base + c) : make_uint4(0, 0, 0, 0);
            } else {
                load_columns<VEC != 0>(a.w, base, c, width, a.dtype, reinterpret_cast<float (&)[4]>(v[i][0]));
                load_columns<VEC != 0>(a.w, base, c + 4, width, a.dtype, reinterpret_cast<float (&)[4]>(v[i][4]));
            }
        }
#pragma unroll
        for (int i = 0; i < TILE_AHEAD; ++i) {
            const int r = r0 + i * 16 + warp * 2 + (lane >> 4);
            uint32_t top = 0;                               // magnitudes are in order as integers, NaN the largest
            if (VEC == 2) {
                const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    top = __vmaxu2(top, w[k] & 0x7fff7fffu);
                    v[i][2 * k] = __uint_as_float(w[k] << 16);
                    v[i][2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
                }
                top = max(top & 0xffff0000u, top << 16);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[i][k]) & 0x7fffffffu);
            }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const uint32_t code = mx4_scale_code(__uint_as_float(top));
            const float inv = mx_inverse_scale(code);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[i][k] *= inv;
            uint32_t word = code << ((lane & 12) * 2);      // lanes 4 q to 4 q + 3 of a row: byte q of the row's word
            word |= __shfl_xor_sync(0xffffffffu, word, 4);
            word |= __shfl_xor_sync(0xffffffffu, word, 8);
            *reinterpret_cast<uint32_t*>(codes + r * (MX_BLOCK / 2) + (lane & 15) * 4) = mx_to_e2m1(v[i]);
            if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(scales + r % 32 * 16 + r / 32 * 4) = word;
        }
    }
}

struct ExpandArgs {
    const uint8_t* codes; const uint8_t* scales;
    void* out; int dtype;
    int rows, columns, blocks, half;
};

template <bool VEC>
__global__ void __launch_bounds__(256) expand_mx4_kernel(const __grid_constant__ ExpandArgs a) {
    rdl_grid_wait();
    rdl_grid_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int tile = blockIdx.x / a.blocks, block = blockIdx.x - tile * a.blocks, c = block * MX_BLOCK + (lane & 15) * 8;
    const uint8_t* codes = a.codes + (long long)blockIdx.x * (MX_ROWS * MX_BLOCK / 2);
    const uint8_t* scales = a.scales + (long long)blockIdx.x * (MX_ROWS * 4);
    __shared__ float turned[VEC ? 1 : 8][2][VEC ? 4 : MX_BLOCK];
#pragma unroll
    for (int r0 = 0; r0 < MX_ROWS; r0 += 16 * TILE_AHEAD) {
        uint32_t w[TILE_AHEAD], sc[TILE_AHEAD];
#pragma unroll
        for (int i = 0; i < TILE_AHEAD; ++i) {
            const int r = r0 + i * 16 + warp * 2 + (lane >> 4);
            w[i] = *reinterpret_cast<const uint32_t*>(codes + r * (MX_BLOCK / 2) + (lane & 15) * 4);
            sc[i] = scales[r % 32 * 16 + r / 32 * 4 + (lane & 15) / 4];
        }
#pragma unroll
        for (int i = 0; i < TILE_AHEAD; ++i) {
            const int row = mx_row_at(tile * MX_ROWS + r0 + i * 16 + warp * 2 + (lane >> 4), a.rows, a.half);
            if (VEC && row < 0) continue;
            uint32_t h[4];
            mx_from_e2m1(w[i], h);
            const float s = mx_scale(sc[i]);
            const long long base = (long long)row * a.columns + c;
            float v[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[k]));
                v[2 * k] = f.x * s;
                v[2 * k + 1] = f.y * s;
            }
            if (VEC) {
                if (c >= a.columns) continue;
                if (a.dtype == RDL_BF16) {
                    uint4 raw;
                    __nv_bfloat162* o = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
                    for (int k = 0; k < 4; ++k) o[k] = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
                    *reinterpret_cast<uint4*>((__nv_bfloat16*)a.out + base) = raw;
                } else {
                    *reinterpret_cast<float4*>((float*)a.out + base) = make_float4(v[0], v[1], v[2], v[3]);
                    *reinterpret_cast<float4*>((float*)a.out + base + 4) = make_float4(v[4], v[5], v[6], v[7]);
                }
            } else {
                // rows that begin anywhere: through shared memory, so that neighbouring lanes store neighbouring columns (777 x 1,003: 6.6 us
                // and 10.1 with eight neighbouring columns a lane)
                float* mine = &turned[warp][lane >> 4][(lane & 15) * 8];
                *reinterpret_cast<float4*>(mine) = make_float4(v[0], v[1], v[2], v[3]);
                *reinterpret_cast<float4*>(mine + 4) = make_float4(v[4], v[5], v[6], v[7]);
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int to = __shfl_sync(0xffffffffu, row, (k >> 2) * 16), col = block * MX_BLOCK + (k & 3) * 32 + lane;
                    if (to >= 0 && col < a.columns) rdl_store(a.out, (long long)to * a.columns + col, a.dtype, turned[warp][k >> 2][(k & 3) * 32 + lane]);
                }
                __syncwarp();
            }
        }
    }
}

// Codes and scales that are there already, to the products' layout; blocks as above.  What lies beyond the last column is cleared.
struct LayArgs {
    const uint8_t* from; long long stride; const uint8_t* from_scales;       // bytes from a row's codes (4 bits) or values (8 bits) to the next one's
    uint8_t* to; uint8_t* to_scales;
    int rows, columns, blocks, half;                        // 8 bits: half is the rows' padded count
};

// four bytes of a row from byte b on; zeros from byte `end` on
template <bool VEC>
__device__ __forceinline__ uint32_t four_bytes(const uint8_t* row, int b, int end) {
    if (VEC && b + 4 <= end) return *reinterpret_cast<const uint32_t*>(row + b);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (b + i < end) w |= (uint32_t)row[b + i] << (8 * i);
    return w;
}

template <bool VEC>
__global__ void __launch_bounds__(256) lay_mx4_kernel(const __grid_constant__ LayArgs a) {
    rdl_grid_wait();
    rdl_grid_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int tile = blockIdx.x / a.blocks, block = blockIdx.x - tile * a.blocks, c = block * MX_BLOCK + (lane & 15) * 8;
    const int groups = (a.columns + MX_GROUP - 1) / MX_GROUP;
    uint8_t* to = a.to + (long long)blockIdx.x * (MX_ROWS * MX_BLOCK / 2);
    uint8_t* to_scales = a.to_scales + (long long)blockIdx.x * (MX_ROWS * 4);
    constexpr int EACH = MX_ROWS / 16;
    uint32_t w[EACH], sc[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {                         // all asked for before the first is stored
        const int src = mx_row_at(tile * MX_ROWS + i * 16 + warp * 2 + (lane >> 4), a.rows, a.half), group = block * 4 + (lane & 15);
        w[i] = src < 0 ? 0u : four_bytes<VEC>(a.from + src * a.stride, c / 2, (a.columns + 1) / 2);
        sc[i] = src < 0 || (lane & 15) >= 4 || group >= groups ? 0u : a.from_scales[(long long)src * groups + group];
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int r = i * 16 + warp * 2 + (lane >> 4);
        // of an odd row's last byte the upper half is padding, whatever it held
        if (c < a.columns && c + 8 > a.columns) w[i] &= 0xffffffffu >> (4 * (c + 8 - a.columns));
        *reinterpret_cast<uint32_t*>(to + r * (MX_BLOCK / 2) + (lane & 15) * 4) = w[i];
        if ((lane & 15) < 4) to_scales[r % 32 * 16 + r / 32 * 4 + (lane & 15)] = (uint8_t)sc[i];
    }
}

template <bool VEC>
__global__ void __launch_bounds__(256) lay_mx8_kernel(const __grid_constant__ LayArgs a) {
    rdl_grid_wait();
    rdl_grid_launch_dependents();
    const int m = blockIdx.x, groups = (a.columns + MX_GROUP - 1) / MX_GROUP;
    const uint8_t* from = a.from + m * a.stride;
    uint8_t* to = a.to + (long long)m * a.blocks * MX_BLOCK;
#pragma unroll 4
    for (int b = threadIdx.x * 4; b < a.blocks * MX_BLOCK; b += 1024) *reinterpret_cast<uint32_t*>(to + b) = four_bytes<VEC>(from, b, a.columns);
    for (int block = threadIdx.x; block < a.blocks; block += 256)
        *reinterpret_cast<uint32_t*>(a.to_scales + ((long long)block * a.half + m) * 4) = four_bytes<false>(a.from_scales + (long long)m * groups, block * 4, groups);
}

// tiles of 128 rows of a weight
int weight_tiles(int rows, int gated) {
    const int places = gated ? (rows / 2 + MX_UNIT - 1) / MX_UNIT * (2 * MX_UNIT) : rows;
    return (places + MX_ROWS - 1) / MX_ROWS;
}

}  // namespace

extern "C" int rdl_norm_mx8(const void* x, int x_dtype, const void* w1, int w1_dtype, float eps1, float off1,
                            const float* residual, float* residual_out, const void* w2, int w2_dtype, float eps2, float off2,
                            void* values, void* scales, int n_rows, int width, void* stream) {
    if (n_rows == 0) return 0;
    RDL_REQUIRE(x && values && scales, "norm_mx8: missing operand");
    RDL_REQUIRE(rdl_valid_dtype(x_dtype) && (!w1 || rdl_valid_dtype(w1_dtype)) && (!w2 || rdl_valid_dtype(w2_dtype)), "norm_mx8: bad dtype");
    RDL_REQUIRE(n_rows >= 0 && width > 0, "norm_mx8: bad sizes rows=%d width=%d", n_rows, width);
    RDL_REQUIRE((uintptr_t)values % 4 == 0 && (uintptr_t)scales % 4 == 0, "norm_mx8: the results must start on 4-byte boundaries");
    const NormMxArgs a{x, x_dtype, w1, w1_dtype, eps1, off1, residual, residual_out, w2, w2_dtype, eps2, off2,
                       (uint8_t*)values, (uint8_t*)scales, n_rows, width, mx_blocks(width), (n_rows + 3) / 4 * 4};
    const bool vec = width % 4 == 0 && aligned16(x) && aligned16(w1) && aligned16(w2) && aligned16(residual) && aligned16(residual_out);
    cudaStream_t st = (cudaStream_t)stream;
    const int quads = a.blocks * (MX_BLOCK / 4);            // groups of four columns
    // the threads, 128 to 256, and the groups of each that leave the fewest of them without one; on the width alone
    int threads = 32, iter = 1;
    if (quads > 32) {
        int best = 1 << 30;
        for (int t = quads < 256 ? (quads + 31) / 32 * 32 : 256; t >= (quads < 128 ? 32 : 128); t -= 32) {
            const int i = (quads + t - 1) / t;
            if (i <= RN_MAX_IT && i * t < best) { best = i * t; threads = t; iter = i; }
        }
    }
    cudaError_t e = cudaErrorInvalidValue;
    const bool half = vec && x_dtype == RDL_BF16;
#define RDL_NORM_MX8(I) case I: e = half ? rdl_launch(norm_mx8_kernel<I, true, true>, dim3(n_rows), dim3(threads), 0, st, a) \
                                    : vec ? rdl_launch(norm_mx8_kernel<I, true, false>, dim3(n_rows), dim3(threads), 0, st, a) \
                                          : rdl_launch(norm_mx8_kernel<I, false, false>, dim3(n_rows), dim3(threads), 0, st, a); break
    if (quads > 256 * RN_MAX_IT)
        e = vec ? rdl_launch(norm_mx8_wide_kernel<true>, dim3(n_rows), dim3(256), 0, st, a) : rdl_launch(norm_mx8_wide_kernel<false>, dim3(n_rows), dim3(256), 0, st, a);
    else
        switch (iter) { RDL_NORM_MX8(1); RDL_NORM_MX8(2); RDL_NORM_MX8(3); RDL_NORM_MX8(4); RDL_NORM_MX8(5); RDL_NORM_MX8(6); RDL_NORM_MX8(7); RDL_NORM_MX8(8); }
#undef RDL_NORM_MX8
    RDL_CHECK_EX(e, "norm_mx8");
    return 0;
}

extern "C" int rdl_pack_mx4(const void* w, int dtype, void* codes, void* scales, int rows, int columns, int gated, void* stream) {
    RDL_REQUIRE(w && codes && scales, "pack_mx4: missing operand");
    RDL_REQUIRE(rdl_valid_dtype(dtype), "pack_mx4: bad dtype %d", dtype);
    RDL_REQUIRE(rows > 0 && columns > 0 && (!gated || rows % 2 == 0), "pack_mx4: bad sizes rows=%d columns=%d", rows, columns);
    RDL_REQUIRE((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 16 == 0, "pack_mx4: the results must start on 16-byte boundaries");
    const PackArgs a{w, dtype, (uint8_t*)codes, (uint8_t*)scales, rows, columns, mx_blocks(columns), gated ? rows / 2 : 0};
    const long long grid = (long long)weight_tiles(rows, gated) * a.blocks;
    RDL_REQUIRE(grid <= 0x7fffffffLL, "pack_mx4: %d x %d is too large", rows, columns);
    cudaStream_t st = (cudaStream_t)stream;
    const int vec = columns % 4 == 0 && aligned16(w) ? (dtype == RDL_BF16 && columns % 8 == 0 ? 2 : 1) : 0;
    const cudaError_t e = vec == 2 ? rdl_launch(pack_mx4_kernel<2>, dim3((unsigned)grid), dim3(256), 0, st, a)
                          : vec == 1 ? rdl_launch(pack_mx4_kernel<1>, dim3((unsigned)grid), dim3(256), 0, st, a)
                                     : rdl_launch(pack_mx4_kernel<0>, dim3((unsigned)grid), dim3(256), 0, st, a);
    RDL_CHECK_EX(e, "pack_mx4");
    // The products read weights before the kernel ahead of them has ended (launch.cuh).  Something that is launched the ordinary way
    // comes in between, so that a product right behind this call finds the codes written.
    RDL_CUDA(cudaMemsetAsync((uint8_t*)scales + grid * (MX_ROWS * 4), 0, 16, st), "pack_mx4");
    return 0;
}

extern "C" int rdl_expand_mx4(const void* codes, const void* scales, void* out, int dtype, int rows, int columns, int gated, void* stream) {
    RDL_REQUIRE(codes && scales && out, "expand_mx4: missing operand");
    RDL_REQUIRE(rdl_valid_dtype(dtype), "expand_mx4: bad dtype %d", dtype);
    RDL_REQUIRE(rows > 0 && columns > 0 && (!gated || rows % 2 == 0), "expand_mx4: bad sizes rows=%d columns=%d", rows, columns);
    RDL_REQUIRE((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 16 == 0, "expand_mx4: the codes must start on 16-byte boundaries");
    const ExpandArgs a{(const uint8_t*)codes, (const uint8_t*)scales, out, dtype, rows, columns, mx_blocks(columns), gated ? rows / 2 : 0};
    const long long grid = (long long)weight_tiles(rows, gated) * a.blocks;
    RDL_REQUIRE(grid <= 0x7fffffffLL, "expand_mx4: %d x %d is too large", rows, columns);
    cudaStream_t st = (cudaStream_t)stream;
    const cudaError_t e = columns % 8 == 0 && aligned16(out) ? rdl_launch(expand_mx4_kernel<true>, dim3((unsigned)grid), dim3(256), 0, st, a)
                                                             : rdl_launch(expand_mx4_kernel<false>, dim3((unsigned)grid), dim3(256), 0, st, a);
    RDL_CHECK_EX(e, "expand_mx4");
    return 0;
}

extern "C" int rdl_lay_mx4(const void* from, long long stride, const void* from_scales, void* codes, void* scales, int rows, int columns, int gated, void* stream) {
    RDL_REQUIRE(from && from_scales && codes && scales, "lay_mx4: missing operand");
    RDL_REQUIRE(rows > 0 && columns > 0 && stride >= (columns + 1) / 2 && (!gated || rows % 2 == 0), "lay_mx4: bad sizes rows=%d columns=%d", rows, columns);
    RDL_REQUIRE((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 16 == 0, "lay_mx4: the results must start on 16-byte boundaries");
    const LayArgs a{(const uint8_t*)from, stride, (const uint8_t*)from_scales, (uint8_t*)codes, (uint8_t*)scales, rows, columns, mx_blocks(columns), gated ? rows / 2 : 0};
    const long long grid = (long long)weight_tiles(rows, gated) * a.blocks;
    RDL_REQUIRE(grid <= 0x7fffffffLL, "lay_mx4: %d x %d is too large", rows, columns);
    cudaStream_t st = (cudaStream_t)stream;
    const bool vec = stride % 4 == 0 && (uintptr_t)from % 4 == 0;
    RDL_CHECK_EX(vec ? rdl_launch(lay_mx4_kernel<true>, dim3((unsigned)grid), dim3(256), 0, st, a)
                     : rdl_launch(lay_mx4_kernel<false>, dim3((unsigned)grid), dim3(256), 0, st, a), "lay_mx4");
    RDL_CUDA(cudaMemsetAsync((uint8_t*)scales + grid * (MX_ROWS * 4), 0, 16, st), "lay_mx4");       // as after the packing
    return 0;
}

extern "C" int rdl_lay_mx8(const void* from, long long stride, const void* from_scales, void* values, void* scales, int rows, int columns, void* stream) {
    if (rows == 0) return 0;
    RDL_REQUIRE(from && from_scales && values && scales, "lay_mx8: missing operand");
    RDL_REQUIRE(rows > 0 && columns > 0 && stride >= 0, "lay_mx8: bad sizes rows=%d columns=%d", rows, columns);
    RDL_REQUIRE((uintptr_t)values % 4 == 0 && (uintptr_t)scales % 4 == 0, "lay_mx8: the results must start on 4-byte boundaries");
    const LayArgs a{(const uint8_t*)from, stride, (const uint8_t*)from_scales, (uint8_t*)values, (uint8_t*)scales, rows, columns, mx_blocks(columns), (rows + 3) / 4 * 4};
    const bool vec = stride % 4 == 0 && (uintptr_t)from % 4 == 0;
    RDL_CHECK_EX(vec ? rdl_launch(lay_mx8_kernel<true>, dim3((unsigned)rows), dim3(256), 0, (cudaStream_t)stream, a)
                     : rdl_launch(lay_mx8_kernel<false>, dim3((unsigned)rows), dim3(256), 0, (cudaStream_t)stream, a), "lay_mx8");
    return 0;
}

extern "C" int rdl_mx4_matrix_bytes(void) { return (int)sizeof(Mx4Matrix); }

extern "C" int rdl_mx4_describe(void* matrix, const void* codes, const void* scales, int rows, int columns, int gated) {
    RDL_REQUIRE(matrix && (uintptr_t)matrix % 64 == 0, "mx4_describe: the description must lie on a 64-byte boundary");
    RDL_REQUIRE(codes && scales && rows > 0 && columns > 0 && (!gated || rows % 2 == 0), "mx4_describe: bad sizes rows=%d columns=%d", rows, columns);
    RDL_REQUIRE((uintptr_t)codes % 32 == 0 && (uintptr_t)scales % 16 == 0, "mx4_describe: the codes must start on a 32-byte boundary, the scales on a 16-byte boundary");
    Mx4Matrix* w = (Mx4Matrix*)matrix;
    *w = Mx4Matrix{};
    w->codes = (const uint8_t*)codes; w->scales = (const uint8_t*)scales;
    w->rows = rows; w->columns = columns; w->gated = gated ? 1 : 0;
    w->blocks = mx_blocks(columns);
    w->tiles = weight_tiles(rows, gated);
    const cuuint64_t pieces = (cuuint64_t)w->tiles * w->blocks * MX_ROWS;
    RDL_REQUIRE(pieces <= 0x7fffffffULL, "mx4_describe: %d x %d is too large", rows, columns);      // a tile's coordinate is an int
    if (int e = mx_make_map(&w->codes_map, codes, {CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, 2, {MX_BLOCK, pieces}, {MX_BLOCK / 2}, {MX_BLOCK, MX_ROWS},
                                                   CU_TENSOR_MAP_SWIZZLE_128B}, "the codes of a 4-bit matrix")) return e;
    return mx_make_map(&w->scales_map, scales, {CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, {MX_ROWS, pieces / MX_ROWS}, {MX_SCALE_BYTES}, {MX_ROWS, 1},
                                                CU_TENSOR_MAP_SWIZZLE_NONE}, "the scales of a 4-bit matrix");
}
