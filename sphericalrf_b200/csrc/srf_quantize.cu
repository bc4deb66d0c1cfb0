// srf_quantize.cu -- 16-bit values to e4m3 values and fp32 scales, for srf_grouped_fp8.cu.
//
// A block shares one scale s = amax / 448, amax over the block's finite values (1 where that is 0, and at least 2^-126,
// below which a quotient could leave the range); q = the e4m3 value nearest to v / s, ties to even.  Infinities and
// NaNs become e4m3's NaN and do not touch the block's other values.  v / s is the fp32 quotient.
//
// v / s must be the correctly rounded quotient: one step off moves values that lie next to a tie.  With r the correctly
// rounded 1 / s and q0 = v r, q0 + r (v - q0 s) -- two fused operations -- is that quotient (Markstein, IBM J. Res. Dev. 34,
// 1990), as long as the remainder does not underflow: it is a multiple of 2^-48 |v| at the least, and a value that is not
// rounded to zero has |v| > 2^-11 s, so s >= 2^-80 is enough.  Blocks with a smaller scale divide.
//
// The maximum is taken on the 16-bit patterns, two at a time: without their sign, floats order as integers.  A block whose
// maximum is not finite is gone through again, value by value.
//
// Bound by memory: two bytes read, one written per value, one pass (the block stays in registers between the maximum
// and the quotients).  65539 x 2048: 71 us alone, 75-78 a call, 5.2-5.4 TB/s; 66 % of the issue slots are taken.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "srf_layers.cuh"
#include "srf_tile.cuh"

namespace srf {

namespace {

constexpr float kE4m3Max = 448.f;
constexpr float kScaleMin = 1.17549435e-38f;      // 2^-126

__device__ __forceinline__ void unpack8(uint4 v, bool bf16, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (bf16) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = t.x;
            f[2 * i + 1] = t.y;
        }
    }
}

// Eight values from `p`, of which `have` (0..8) exist; zeros behind them.
__device__ __forceinline__ uint4 load8(const uint16_t* p, int have) {
    if (have >= 8) return __ldcg(reinterpret_cast<const uint4*>(p));
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < have) w[i >> 1] |= (uint32_t)__ldcg(p + i) << ((i & 1) * 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __int_as_float(0x7f800000); }

// Largest magnitude of each half, as 16-bit patterns.
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t amax_pattern(uint4 v, uint32_t top) {
    constexpr uint32_t kAbs = 0x7fff7fffu;
    top = max_u16x2(top, max_u16x2(v.x & kAbs, v.y & kAbs));
    return max_u16x2(top, max_u16x2(v.z & kAbs, v.w & kAbs));
}

__device__ __forceinline__ float amax_finite(const float (&f)[8], float top) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = finite(f[i]) ? fmaxf(top, fabsf(f[i])) : top;
    return top;
}

__device__ __forceinline__ float scale_of(float amax) { return amax > 0.f ? fmaxf(amax / kE4m3Max, kScaleMin) : 1.f; }

// What a block's values need to become e4m3: plain (all values finite, scale not tiny) takes the short way.
struct BlockScale {
    float scale, inverse;
    bool plain;
};
__device__ __forceinline__ BlockScale block_scale(float amax, bool all_finite) {
    BlockScale b;
    b.scale = scale_of(amax);
    b.inverse = 1.f / b.scale;
    b.plain = all_finite && b.scale >= 8.2718061e-25f;      // 2^-80
    return b;
}

__device__ __forceinline__ uint2 to_e4m3(const float (&q)[8]) {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint16_t t;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(t) : "f"(q[2 * i + 1]), "f"(q[2 * i]));
        h[i] = t;
    }
    return make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
}

// The short way, two values to an instruction.  It makes the negative of the quotient, -q0 - r (v - q0 s), and turns the sign of
// the result: where q0 is exact the remainder is +0, which leaves the sign of -q0 = -0 or +0 alone (added to q0 = -0, it would
// make it +0).
__device__ __forceinline__ uint2 quantize8_plain(const float (&f)[8], float scale, float inverse) {
    uint64_t up, inv;
    asm("mov.b64 %0, {%1, %1};" : "=l"(up) : "f"(scale));
    asm("mov.b64 %0, {%1, %1};" : "=l"(inv) : "f"(-inverse));
    float q[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint64_t v, q0, rest;
        asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(f[2 * i]), "f"(f[2 * i + 1]));
        asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(q0) : "l"(v), "l"(inv));
        asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(rest) : "l"(q0), "l"(up), "l"(v));
        asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(q0) : "l"(rest), "l"(inv));
        asm("mov.b64 {%0, %1}, %2;" : "=f"(q[2 * i]), "=f"(q[2 * i + 1]) : "l"(q0));
    }
    const uint2 n = to_e4m3(q);
    return make_uint2(n.x ^ 0x80808080u, n.y ^ 0x80808080u);
}

__device__ __forceinline__ uint2 quantize8(const float (&f)[8], const BlockScale& b) {
    if (b.plain) return quantize8_plain(f, b.scale, b.inverse);
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = finite(f[i]) ? f[i] / b.scale : __int_as_float(0x7fffffff);
    return to_e4m3(q);
}

__device__ __forceinline__ float pattern_value(uint32_t h, bool bf16) {
    return bf16 ? __uint_as_float(h << 16) : __half2float(__ushort_as_half((unsigned short)h));
}
__device__ __forceinline__ bool pattern_finite(uint32_t h, bool bf16) { return h < (bf16 ? 0x7f80u : 0x7c00u); }

__device__ __forceinline__ void store8(unsigned char* p, int have, uint2 v) {
    if (have >= 8) { *reinterpret_cast<uint2*>(p) = v; return; }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < have) p[i] = (unsigned char)((i < 4 ? v.x >> (8 * i) : v.y >> (8 * (i - 4))) & 255u);
}

// Rows x 128: half a warp holds one block of one row (eight values a lane); a warp takes two neighbouring blocks of
// four rows, so that four loads of 16 bytes per lane are in flight.
constexpr int kRowsPerWarp = 4;

__global__ void __launch_bounds__(256)
k_quantize_rows(int bf16, uint64_t n_rows, const uint64_t* __restrict__ n_used, uint32_t n_cols, const uint16_t* __restrict__ in,
                uint64_t ld_in, unsigned char* __restrict__ out, uint64_t ld_out, float* __restrict__ scales) {
    uint64_t rows = n_rows;
    tile::wait_for_inputs();
    tile::let_next_start();
    if (n_used) { const uint64_t u = __ldcg((const unsigned long long*)n_used); rows = u < rows ? u : rows; }
    const int lane = threadIdx.x & 31;
    const uint32_t block = blockIdx.y * 2 + (lane >> 4);
    const uint64_t row0 = ((uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * kRowsPerWarp;
    if (row0 >= rows) return;
    const uint32_t col = block * 128 + (lane & 15) * 8;
    const int have = col >= n_cols ? 0 : n_cols - col < 8 ? (int)(n_cols - col) : 8;
    uint4 v[kRowsPerWarp];
    const bool full = (blockIdx.y + 1) * 256 <= n_cols && row0 + kRowsPerWarp <= rows;       // no edge: the same for the warp
    in += row0 * ld_in;
    out += row0 * ld_out;
    if (full) {
#pragma unroll
        for (int i = 0; i < kRowsPerWarp; ++i) v[i] = __ldcg(reinterpret_cast<const uint4*>(in + i * ld_in + col));
    } else {
#pragma unroll
        for (int i = 0; i < kRowsPerWarp; ++i) v[i] = row0 + i < rows ? load8(in + i * ld_in + col, have) : make_uint4(0u, 0u, 0u, 0u);
    }
    // Every lane makes the scale of one of its half's four blocks -- the two divisions of a scale cost as much as all the rest
    // of a block, and 16 lanes repeating them for every row made the kernel issue-bound (7 % of 65539 x 2048's time).
    uint32_t mine = 0;
    bool finite_all = true;
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i) {
        uint32_t top = amax_pattern(v[i], 0u);
#pragma unroll
        for (int d = 8; d; d >>= 1) top = max_u16x2(top, __shfl_xor_sync(0xffffffffu, top, d));
        top = max(top & 0xffffu, top >> 16);
        mine = (lane & (kRowsPerWarp - 1)) == i ? top : mine;
        finite_all = finite_all && pattern_finite(top, bf16 != 0);
    }
    const bool mine_finite = pattern_finite(mine, bf16 != 0);
    float amax = pattern_value(mine, bf16 != 0);
    if (!__all_sync(0xffffffffu, finite_all)) {
#pragma unroll
        for (int i = 0; i < kRowsPerWarp; ++i) {
            float f[8];
            unpack8(v[i], bf16 != 0, f);
            float a = amax_finite(f, 0.f);
#pragma unroll
            for (int d = 8; d; d >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, d));
            amax = (lane & (kRowsPerWarp - 1)) == i ? a : amax;
        }
    }
    const BlockScale own = block_scale(amax, mine_finite);
    if ((lane & 15) < kRowsPerWarp && row0 + (lane & 15) < rows && block * 128 < n_cols) scales[(uint64_t)block * n_rows + row0 + (lane & 15)] = own.scale;
    const bool plain_all = __all_sync(0xffffffffu, own.plain);
    if (full && plain_all) {
#pragma unroll
        for (int i = 0; i < kRowsPerWarp; ++i) {
            float f[8];
            unpack8(v[i], bf16 != 0, f);
            *reinterpret_cast<uint2*>(out + i * ld_out + col) = quantize8_plain(f, __shfl_sync(0xffffffffu, own.scale, (lane & 16) | i),
                                                                                __shfl_sync(0xffffffffu, own.inverse, (lane & 16) | i));
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i) {
        BlockScale b;
        b.scale = __shfl_sync(0xffffffffu, own.scale, (lane & 16) | i);
        b.inverse = __shfl_sync(0xffffffffu, own.inverse, (lane & 16) | i);
        b.plain = true;
        if (!plain_all) b.plain = __shfl_sync(0xffffffffu, (int)own.plain, (lane & 16) | i);
        float f[8];
        unpack8(v[i], bf16 != 0, f);
        if (row0 + i < rows && have > 0) store8(out + i * ld_out + col, have, quantize8(f, b));
    }
}

// 128 x 128: a CTA holds one block, 64 values a thread.
__global__ void __launch_bounds__(256)
k_quantize_weights(int bf16, uint32_t n_rows, uint32_t n_cols, const uint16_t* __restrict__ in, uint64_t ld_in, uint64_t stride_in,
                   unsigned char* __restrict__ out, uint64_t ld_out, uint64_t stride_out, float* __restrict__ scales) {
    const uint32_t bx = blockIdx.x, by = blockIdx.y, mat = blockIdx.z;
    const uint32_t col = bx * 128 + (threadIdx.x & 15) * 8, row0 = by * 128 + (threadIdx.x >> 4);
    const int have = col >= n_cols ? 0 : n_cols - col < 8 ? (int)(n_cols - col) : 8;
    tile::wait_for_inputs();
    tile::let_next_start();
    in += mat * stride_in;
    out += mat * stride_out;
    uint4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = row0 + 16 * i < n_rows ? load8(in + (uint64_t)(row0 + 16 * i) * ld_in + col, have) : make_uint4(0u, 0u, 0u, 0u);
    __shared__ uint32_t sh[8];
    __shared__ float sh_finite[8];
    const int warp = threadIdx.x >> 5;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = amax_pattern(v[i], top);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = max_u16x2(top, __shfl_xor_sync(0xffffffffu, top, d));
    if ((threadIdx.x & 31) == 0) sh[warp] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max_u16x2(top, sh[i]);
    top = max(top & 0xffffu, top >> 16);
    const bool all_finite = pattern_finite(top, bf16 != 0);
    float amax = pattern_value(top, bf16 != 0);
    if (!all_finite) {                                  // the same for the whole CTA
        amax = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float f[8];
            unpack8(v[i], bf16 != 0, f);
            amax = amax_finite(f, amax);
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
        if ((threadIdx.x & 31) == 0) sh_finite[warp] = amax;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf(amax, sh_finite[i]);
    }
    const BlockScale b = block_scale(amax, all_finite);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (row0 + 16 * i < n_rows && have > 0) {
            float f[8];
            unpack8(v[i], bf16 != 0, f);
            store8(out + (uint64_t)(row0 + 16 * i) * ld_out + col, have, quantize8(f, b));
        }
    }
    if (threadIdx.x == 0) scales[((uint64_t)mat * gridDim.y + by) * gridDim.x + bx] = b.scale;
}

}  // namespace

const char* launch_quantize_rows(int type, uint64_t n_rows, const uint64_t* n_rows_used, uint32_t n_cols, const void* in, uint64_t ld_in,
                                 void* out, uint64_t ld_out, float* scales, cudaStream_t stream) {
    if (!n_rows) return nullptr;
    const dim3 grid((uint32_t)((n_rows + 8 * kRowsPerWarp - 1) / (8 * kRowsPerWarp)), (n_cols + 255) / 256);
    return launch_layer(k_quantize_rows, 0, 256, 1, grid, stream, (int)(type == SRF_TYPE_BF16), n_rows, n_rows_used, n_cols, (const uint16_t*)in,
                        ld_in, (unsigned char*)out, ld_out, scales);
}

const char* launch_quantize_weights(int type, uint32_t n_matrices, uint32_t n_rows, uint32_t n_cols, const void* in, uint64_t ld_in,
                                    uint64_t stride_in, void* out, uint64_t ld_out, uint64_t stride_out, float* scales, cudaStream_t stream) {
    const dim3 grid((n_cols + 127) / 128, (n_rows + 127) / 128, n_matrices);
    return launch_layer(k_quantize_weights, 0, 256, 1, grid, stream, (int)(type == SRF_TYPE_BF16), n_rows, n_cols, (const uint16_t*)in, ld_in,
                        stride_in, (unsigned char*)out, ld_out, stride_out, scales);
}

}  // namespace srf
