// maya_mmq_image.cuh - the prompt path's activation image (maya_mmq_quantize's rows): its geometry and its rounding, shared by the quantizer, the
// grouped GEMM's write-back and the norm that leaves it (rms_q8.cu).
#pragma once

#include "maya_common.cuh"

namespace maya {

// The activation image: a row is its w_cols f16 values d * q, then one f16 per 32 values - the group's SUM CORRECTION
// xa = f16(sum of the unquantized values) - sum of the row's stored d * q values - padded with zeros to a multiple of 64.  llama.cpp's
// MMQ keeps that unquantized sum beside the block (the "ds4" q8_1 layout) and a type with a constant term per group
// (Q4_K: -dmin * m) multiplies the term by it, not by the sum of the rounded values; here the same result comes from
// extra K steps inside a Q4_K product: A = -dmin * m of a row's groups, B = xa.  Other types do not read the tail.
__host__ __device__ constexpr int64_t xq_tail(int64_t cols) { return ((cols / 32) + 63) & ~(int64_t) 63; }
__host__ __device__ constexpr int64_t xq_ld(int64_t cols) { return cols + xq_tail(cols); }

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *(uint32_t*) &h; }

// The q8_1 rounding of maya_mmq_quantize for a thread that holds 8 consecutive values of a 32-value group (the group's
// four threads are four consecutive lanes; every lane of the warp must call): llama.cpp's quantize_mmq_q8_1 as the
// reference's host model states it - d_inv = 127 / amax, q = round(v * d_inv) clamped to +-127, d = min(1 / d_inv, 65504)
// kept as f16, stored f16(d) * q.  o = the 8 stored values; the return value is the group's sum correction
// f16(S) - sum of the stored values, with S added in quantize_mmq_q8_1's order: four consecutive values left to right
// (this thread holds partial sums 2j and 2j + 1 of the group's eight), then the tree at distances 4, 2, 1.
__device__ __forceinline__ __half q8_1_round8(const float (&v)[8], uint32_t (&o)[4]) {
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[i]));
    amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
    const float d_inv = __fdiv_rn(127.0f, amax);
    const float dh = amax == 0.0f ? 0.0f : __half2float(__float2half_rn(fminf(__fdiv_rn(1.0f, d_inv), 65504.0f)));
    float bsum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float q0 = 0.0f, q1 = 0.0f;
        if (amax != 0.0f) {
            q0 = fmaxf(-127.0f, fminf(127.0f, roundf(__fmul_rn(v[2 * i], d_inv))));
            q1 = fmaxf(-127.0f, fminf(127.0f, roundf(__fmul_rn(v[2 * i + 1], d_inv))));
        }
        const __half2 r = __floats2half2_rn(dh * q0, dh * q1);
        o[i] = h2_bits(r);
        bsum += __low2float(r) + __high2float(r);     // the stored values: multiples of one power of two, 24 bits in all - exact
    }
    float s0 = __fadd_rn(__fadd_rn(__fadd_rn(v[0], v[1]), v[2]), v[3]), s1 = __fadd_rn(__fadd_rn(__fadd_rn(v[4], v[5]), v[6]), v[7]);
    s0 = __fadd_rn(s0, __shfl_xor_sync(0xFFFFFFFFu, s0, 2));
    s1 = __fadd_rn(s1, __shfl_xor_sync(0xFFFFFFFFu, s1, 2));
    s0 = __fadd_rn(s0, __shfl_xor_sync(0xFFFFFFFFu, s0, 1));
    s1 = __fadd_rn(s1, __shfl_xor_sync(0xFFFFFFFFu, s1, 1));
    bsum += __shfl_xor_sync(0xFFFFFFFFu, bsum, 1);
    bsum += __shfl_xor_sync(0xFFFFFFFFu, bsum, 2);
    return __float2half_rn(__half2float(__float2half_rn(__fadd_rn(s0, s1))) - bsum);
}

}  // namespace maya
