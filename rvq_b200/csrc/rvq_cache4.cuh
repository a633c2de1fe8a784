// The 4-bit cache record (layout in include/rvq_b200.h) and its arithmetic.
#pragma once

#include "rvq_common.cuh"

namespace rvq {
namespace cache4 {

constexpr int kGroup = 32;                   // values that share a zero and a step

__host__ __device__ constexpr int record_bytes(int hd) { return hd * 5 / 4; }

// (zero, step) of a group as one word: bf16 zero in the low half, bf16 step in the high half.
__device__ __forceinline__ float zero_of(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float step_of(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// The parameters of a group with the given extremes.  fminf and fmaxf drop a
// NaN, so the caller passes NaN extremes for a group that holds one.
__device__ __forceinline__ uint32_t params_of(float lo, float hi) {
    const float step = __fdiv_rn(__fsub_rn(hi, lo), 15.0f);
    return (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(lo)) |
           (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(step)) << 16;
}

// clamp(rint((x - z) / s), 0, 15) with an IEEE quotient; 0 for s = 0 and for a quotient that is NaN.
__device__ __forceinline__ uint32_t code_of(float x, float zero, float step) {
    const float q = rintf(__fdiv_rn(__fsub_rn(x, zero), step));
    return step > 0.f && q > 0.f ? (uint32_t)fminf(q, 15.0f) : 0u;
}

// The same with inv = 1 / step (approximate), unless *near is set: where d inv is clearly nearer to one integer than to the
// next, that integer is the quotient's too (|d - k s| < 0.4999 s leaves 2^-13 s for the roundings of inv, of d inv, of
// d - k s and of the quotient, about 2^-22 s each).  Near the middle between two, and for a step that is 0, subnormal (inv is
// infinite then) or not finite, *near is set and the caller divides.  kClamp false: zero is the group's minimum itself
// (bf16 values), so that 0 <= d <= 15 s (1 + 2^-8) and the integer is in range.
template <bool kClamp>
__device__ __forceinline__ uint32_t code_near(float x, float zero, float step, float inv, bool* near) {
    constexpr float kInt = 12582912.f;                       // 1.5 2^23: a sum with it ends at an integer
    const float d = __fsub_rn(x, zero), t = fmaf(d, inv, kInt), k = __fsub_rn(t, kInt);
    *near = !(fabsf(fmaf(-k, step, d)) < 0.4999f * step);
    return __float_as_uint(kClamp ? __fadd_rn(fminf(fmaxf(k, 0.f), 15.f), kInt) : t) & 15u;
}

// z + s c (s c is exact: 8 by 4 bits)
__device__ __forceinline__ float value_of(uint32_t c, float zero, float step) {
    const float f = __fsub_rn(__uint_as_float(0x4b000000u | c), 8388608.f);      // 2^23 + c less 2^23
    return __fadd_rn(zero, __fmul_rn(step, f));
}

inline int status(cudaError_t e) {
    if (e != cudaSuccess) last_cuda_error_slot() = (int)e;
    return e == cudaSuccess ? RVQ_OK : RVQ_ERR_CUDA;
}

}  // namespace cache4
}  // namespace rvq
