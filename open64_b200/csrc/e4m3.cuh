// e4m3 results with a scale for each block: scale = (largest magnitude of the block) / 448, q = e4m3(h / scale).
// One definition for the norm and for the SwiGLU tails, so that the same h becomes the same q wherever it is made.
#pragma once
#include <cfloat>
#include <cstdint>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

namespace o64 {

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN wins, as in a maximum of the definition
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// amax / 448, or 1 where that is no normal number (NaN stays NaN).
__device__ __forceinline__ float block_scale_of(float amax) {
    const float s = amax / 448.0f;
    return s < FLT_MIN ? 1.0f : s;
}

// h / scale with inv = 1 / scale. One division per block (one per value took RMS norm of 16384 x 8192 from 157 to 194 us): the
// product with inv is off by up to 1.5 ulp, which puts some values on the other side of a rounding to four bits, so a
// step with the product's own remainder follows, q - (q scale - h) inv, in two multiply-adds; q is then the quotient rounded
// once. (With q scale - h and not h - q scale a zero keeps its sign.) `back` is remainder_scale(scale): under an infinite
// scale inv is 0 and nothing is to be put right, the remainder would be 0 * inf.
__device__ __forceinline__ float remainder_scale(float scale) { return scale <= FLT_MAX ? scale : 0.0f; }
__device__ __forceinline__ float quotient(float h, float back, float inv) {
    const float q = h * inv;
    return fmaf(fmaf(q, back, -h), -inv, q);
}
__device__ __forceinline__ float2 quotient2(float2 h, float back, float inv) {
    const float2 q = make_float2(h.x * inv, h.y * inv);
    return __ffma2_rn(__ffma2_rn(q, make_float2(back, back), make_float2(-h.x, -h.y)), make_float2(-inv, -inv), q);
}
__device__ __forceinline__ uint32_t quant2(float2 h, float back, float inv) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(quotient2(h, back, inv), __NV_SATFINITE, __NV_E4M3);
}

}  // namespace o64
