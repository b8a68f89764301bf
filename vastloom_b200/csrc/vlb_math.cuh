// Fast single-precision functions of the row operators, which are bound by instruction issue next to
// HBM: approximate reciprocal, root (1 ulp each) and power of two (2 ulp); subnormals are 0.
#pragma once

namespace vlb {

__device__ __forceinline__ float fast_rcp(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float fast_rsqrt(float x) {
    float r;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// e^x for x in [-1000, 88], as 2^t with t = x log2 e rounded, times e^d, d = x - t ln 2 being what the
// rounding left out (with the constant's own error up to 60 units of 2^-24 at x = 88). ln 2 in two
// parts, 24 bits and the rest: the first alone would leave 0.05 |x| units. In all within 5 units of
// 2^-24: 4 of the power of two, one of the last rounding, d and d^2 / 2 a few hundredths.
__device__ __forceinline__ float fast_exp(float x) {
    const float t = x * 1.44269504f;
    const float d = fmaf(-t, -1.90465421e-9f, fmaf(-t, 0.693147182f, x));
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    return fmaf(e, d, e);
}

}  // namespace vlb
