// Fast single-precision functions of the row operators, which are bound by instruction issue next to
// HBM: approximate reciprocal, root and power of two (2 units of 2^-23 each; subnormals are 0).
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
// e^x for x in [-1000, 88], as 2^(x log2 e). The rounding of the exponent's product, which grows
// with |x|, is put back: 2^(t + c) = 2^t (1 + c ln 2), c the product's rest.
__device__ __forceinline__ float fast_exp(float x) {
    const float t = x * 1.44269504f;
    const float c = fmaf(x, 1.44269504f, -t);
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    return fmaf(e, c * 0.693147181f, e);
}

}  // namespace vlb
