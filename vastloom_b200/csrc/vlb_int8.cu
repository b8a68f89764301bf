// Products on 8-bit integers with a scale for each token and each output channel.
//
//   quantize   row r of x (plain, gathered, or SwiGLU of two operands):
//                a = max_c |x_rc|,  s_r = a / 127,  q_rc = rint(x_rc * (127 / a))
//   linear     y_rn = (sum_k q_rk w_nk) * s_r * t_n, the sum exact in 32-bit integers
//              (cols <= 131,071: 128 * 128 * cols < 2^31), for one matrix or grouped: row r uses
//              the matrix of the group whose range [offsets[g], offsets[g + 1]) holds it.
//
// The reference has no 8-bit integer path; the row scheme follows from the formulas above.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <mutex>
#include <utility>
#include <vector>

#include "vlb_launch.h"

namespace vlb {
namespace {

// ---- elements --------------------------------------------------------------------------------

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// silu(g) * u with the clamp of the layer's experts (gate from above, up on both sides). The
// comparisons keep a NaN, which fminf / fmaxf would drop.
__device__ __forceinline__ float swiglu(float g, float u, float limit) {
    if (limit > 0.f) {
        g = g > limit ? limit : g;
        u = u > limit ? limit : (u < -limit ? -limit : u);
    }
    return g / (1.f + expf(-g)) * u;
}

// ---- row quantizer ---------------------------------------------------------------------------

// What a row's largest |x| (as float bits, so that a NaN is the largest of all) makes of the row:
// its scale, and the factor that brings it to [-127, 127]. Rows below 2^-100 are first lifted by
// 2^100 (exact), or 127 / a would overflow. A row that is not finite keeps q = 0 and the scale
// NaN, so the products' rows that come from it are NaN and no others.
struct RowStep {
    float lift, inv, scale;
};
__device__ __forceinline__ RowStep row_step(uint32_t amax_bits) {
    const float a = __uint_as_float(amax_bits);
    if (amax_bits == 0u) return RowStep{0.f, 0.f, 0.f};
    if (amax_bits >= 0x7f800000u) return RowStep{0.f, 0.f, __uint_as_float(0x7fc00000u)};
    const float lift = a < 0x1p-100f ? 0x1p100f : 1.f;
    return RowStep{lift, __fdiv_rn(127.f, a * lift), __fdiv_rn(a, 127.f)};
}

// rint(x * inv) as the low byte of an integer: adding 1.5 * 2^23 leaves the rounded integer in
// the mantissa's low bits. The product rounds to 32 bits first (the operator's definition), so it
// must not be contracted into the addition.
__device__ __forceinline__ uint32_t quant_byte(float x, const RowStep& st) {
    if (st.inv == 0.f) return 0u;
    return __float_as_uint(__fadd_rn(__fmul_rn(x * st.lift, st.inv), 12582912.f)) & 0xffu;
}

template <typename T, bool SWIGLU>
__device__ __forceinline__ float row_value(const Int8QuantParams& p, size_t at) {
    const float x = to_float(static_cast<const T*>(p.x)[at]);
    if (!SWIGLU) return x;
    return swiglu(x, to_float(static_cast<const T*>(p.up)[at]), p.limit);
}

// One CTA a row: the row's largest |x|, then its bytes (zeros up to the row's pitch).
template <typename T, bool SWIGLU>
__global__ void __launch_bounds__(256) int8_quantize_kernel(const Int8QuantParams p) {
    __shared__ uint32_t top[8];
    const uint32_t tid = threadIdx.x;
    for (size_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const uint64_t src = p.row_index ? p.row_index[r] : r;
        const bool have = src < p.x_rows;
        const size_t base = src * p.x_stride;
        uint32_t m = 0;
        if (have)
            for (uint32_t c = tid; c < p.cols; c += blockDim.x)
                m = max(m, __float_as_uint(row_value<T, SWIGLU>(p, base + c)) & 0x7fffffffu);
        m = __reduce_max_sync(0xffffffffu, m);
        __syncthreads();
        if ((tid & 31u) == 0) top[tid >> 5] = m;
        __syncthreads();
        m = 0;
        for (uint32_t i = 0; i < blockDim.x / 32u; ++i) m = max(m, top[i]);
        const RowStep st = row_step(m);
        if (tid == 0) p.scale[r] = st.scale;
        for (uint32_t c = tid; c < p.fill_cols; c += blockDim.x) {
            const bool in = have && c < p.cols;
            p.q[r * p.q_stride + c] = (int8_t)(in ? quant_byte(row_value<T, SWIGLU>(p, base + c), st) : 0u);
        }
    }
}

// ---- groups ----------------------------------------------------------------------------------

// Rows of group g, kept inside [0, rows] whatever the offsets hold.
__device__ __forceinline__ void group_range(const Int8LinearParams& p, uint32_t g, uint32_t& lo, uint32_t& hi) {
    if (!p.offsets) {
        lo = 0;
        hi = p.rows;
        return;
    }
    lo = min(p.offsets[g], p.rows);
    hi = max(lo, min(p.offsets[g + 1], p.rows));
}

// ---- product, any alignment ------------------------------------------------------------------

constexpr uint32_t kGenTile = 64, kGenK = 64;

// 4 bytes of a row from column c on, zeros past the row's end.
__device__ __forceinline__ uint32_t load_word(const int8_t* row, uint32_t c, uint32_t cols) {
    if (c + 4u <= cols && ((uintptr_t)(row + c) & 3u) == 0) return *reinterpret_cast<const uint32_t*>(row + c);
    uint32_t v = 0;
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i)
        if (c + i < cols) v |= (uint32_t)(uint8_t)row[c + i] << (8u * i);
    return v;
}

template <typename TY>
__global__ void __launch_bounds__(256) int8_linear_kernel(const Int8LinearParams p) {
    __shared__ uint32_t xs[kGenTile][kGenK / 4 + 1], ws[kGenTile][kGenK / 4 + 1];
    const uint32_t tid = threadIdx.x, tr = tid / 16u, tc = tid % 16u;
    const uint32_t n0 = blockIdx.x * kGenTile;
    for (uint32_t g = blockIdx.z; g < p.groups; g += gridDim.z) {
        uint32_t lo, hi;
        group_range(p, g, lo, hi);
        const int8_t* w = p.w + (size_t)g * p.out_cols * p.w_stride;
        for (uint32_t r0 = lo + blockIdx.y * kGenTile; r0 < hi; r0 += gridDim.y * kGenTile) {
            int32_t acc[4][4] = {};
            for (uint32_t k0 = 0; k0 < p.cols; k0 += kGenK) {
                for (uint32_t i = tid; i < kGenTile * kGenK / 4u; i += 256u) {
                    const uint32_t row = i / (kGenK / 4u), c = i % (kGenK / 4u);
                    xs[row][c] = r0 + row < hi ? load_word(p.x + (size_t)(r0 + row) * p.x_stride, k0 + 4u * c, p.cols) : 0u;
                    ws[row][c] = n0 + row < p.out_cols ? load_word(w + (size_t)(n0 + row) * p.w_stride, k0 + 4u * c, p.cols)
                                                       : 0u;
                }
                __syncthreads();
#pragma unroll 4
                for (uint32_t c = 0; c < kGenK / 4u; ++c)
#pragma unroll
                    for (uint32_t i = 0; i < 4u; ++i)
#pragma unroll
                        for (uint32_t j = 0; j < 4u; ++j)
                            acc[i][j] = __dp4a((int)xs[tr + 16u * i][c], (int)ws[tc + 16u * j][c], acc[i][j]);
                __syncthreads();
            }
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) {
                const uint32_t r = r0 + tr + 16u * i;
                if (r >= hi) continue;
                const float s = p.row_weight ? p.x_scale[r] * p.row_weight[r] : p.x_scale[r];
#pragma unroll
                for (uint32_t j = 0; j < 4u; ++j) {
                    const uint32_t n = n0 + tc + 16u * j;
                    if (n < p.out_cols)
                        static_cast<TY*>(p.y)[(size_t)r * p.y_stride + n] =
                            from_float<TY>((float)acc[i][j] * s * p.w_scale[(size_t)g * p.out_cols + n]);
                }
            }
        }
    }
}

template <typename T>
cudaError_t quantize_type(const Int8QuantParams& p, cudaStream_t s) {
    const unsigned grid = p.rows < 65535u ? p.rows : 65535u;
    if (p.up)
        int8_quantize_kernel<T, true><<<grid, 256, 0, s>>>(p);
    else
        int8_quantize_kernel<T, false><<<grid, 256, 0, s>>>(p);
    return cudaGetLastError();
}

template <typename TY>
cudaError_t linear_type(const Int8LinearParams& p, cudaStream_t s) {
    const uint32_t tiles_n = (p.out_cols + kGenTile - 1u) / kGenTile, tiles_r = (p.rows + kGenTile - 1u) / kGenTile;
    const dim3 grid(tiles_n, tiles_r < 1024u ? tiles_r : 1024u, p.groups < 1024u ? p.groups : 1024u);
    int8_linear_kernel<TY><<<grid, 256, 0, s>>>(p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_int8_quantize(const Int8QuantParams& p, int x_type, cudaStream_t s) {
    switch (x_type) {
        case VLB_DTYPE_F32: return quantize_type<float>(p, s);
        case VLB_DTYPE_F16: return quantize_type<__half>(p, s);
        case VLB_DTYPE_BF16: return quantize_type<__nv_bfloat16>(p, s);
        default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_int8_linear(const Int8LinearParams& p, int y_type, cudaStream_t s) {
    switch (y_type) {
        case VLB_DTYPE_F32: return linear_type<float>(p, s);
        case VLB_DTYPE_F16: return linear_type<__half>(p, s);
        case VLB_DTYPE_BF16: return linear_type<__nv_bfloat16>(p, s);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace vlb
