// The residual's addition and RMS norm, with rows in the activations' type and in 8 bits, and its gradient.
//
//   forward    h = x + residual,  s = 1 / sqrt(mean h^2 + eps),  y = h s w;  a = max |y|,
//              q = rint(y * (127 / a)), scale = a / 127
//   gradient   n = h s,  g = dy w,  d = s (g - n mean(g n)) + dh,  dw = sum over rows of dy n
//
// Both move every element once and do a handful of operations on it: HBM bounds them. The sums are in
// 32 bits. Where the squares pass them (h above 1.8e19) the row is taken again with h lifted by 2^-70.
//
// The reference's norm is deepseek_v4_rms_norm (deepseek_v4_reference.cpp:170-206), without residual,
// other types or gradient; the formulas above are this file's own.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "vlb_launch.h"
#include "vlb_rows.cuh"
#include "vlb_tcgen05.cuh"

namespace vlb {
namespace {

constexpr float kNormLift = 0x1p-70f;

// 1 / sqrt(mean + eps) of a row's sum of lifted squares.
__device__ __forceinline__ float norm_step(float sum, uint32_t cols, float eps, float lift) {
    return __frsqrt_rn(__fdiv_rn(sum, (float)cols) + eps * lift * lift);
}

// ROW threads a row.
template <typename T, typename R, uint32_t ROW>
__global__ void __launch_bounds__(256) add_norm_kernel(const NormParams p) {
    __shared__ float scratch[2][ROW / 32u];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    RowReduce<ROW> reduce{scratch};
    const uint32_t tid = threadIdx.x % ROW;
    for (size_t r = (size_t)blockIdx.x * (256u / ROW) + threadIdx.x / ROW; r < p.rows;
         r += (size_t)gridDim.x * (256u / ROW)) {
        const T* x = static_cast<const T*>(p.x) + r * p.x_stride;
        const R* res = p.residual ? static_cast<const R*>(p.residual) + r * p.residual_stride : nullptr;
        const auto value = [&](uint32_t c) { return to_float(x[c]) + (res ? to_float(res[c]) : 0.f); };
        float lift = 1.f, sum = 0.f;
        for (uint32_t c = tid; c < p.cols; c += ROW) sum += value(c) * value(c);
        sum = reduce.sum(sum);
        if (!(sum < INFINITY)) {
            lift = kNormLift;
            sum = 0.f;
            for (uint32_t c = tid; c < p.cols; c += ROW) sum += value(c) * lift * (value(c) * lift);
            sum = reduce.sum(sum);
        }
        const float s = norm_step(sum, p.cols, p.eps, lift);
        const auto norm = [&](float h, uint32_t c) { return h * lift * s * (p.weight ? p.weight[c] : 1.f); };
        RowStep st{};
        if (p.q) {
            uint32_t most = 0;
            for (uint32_t c = tid; c < p.cols; c += ROW)
                most = max(most, __float_as_uint(norm(value(c), c)) & 0x7fffffffu);
            st = row_step(reduce.most(most));
            if (tid == 0) p.scale[r] = st.scale;
        }
        for (uint32_t c = tid; c < p.cols; c += ROW) {
            const float h = value(c), y = norm(h, c);
            if (p.h) static_cast<R*>(p.h)[r * p.h_stride + c] = from_float<R>(h);
            if (p.y) static_cast<T*>(p.y)[r * p.y_stride + c] = from_float<T>(y);
            if (p.q) p.q[r * p.q_stride + c] = (int8_t)quant_byte(y, st);
        }
    }
}

// A row's dx and dresidual; with dw only its lift, step and mean(g n), for the kernel below.
template <typename T, typename R, uint32_t ROW>
__global__ void __launch_bounds__(256) norm_grad_rows_kernel(const NormGradParams p) {
    __shared__ float scratch[2][ROW / 32u];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    RowReduce<ROW> reduce{scratch};
    const uint32_t tid = threadIdx.x % ROW;
    for (size_t r = (size_t)blockIdx.x * (256u / ROW) + threadIdx.x / ROW; r < p.rows;
         r += (size_t)gridDim.x * (256u / ROW)) {
        const T* dy = static_cast<const T*>(p.dy) + r * p.dy_stride;
        const R* h = static_cast<const R*>(p.h) + r * p.h_stride;
        const R* dh = p.dh ? static_cast<const R*>(p.dh) + r * p.dh_stride : nullptr;
        const auto grad = [&](uint32_t c) { return to_float(dy[c]) * (p.weight ? p.weight[c] : 1.f); };
        float lift = 1.f, sum = 0.f, along = 0.f;
        const auto sums = [&] {
            sum = along = 0.f;
            for (uint32_t c = tid; c < p.cols; c += ROW) {
                const float v = to_float(h[c]) * lift;
                sum += v * v;
                along += grad(c) * v;
            }
            sum = reduce.sum(sum);
            along = reduce.sum(along);
        };
        sums();
        if (!(sum < INFINITY)) {
            lift = kNormLift;
            sums();
        }
        const float s = norm_step(sum, p.cols, p.eps, lift);
        const float mean = __fdiv_rn(along * s, (float)p.cols);
        if (p.dw) {
            if (tid == 0) p.row[r] = make_float4(lift, s, mean, 0.f);
            continue;
        }
        for (uint32_t c = tid; c < p.cols; c += ROW) {
            const float n = to_float(h[c]) * lift * s;
            const float d = (grad(c) - n * mean) * s * lift + (dh ? to_float(dh[c]) : 0.f);
            if (p.dx) static_cast<T*>(p.dx)[r * p.dx_stride + c] = from_float<T>(d);
            if (p.dres) static_cast<R*>(p.dres)[r * p.dres_stride + c] = from_float<R>(d);
        }
    }
}

// dx, dresidual, and part[y][c] = sum of dy n over the rows of part y. A thread a column.
template <typename T, typename R>
__global__ void __launch_bounds__(256) norm_grad_cols_kernel(const NormGradParams p, uint32_t rows_each) {
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    const uint32_t c = blockIdx.x * 256u + threadIdx.x;
    if (c >= p.cols) return;
    const uint32_t lo = blockIdx.y * rows_each, hi = min(p.rows, lo + rows_each);
    const float w = p.weight ? p.weight[c] : 1.f;
    float acc = 0.f;
    for (size_t r = lo; r < hi; ++r) {
        const float4 row = p.row[r];
        const float dy = to_float(static_cast<const T*>(p.dy)[r * p.dy_stride + c]);
        const float n = to_float(static_cast<const R*>(p.h)[r * p.h_stride + c]) * row.x * row.y;
        const float d = (dy * w - n * row.z) * row.y * row.x +
                        (p.dh ? to_float(static_cast<const R*>(p.dh)[r * p.dh_stride + c]) : 0.f);
        if (p.dx) static_cast<T*>(p.dx)[r * p.dx_stride + c] = from_float<T>(d);
        if (p.dres) static_cast<R*>(p.dres)[r * p.dres_stride + c] = from_float<R>(d);
        acc += dy * n;
    }
    p.part[(size_t)blockIdx.y * p.cols + c] = acc;
}

// dw[c] = sum of the parts, in order: 32 columns by 8 shares of the parts a CTA.
__global__ void __launch_bounds__(256) norm_grad_sum_kernel(const NormGradParams p, uint32_t parts) {
    __shared__ float at[8][32];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    const uint32_t lane = threadIdx.x & 31u, share = threadIdx.x >> 5, c = blockIdx.x * 32u + lane;
    float acc = 0.f;
    if (c < p.cols)
#pragma unroll 8
        for (uint32_t i = share; i < parts; i += 8u) acc += p.part[(size_t)i * p.cols + c];
    at[share][lane] = acc;
    __syncthreads();
    if (share || c >= p.cols) return;
#pragma unroll
    for (uint32_t i = 1; i < 8u; ++i) acc += at[i][lane];
    p.dw[c] = acc;
}

template <typename T, typename R>
cudaError_t norm_typed(const NormParams& p, cudaStream_t s) {
    return launch_chained(add_norm_kernel<T, R, 256>, dim3(p.rows < 65535u ? p.rows : 65535u), 256, 0, 0, s, p);
}

template <typename T, typename R>
cudaError_t grad_typed(const NormGradParams& p, cudaStream_t s) {
    cudaError_t e = launch_chained(norm_grad_rows_kernel<T, R, 256>, dim3(p.rows < 65535u ? p.rows : 65535u), 256, 0, 0, s, p);
    if (e != cudaSuccess || !p.dw) return e;
    const uint32_t each = (p.rows + kNormParts - 1u) / kNormParts, parts = (p.rows + each - 1u) / each;
    e = launch_chained(norm_grad_cols_kernel<T, R>, dim3((p.cols + 255u) / 256u, parts), 256, 0, 0, s, p, each);
    if (e != cudaSuccess) return e;
    return launch_chained(norm_grad_sum_kernel, dim3((p.cols + 31u) / 32u), 256, 0, 0, s, p, parts);
}

// The pairs of types: one type throughout, or the residual in f32.
template <typename F>
cudaError_t by_types(int type, int residual_type, F&& f) {
    if (type == VLB_DTYPE_F32 && residual_type == VLB_DTYPE_F32) return f(float{}, float{});
    if (type == VLB_DTYPE_F16 && residual_type == VLB_DTYPE_F16) return f(__half{}, __half{});
    if (type == VLB_DTYPE_F16 && residual_type == VLB_DTYPE_F32) return f(__half{}, float{});
    if (type == VLB_DTYPE_BF16 && residual_type == VLB_DTYPE_BF16) return f(__nv_bfloat16{}, __nv_bfloat16{});
    if (type == VLB_DTYPE_BF16 && residual_type == VLB_DTYPE_F32) return f(__nv_bfloat16{}, float{});
    return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_add_norm(const NormParams& p, int type, int residual_type, cudaStream_t s) {
    return by_types(type, residual_type, [&](auto t, auto r) { return norm_typed<decltype(t), decltype(r)>(p, s); });
}

cudaError_t launch_add_norm_grad(const NormGradParams& p, int type, int residual_type, cudaStream_t s) {
    return by_types(type, residual_type, [&](auto t, auto r) { return grad_typed<decltype(t), decltype(r)>(p, s); });
}

}  // namespace vlb
