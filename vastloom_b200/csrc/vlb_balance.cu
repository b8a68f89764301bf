// The router's load-balance loss with per-expert counts and the gradient of the logits.
//
//   n_s   live tokens of sequence s;  c_se  their (token, slot) pairs on expert e
//   f_se = E c_se / (k n_s)           p_te = u(z_te) / sum_j u(z_tj),  u = exp, sigmoid or
//                                     sqrt(softplus)
//   d_t  = sum_e f_se p_te            L = coefficient * mean over the S' sequences with a live
//                                     token of (1 / n_s) sum_t d_t
//   dL/dz_te = coefficient / (S' n_s) * p_te (f_se - d_t) * r(z_te),   r = u' / u:
//              1, 1 - sigmoid(z), sigmoid(z) / (2 softplus(z))
//
// The counts carry no gradient, so they are taken first and one pass over the logits then gives
// both the loss (the sum of d_t) and the gradient. The reference routes only (it does not train):
// the scores are its routers' (deepseek_v4_reference.cpp:65-69, olmoe_runtime.cpp:1120-1137).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "vlb_launch.h"

namespace vlb {
namespace {

__device__ __forceinline__ float bl_float(float v) { return v; }
__device__ __forceinline__ float bl_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float bl_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void bl_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void bl_store(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void bl_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// The sequence that holds token t, or S when none does (offsets that do not rise hold none).
__device__ __forceinline__ uint32_t sequence_of(const BalanceParams& p, uint32_t t) {
    if (!p.seq_offsets) return 0;
    uint32_t lo = 0, hi = p.S;  // first s with offsets[s + 1] > t
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2u;
        if (p.seq_offsets[mid + 1] > t) hi = mid;
        else lo = mid + 1;
    }
    return lo < p.S && p.seq_offsets[lo] <= t ? lo : p.S;
}

__global__ void __launch_bounds__(256) balance_count_kernel(const BalanceParams p) {
    for (uint64_t t = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; t < p.T; t += (uint64_t)gridDim.x * blockDim.x) {
        if (p.mask && !p.mask[t]) continue;
        const uint32_t s = sequence_of(p, (uint32_t)t);
        if (s == p.S) continue;
        atomicAdd(p.live + s, 1u);
        for (uint32_t j = 0; j < p.k; ++j) {
            const uint32_t e = p.idx[t * p.k + j];
            if (e < p.E) atomicAdd(p.counts + (size_t)s * p.E + e, 1u);
        }
    }
}

// ln u(z) up to a row constant, as u(z) / scale(row), and r(z). With m = min(0, max z) taken out,
// the sums stay normal numbers however low a row's logits are.
template <int SCORE>
__device__ __forceinline__ void balance_score(float z, float m, float& u, float& r) {
    if (SCORE == VLB_SCORE_SOFTMAX) {
        u = expf(z - m);
        r = 1.f;
    } else if (SCORE == VLB_SCORE_SIGMOID) {
        const float e = expf(-fabsf(z)), d = 1.f / (1.f + e);
        u = expf(fminf(z, 0.f) - m) * d;
        r = z > 0.f ? e * d : d;
    } else {
        const float e = expf(-fabsf(z)), d = 1.f / (1.f + e), l = log1pf(e);
        if (z > 0.f) {
            const float sp = z + l;
            u = sqrtf(sp);
            r = d / (2.f * sp);
        } else {
            const float q = e > 0.f ? l / e : 1.f;  // softplus(z) / e^z
            u = sqrtf(q) * expf(0.5f * (z - m));
            r = d / (2.f * q);
        }
    }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

constexpr uint32_t kBalValues = 16;  // logits a lane holds: E <= 512

// One warp a token.
template <typename T, int SCORE>
__global__ void __launch_bounds__(256) balance_kernel(const BalanceParams p) {
    const uint32_t lane = threadIdx.x & 31u, warps = gridDim.x * (blockDim.x / 32u);
    __shared__ double part[8];
    __shared__ uint32_t alive_s;
    if (threadIdx.x == 0) alive_s = 0;
    __syncthreads();
    uint32_t mine = 0;
    for (uint32_t s = threadIdx.x; s < p.S; s += blockDim.x) mine += p.live[s] != 0;
    if (mine) atomicAdd(&alive_s, mine);
    __syncthreads();
    const float up = p.upstream ? *p.upstream : 1.f;
    const float base = alive_s ? p.coefficient / (float)alive_s : 0.f;
    double sum = 0.0;
    for (uint64_t t = blockIdx.x * (blockDim.x / 32u) + (threadIdx.x >> 5); t < p.T; t += warps) {
        const uint32_t s = p.mask && !p.mask[t] ? p.S : sequence_of(p, (uint32_t)t);
        T* grad = p.dlogits ? static_cast<T*>(p.dlogits) + t * p.grad_stride : nullptr;
        if (s == p.S) {
            if (grad)
                for (uint32_t e = lane; e < p.E; e += 32u) bl_store(grad + e, 0.f);
            continue;
        }
        const T* z = static_cast<const T*>(p.logits) + t * p.stride;
        const float n = (float)p.live[s], fs = (float)p.E / ((float)p.k * n);
        float u[kBalValues], r[kBalValues], f[kBalValues];
        float m = -INFINITY;
        bool nan = false;
#pragma unroll
        for (uint32_t j = 0; j < kBalValues; ++j) {
            const uint32_t e = lane + 32u * j;
            u[j] = e < p.E ? bl_float(z[e]) : -INFINITY;
            f[j] = e < p.E ? (float)p.counts[(size_t)s * p.E + e] * fs : 0.f;
            m = fmaxf(m, u[j]);
            nan |= u[j] != u[j];
        }
        m = warp_max(m);
        // no expert left by the row's mask: it adds nothing and gets no gradient
        const bool none = m == -INFINITY && !__any_sync(0xffffffffu, nan);
        if (SCORE != VLB_SCORE_SOFTMAX) m = fminf(m, 0.f);
        float total = 0.f, dot = 0.f;
#pragma unroll
        for (uint32_t j = 0; j < kBalValues; ++j) {
            const uint32_t e = lane + 32u * j;
            const float zj = u[j];
            if (e < p.E && !none) balance_score<SCORE>(zj, m, u[j], r[j]);
            else u[j] = 0.f, r[j] = 0.f;
            total += u[j];
            dot += u[j] * f[j];
        }
        total = warp_sum(total);
        dot = warp_sum(dot);
        const float inv = none ? 0.f : 1.f / total, d = dot * inv, weight = base / n;
        if (lane == 0) sum += (double)(weight * d);
        if (grad) {
            const float gw = up * weight * inv;
#pragma unroll
            for (uint32_t j = 0; j < kBalValues; ++j) {
                const uint32_t e = lane + 32u * j;
                if (e < p.E) bl_store(grad + e, u[j] > 0.f || u[j] != u[j] ? gw * u[j] * (f[j] - d) * r[j] : 0.f);
            }
        }
    }
    if (lane == 0) part[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t i = 1; i < blockDim.x / 32u; ++i) sum += part[i];
        p.partial[blockIdx.x] = sum;
    }
}

// The blocks' partial sums in one fixed order.
__global__ void balance_finish_kernel(const BalanceParams p, uint32_t n) {
    double v = 0.0;
    for (uint32_t i = threadIdx.x; i < n; i += 32u) v += p.partial[i];
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (threadIdx.x == 0) *p.loss = (float)v;
}

template <typename T>
cudaError_t balance_typed(const BalanceParams& p, unsigned grid, cudaStream_t s) {
    switch (p.score) {
        case VLB_SCORE_SQRT_SOFTPLUS: balance_kernel<T, VLB_SCORE_SQRT_SOFTPLUS><<<grid, 256, 0, s>>>(p); break;
        case VLB_SCORE_SIGMOID: balance_kernel<T, VLB_SCORE_SIGMOID><<<grid, 256, 0, s>>>(p); break;
        default: balance_kernel<T, VLB_SCORE_SOFTMAX><<<grid, 256, 0, s>>>(p); break;
    }
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_balance(const BalanceParams& p, cudaStream_t s) {
    cudaError_t e = cudaMemsetAsync(p.counts, 0, (size_t)p.S * p.E * 4, s);
    if (e == cudaSuccess) e = cudaMemsetAsync(p.live, 0, (size_t)p.S * 4, s);
    if (e != cudaSuccess) return e;
    unsigned grid = 0;
    if (p.T) {
        const unsigned blocks = (unsigned)((p.T + 255u) / 256u);
        balance_count_kernel<<<blocks < 1024u ? blocks : 1024u, 256, 0, s>>>(p);
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
        const unsigned want = (unsigned)((p.T + 7u) / 8u);
        grid = want < kBalanceBlocks ? want : kBalanceBlocks;
        switch (p.logits_type) {
            case VLB_DTYPE_F32: e = balance_typed<float>(p, grid, s); break;
            case VLB_DTYPE_F16: e = balance_typed<__half>(p, grid, s); break;
            default: e = balance_typed<__nv_bfloat16>(p, grid, s); break;
        }
        if (e != cudaSuccess) return e;
    }
    if (p.loss) {
        balance_finish_kernel<<<1, 32, 0, s>>>(p, grid);
        e = cudaGetLastError();
    }
    return e;
}

}  // namespace vlb
