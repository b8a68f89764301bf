// Tokens sorted by expert and back: the (token, slot) pairs of a route in the dispatch's stable order
// (expert, then token, then slot; deepseek_v4_graph.cpp:2134-2223), each pair's row, the weighted sum of
// a token's rows, and its gradient.
//
//   sort      a stable counting sort by expert: each block counts its pairs' experts, a block turns the
//             counts into every block's first place for every expert, and each pair then takes its place
//             by the pairs of its expert before it in its block
//   rows      rows[place(t, s)] = x[t]
//   combine   out[t] = sum_s w_ts rows[place(t, s)] + residual[t]
//   gradient  drows[place(t, s)] = w_ts dout[t],  dw_ts = <dout[t], rows[place(t, s)]>
//
// The order costs a few bytes a pair; moving the rows is what takes the time, and HBM bounds that.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "vlb_launch.h"
#include "vlb_rows.cuh"
#include "vlb_tcgen05.cuh"

namespace vlb {
namespace {

constexpr uint32_t kSortThreads = 512, kSortWarps = kSortThreads / 32u;

// The expert of pair i; E where it was dropped.
__device__ __forceinline__ uint32_t pair_expert(const SortParams& p, uint32_t i) {
    const uint32_t e = p.idx[i];
    return e < p.E && (!p.mask || p.mask[i / p.k]) ? e : p.E;
}

// counts[b][e] = pairs of block b (kSortThreads neighbours) on expert e.
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const SortParams p) {
    __shared__ uint32_t hist[kSortMaxExperts];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    const uint32_t n = p.T * p.k, i = blockIdx.x * kSortThreads + threadIdx.x;
    for (uint32_t e = threadIdx.x; e < p.E; e += kSortThreads) hist[e] = 0;
    __syncthreads();
    const uint32_t e = i < n ? pair_expert(p, i) : p.E;
    if (e < p.E) atomicAdd(hist + e, 1u);
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < p.E; e += kSortThreads) p.counts[(size_t)blockIdx.x * p.E + e] = hist[e];
}

// counts[b][e] = first place of block b's pairs on expert e; offsets. One block, a thread an expert.
__global__ void __launch_bounds__(kSortMaxExperts) sort_scan_kernel(const SortParams p, uint32_t blocks) {
    __shared__ uint32_t warps[32];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    const uint32_t e = threadIdx.x, lane = e & 31u;
    uint32_t sum = 0;
    if (e < p.E)
        for (uint32_t b = 0; b < blocks; ++b) {
            uint32_t* at = p.counts + (size_t)b * p.E + e;
            const uint32_t v = *at;
            *at = sum;
            sum += v;
        }
    uint32_t before = sum;
#pragma unroll
    for (uint32_t d = 1; d < 32u; d <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, before, d);
        if (lane >= d) before += v;
    }
    if (lane == 31u) warps[e >> 5] = before;
    __syncthreads();
    before -= sum;
    for (uint32_t w = 0; w < (e >> 5); ++w) before += warps[w];
    if (e >= p.E) return;
    p.offsets[e] = before;
    if (e + 1u == p.E) p.offsets[p.E] = before + sum;
    for (uint32_t b = 0; b < blocks; ++b) p.counts[(size_t)b * p.E + e] += before;
}

// Every pair's place and what goes there of it. Shared: [kSortWarps][E] the warps' pairs of each expert.
__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(const SortParams p) {
    extern __shared__ uint32_t by_warp[];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    const uint32_t n = p.T * p.k, i = blockIdx.x * kSortThreads + threadIdx.x;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    for (uint32_t q = threadIdx.x; q < kSortWarps * p.E; q += kSortThreads) by_warp[q] = 0;
    __syncthreads();
    const uint32_t e = i < n ? pair_expert(p, i) : p.E;
    const uint32_t same = __match_any_sync(0xffffffffu, e), ahead = __popc(same & ((1u << lane) - 1u));
    if (e < p.E && ahead == 0) by_warp[warp * p.E + e] = __popc(same);
    __syncthreads();
    if (i >= n) return;
    uint32_t place = VLB_NO_ROW;
    if (e < p.E) {
        place = p.counts[(size_t)blockIdx.x * p.E + e] + ahead;
        for (uint32_t w = 0; w < warp; ++w) place += by_warp[w * p.E + e];
        const uint32_t t = i / p.k;
        if (p.row_index) p.row_index[place] = t;
        if (p.row_weight) p.row_weight[place] = p.weights[i];
        if (p.row_scale) p.row_scale[place] = p.x_scale[t];
    }
    p.elem_row[i] = place;
}

// A token's row to its places: read once, written once a live slot. U: what a thread moves at a time.
template <typename U>
__global__ void __launch_bounds__(256) sort_rows_kernel(const SortParams p) {
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    const uint32_t units = (uint32_t)(p.row_bytes / sizeof(U));
    for (size_t t = blockIdx.x; t < p.T; t += gridDim.x) {
        const U* x = reinterpret_cast<const U*>(p.x + t * p.x_stride);
        for (uint32_t c = threadIdx.x; c < units; c += 256u) {
            const U v = x[c];
            for (uint32_t s = 0; s < p.k; ++s) {
                const uint32_t row = p.elem_row[t * p.k + s];
                if (row != VLB_NO_ROW) reinterpret_cast<U*>(p.rows + row * p.rows_stride)[c] = v;
            }
        }
    }
}

template <typename T, typename O>
__global__ void __launch_bounds__(256) combine_kernel(const CombineParams p) {
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    for (size_t t = blockIdx.x; t < p.T; t += gridDim.x)
        for (uint32_t c = threadIdx.x; c < p.H; c += 256u) {
            float acc = 0.f;
            for (uint32_t s = 0; s < p.k; ++s) {
                const uint32_t row = p.elem_row[t * p.k + s];
                if (row >= p.n_rows) continue;
                const float v = to_float(static_cast<const T*>(p.rows)[row * p.rows_stride + c]);
                acc = p.weights ? fmaf(p.weights[t * p.k + s], v, acc) : acc + v;
            }
            if (p.residual) acc += to_float(static_cast<const O*>(p.residual)[t * p.residual_stride + c]);
            static_cast<O*>(p.out)[t * p.out_stride + c] = from_float<O>(acc);
        }
}

template <typename T, typename O>
__global__ void __launch_bounds__(256) combine_grad_kernel(const CombineGradParams p) {
    __shared__ float scratch[2][8];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    RowReduce<256> reduce{scratch};
    for (size_t t = blockIdx.x; t < p.T; t += gridDim.x) {
        const O* dout = static_cast<const O*>(p.dout) + t * p.dout_stride;
        for (uint32_t s = 0; s < p.k; ++s) {
            const uint32_t row = p.elem_row[t * p.k + s];
            if (row >= p.n_rows) {
                if (p.dweights && threadIdx.x == 0) p.dweights[t * p.k + s] = 0.f;
                continue;
            }
            const float w = p.weights ? p.weights[t * p.k + s] : 1.f;
            float acc = 0.f;
            for (uint32_t c = threadIdx.x; c < p.H; c += 256u) {
                const float d = to_float(dout[c]);
                if (p.dweights) acc += d * to_float(static_cast<const T*>(p.rows)[row * p.rows_stride + c]);
                if (p.drows) static_cast<T*>(p.drows)[row * p.drows_stride + c] = from_float<T>(w * d);
            }
            if (!p.dweights) continue;
            acc = reduce.sum(acc);
            if (threadIdx.x == 0) p.dweights[t * p.k + s] = acc;
        }
    }
}

template <typename F>
cudaError_t by_type(int type, F&& f) {
    switch (type) {
        case VLB_DTYPE_F32: return f(float{});
        case VLB_DTYPE_F16: return f(__half{});
        case VLB_DTYPE_BF16: return f(__nv_bfloat16{});
        default: return cudaErrorInvalidValue;
    }
}

uint32_t token_blocks(uint32_t T) { return T < 65535u ? T : 65535u; }

}  // namespace

uint32_t sort_blocks(uint64_t pairs) { return (uint32_t)((pairs + kSortThreads - 1u) / kSortThreads); }

cudaError_t launch_sort_tokens(const SortParams& p, cudaStream_t s) {
    const uint32_t blocks = sort_blocks(p.T * p.k);
    cudaError_t e = launch_chained(sort_count_kernel, dim3(blocks), kSortThreads, 0, 0, s, p);
    if (e != cudaSuccess) return e;
    if ((e = launch_chained(sort_scan_kernel, dim3(1), kSortMaxExperts, 0, 0, s, p, blocks)) != cudaSuccess) return e;
    const size_t smem = (size_t)kSortWarps * p.E * 4u;
    if (smem > 48u * 1024u &&
        (e = cudaFuncSetAttribute(sort_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  (int)(kSortWarps * kSortMaxExperts * 4u))) != cudaSuccess)
        return e;
    if ((e = launch_chained(sort_place_kernel, dim3(blocks), kSortThreads, smem, 0, s, p)) != cudaSuccess) return e;
    if (!p.rows) return cudaSuccess;
    const dim3 grid(token_blocks(p.T));
    switch (p.elem) {
        case 1: return launch_chained(sort_rows_kernel<uint8_t>, grid, 256, 0, 0, s, p);
        case 2: return launch_chained(sort_rows_kernel<uint16_t>, grid, 256, 0, 0, s, p);
        default: return launch_chained(sort_rows_kernel<uint32_t>, grid, 256, 0, 0, s, p);
    }
}

cudaError_t launch_combine(const CombineParams& p, int type, int out_type, cudaStream_t s) {
    return by_type(type, [&](auto t) {
        return by_type(out_type, [&](auto o) {
            return launch_chained(combine_kernel<decltype(t), decltype(o)>, dim3(token_blocks(p.T)), 256, 0, 0, s, p);
        });
    });
}

cudaError_t launch_combine_grad(const CombineGradParams& p, int type, int out_type, cudaStream_t s) {
    return by_type(type, [&](auto t) {
        return by_type(out_type, [&](auto o) {
            return launch_chained(combine_grad_kernel<decltype(t), decltype(o)>, dim3(token_blocks(p.T)), 256, 0, 0, s, p);
        });
    });
}

}  // namespace vlb
