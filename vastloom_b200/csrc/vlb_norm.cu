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
// Rows from which a ring pays, the threads and CTAs an SM of its kernels, and its depth: as many rows as a CTA's
// share of the shared memory holds, 16-byte pieces for each thread, at most 6.
constexpr uint32_t kRingRows = 1024, kRingSmem = 216u * 1024u, kNormThreads = 256, kGradThreads = 512;
__host__ __device__ constexpr uint32_t norm_ctas(uint32_t keep) { return keep > 2u ? 2u : 4u; }
__host__ __device__ constexpr uint32_t ring_depth(uint32_t pieces, uint32_t threads, uint32_t ctas) {
    return kRingSmem / ctas / (pieces * threads * 16u) < 6u ? kRingSmem / ctas / (pieces * threads * 16u) : 6u;
}

// 1 / sqrt(mean + eps) of a row's sum of lifted squares; share: 1 / cols.
__device__ __forceinline__ float norm_step(float sum, float share, float eps, float lift) {
    return __frsqrt_rn(fmaf(sum, share, eps * lift * lift));
}

// Bytes of y: V of them from column c on, n inside the row.
template <uint32_t V>
__device__ __forceinline__ void store_row_bytes(int8_t* q, const float (&y)[V], const RowStep& st, uint32_t n) {
    if constexpr (V == 1) {
        if (n) q[0] = (int8_t)quant_byte(y[0], st);
    } else {
        float v[V];
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) v[i] = st.inv == 0.f ? 0.f : y[i] * st.lift;
        store_bytes<V>(q, v, st, n);
    }
}

// What is done with row r once its pieces h are in registers: KEEP of V elements a thread, the first of them
// at column `first`, ROW * V apart. LONG: the row may go on behind them; that is read again in each step.
// Every element is read and written by one thread: outputs may lie over inputs.
template <typename T, typename R, uint32_t V, uint32_t ROW, uint32_t KEEP, bool LONG, typename REDUCE>
__device__ __forceinline__ void norm_row(const NormParams& p, size_t r, float (&h)[KEEP][V], REDUCE& reduce) {
    constexpr uint32_t kStep = ROW * V;
    const uint32_t first = threadIdx.x % ROW * V, end = LONG ? p.cols : 0u;
    const auto left = [&](uint32_t c) { return c < p.cols ? p.cols - c : 0u; };
    const auto again = [&](uint32_t c, float (&f)[V]) {
        unpack(load_pack<V>(static_cast<const T*>(p.x) + r * p.x_stride + c, left(c)), f);
        if (!p.residual) return;
        float more[V];
        unpack(load_pack<V>(static_cast<const R*>(p.residual) + r * p.residual_stride + c, left(c)), more);
#pragma unroll
        for (uint32_t j = 0; j < V; ++j) f[j] += more[j];
    };
    const auto squares = [&](float lift) {
        float sum = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i)
#pragma unroll
            for (uint32_t j = 0; j < V; ++j) sum = fmaf(h[i][j] * lift, h[i][j] * lift, sum);
        for (uint32_t c = first + KEEP * kStep; c < end; c += kStep) {
            float f[V];
            again(c, f);
#pragma unroll
            for (uint32_t j = 0; j < V; ++j) sum = fmaf(f[j] * lift, f[j] * lift, sum);
        }
        return reduce.sum(sum);
    };
    float lift = 1.f, sum = squares(1.f);
    if (!(sum < INFINITY)) sum = squares(lift = kNormLift);
    const float s = norm_step(sum, p.share, p.eps, lift) * lift;
    // h to y, from column c on
    const auto norm = [&](float (&f)[V], uint32_t c) {
#pragma unroll
        for (uint32_t j = 0; j < V; ++j) f[j] *= s;
        if (!p.weight) return;
        const Pack<float, V> w = load_pack<V>(p.weight + c, left(c));
#pragma unroll
        for (uint32_t j = 0; j < V; ++j) f[j] *= w.v[j];
    };
#pragma unroll
    for (uint32_t i = 0; i < KEEP; ++i) {
        const uint32_t c = first + i * kStep;
        if (p.h) store_pack<V>(static_cast<R*>(p.h) + r * p.h_stride + c, h[i], left(c));
        norm(h[i], c);
        if (p.y) store_pack<V>(static_cast<T*>(p.y) + r * p.y_stride + c, h[i], left(c));
    }
    RowStep st{};
    if (p.q) {
        uint32_t most = 0;
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i)  // zeros behind the row's end, also where the row is NaN
#pragma unroll
            for (uint32_t j = 0; j < V; ++j)
                if (first + i * kStep + j < p.cols) most = max(most, __float_as_uint(h[i][j]) & 0x7fffffffu);
        for (uint32_t c = first + KEEP * kStep; c < end; c += kStep) {
            float f[V];
            again(c, f);
            norm(f, c);
#pragma unroll
            for (uint32_t j = 0; j < V; ++j)
                if (c + j < p.cols) most = max(most, __float_as_uint(f[j]) & 0x7fffffffu);
        }
        st = row_step(reduce.most(most));
        if (threadIdx.x % ROW == 0) p.scale[r] = st.scale;
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i)
            store_row_bytes<V>(p.q + r * p.q_stride + first + i * kStep, h[i], st, min(V, left(first + i * kStep)));
    }
    for (uint32_t c = first + KEEP * kStep; c < end; c += kStep) {
        float f[V];
        again(c, f);
        if (p.h) store_pack<V>(static_cast<R*>(p.h) + r * p.h_stride + c, f, left(c));
        norm(f, c);
        if (p.y) store_pack<V>(static_cast<T*>(p.y) + r * p.y_stride + c, f, left(c));
        if (p.q) store_row_bytes<V>(p.q + r * p.q_stride + c, f, st, min(V, left(c)));
    }
}

// Few rows, rows at any alignment (V 1), rows longer than the pieces: a CTA a row, loads straight to registers.
template <typename T, typename R, uint32_t V, uint32_t ROW, uint32_t KEEP, bool LONG>
__global__ void __launch_bounds__(ROW) add_norm_kernel(const NormParams p) {
    constexpr uint32_t kStep = ROW * V;
    __shared__ float scratch[2][ROW / 32u];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    RowReduce<ROW> reduce{scratch};
    const uint32_t first = threadIdx.x * V;
    for (size_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const auto left = [&](uint32_t c) { return c < p.cols ? p.cols - c : 0u; };
        const T* x = static_cast<const T*>(p.x) + r * p.x_stride;
        Pack<T, V> a[KEEP];  // all loads first
        Pack<R, V> b[KEEP];
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i) a[i] = load_pack<V>(x + first + i * kStep, left(first + i * kStep));
        if (p.residual) {
            const R* res = static_cast<const R*>(p.residual) + r * p.residual_stride;
#pragma unroll
            for (uint32_t i = 0; i < KEEP; ++i) b[i] = load_pack<V>(res + first + i * kStep, left(first + i * kStep));
        }
        float h[KEEP][V];
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i) {
            unpack(a[i], h[i]);
            if (!p.residual) continue;
            float more[V];
            unpack(b[i], more);
#pragma unroll
            for (uint32_t j = 0; j < V; ++j) h[i][j] += more[j];
        }
        norm_row<T, R, V, ROW, KEEP, LONG>(p, r, h, reduce);
    }
}

// A ring of rows in shared memory, filled by cp.async: thread by thread, each reading back what it asked for
// itself, so that waiting for its own copies is all the synchronisation there is. PIECES 16-byte pieces of a
// row a thread, DEPTH rows.
template <uint32_t THREADS, uint32_t PIECES, uint32_t DEPTH>
struct RowRing {
    uint4* at;  // [DEPTH][PIECES][THREADS]
    uint32_t stage = 0;
    __device__ __forceinline__ uint4* slot(uint32_t st, uint32_t piece) { return at + (st * PIECES + piece) * THREADS + threadIdx.x; }
    // V elements from p on, `left` of them inside the row (zeros behind), as pieces `piece` on of stage st
    template <uint32_t V, typename E>
    __device__ __forceinline__ void ask(uint32_t st, uint32_t piece, const E* p, uint32_t left) {
        constexpr uint32_t kPer = 16u / sizeof(E);
#pragma unroll
        for (uint32_t i = 0; i < V / kPer; ++i) {
            const uint32_t have = left > i * kPer ? min(left - i * kPer, kPer) : 0u;
            tc::cp_async16(slot(st, piece + i), have ? p + i * kPer : p, have * (uint32_t)sizeof(E));
        }
    }
    template <uint32_t V, typename E>
    __device__ __forceinline__ Pack<E, V> get(uint32_t piece) {
        constexpr uint32_t kPer = 16u / sizeof(E);
        Pack<E, V> a;
#pragma unroll
        for (uint32_t i = 0; i < V / kPer; ++i) reinterpret_cast<uint4*>(&a)[i] = *slot(stage, piece + i);
        return a;
    }
    __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory"); }
};

// Many rows: persistent CTAs, DEPTH rows ahead on their way to shared memory, since the registers that h
// takes leave too few threads to hold enough loads in flight themselves.
template <typename T, typename R, uint32_t ROW, uint32_t KEEP, uint32_t DEPTH>
__global__ void __launch_bounds__(kNormThreads, norm_ctas(KEEP)) add_norm_ring_kernel(const NormParams p) {
    constexpr uint32_t V = 16u / sizeof(T), kThreads = kNormThreads, kRows = kThreads / ROW, kStep = ROW * V, kRes = sizeof(R) / sizeof(T);
    constexpr uint32_t kPieces = KEEP * (1u + kRes);
    static_assert(DEPTH >= 1u, "a row has to fit");
    extern __shared__ uint4 ring_smem[];
    __shared__ float scratch[kRows][2][ROW / 32u];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    RowReduce<ROW, kThreads> reduce{scratch[threadIdx.x / ROW]};
    RowRing<kThreads, kPieces, DEPTH> ring{ring_smem};
    const uint32_t first = threadIdx.x % ROW * V;
    const size_t step = (size_t)gridDim.x * kRows;
    size_t ahead = (size_t)blockIdx.x * kRows + threadIdx.x / ROW;
    const auto ask = [&](uint32_t st) {
        if (ahead < p.rows) {
            const T* x = static_cast<const T*>(p.x) + ahead * p.x_stride;
            const R* res = static_cast<const R*>(p.residual) + ahead * p.residual_stride;
#pragma unroll
            for (uint32_t i = 0; i < KEEP; ++i) {
                const uint32_t c = first + i * kStep, left = c < p.cols ? p.cols - c : 0u;
                ring.template ask<V>(st, i, x + (left ? c : 0u), left);
                if (p.residual) ring.template ask<V>(st, KEEP + i * kRes, res + (left ? c : 0u), left);
            }
        }
        tc::cp_async_commit();
        ahead += step;
    };
    size_t r = ahead;
#pragma unroll
    for (uint32_t i = 0; i + 1u < DEPTH; ++i) ask(i);
    for (; r < p.rows; r += step) {
        ask(ring.stage ? ring.stage - 1u : DEPTH - 1u);
        ring.wait();
        float h[KEEP][V];
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i) {
            unpack(ring.template get<V, T>(i), h[i]);
            if (!p.residual) continue;
            float more[V];
            unpack(ring.template get<V, R>(KEEP + i * kRes), more);
#pragma unroll
            for (uint32_t j = 0; j < V; ++j) h[i][j] += more[j];
        }
        norm_row<T, R, V, ROW, KEEP, false>(p, r, h, reduce);
        if (++ring.stage == DEPTH) ring.stage = 0;
    }
    tc::cp_async_wait_all();
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
        const float s = norm_step(sum, p.share, p.eps, lift);
        const float mean = along * s * p.share;
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

// The weights of a thread's columns (zeros behind the row's end), the same in every row.
template <uint32_t V, uint32_t ROW, uint32_t KEEP>
__device__ __forceinline__ void row_weights(const float* weight, uint32_t cols, float (&w)[KEEP][V]) {
#pragma unroll
    for (uint32_t i = 0; i < KEEP; ++i) {
        const uint32_t c = threadIdx.x % ROW * V + i * ROW * V, left = c < cols ? cols - c : 0u;
        Pack<float, V> a;
        if (weight) a = load_pack<V>(weight + (left ? c : 0u), left);
#pragma unroll
        for (uint32_t j = 0; j < V; ++j) w[i][j] = weight ? a.v[j] : 1.f;
    }
}

// Row r; adds dy n to acc. dy, h and dh give piece i (from registers, or again from shared memory: holding all
// three beside the weights and the sums would take more registers than there are).
template <typename T, typename R, uint32_t V, uint32_t ROW, uint32_t KEEP, typename DY, typename H, typename DH, typename REDUCE>
__device__ __forceinline__ void norm_grad_row(const NormGradParams& p, size_t r, DY&& dy, H&& h, DH&& dh,
                                              const float (&w)[KEEP][V], float (&acc)[KEEP][V], REDUCE& reduce, REDUCE& reduce2) {
    constexpr uint32_t kStep = ROW * V;
    const uint32_t first = threadIdx.x % ROW * V;
    const auto left = [&](uint32_t c) { return c < p.cols ? p.cols - c : 0u; };
    float sum, along;
    const auto sums = [&](float lift) {
        sum = along = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i) {
            float g[V], v[V];
            unpack(dy(i), g);
            unpack(h(i), v);
#pragma unroll
            for (uint32_t j = 0; j < V; ++j) {
                const float n = v[j] * lift;
                sum = fmaf(n, n, sum);
                along = fmaf(g[j] * w[i][j], n, along);
            }
        }
        reduce_two(reduce, reduce2, sum, along);
    };
    float lift = 1.f;
    sums(1.f);
    if (!(sum < INFINITY)) sums(lift = kNormLift);
    const float step = norm_step(sum, p.share, p.eps, lift), s = step * lift;
    const float mean = along * step * p.share;
#pragma unroll
    for (uint32_t i = 0; i < KEEP; ++i) {
        const uint32_t c = first + i * kStep;
        float g[V], v[V], d[V];
        unpack(dy(i), g);
        unpack(h(i), v);
#pragma unroll
        for (uint32_t j = 0; j < V; ++j) {
            const float n = v[j] * s;
            d[j] = fmaf(-n, mean, g[j] * w[i][j]) * s;
            acc[i][j] = fmaf(g[j], n, acc[i][j]);
        }
        if (p.dh) {
            unpack(dh(i), v);
#pragma unroll
            for (uint32_t j = 0; j < V; ++j) d[j] += v[j];
        }
        if (p.dx) store_pack<V>(static_cast<T*>(p.dx) + r * p.dx_stride + c, d, left(c));
        if (p.dres) store_pack<V>(static_cast<R*>(p.dres) + r * p.dres_stride + c, d, left(c));
    }
}

// The CTA's part of the weight's gradient. all: where it holds several rows, room for a piece of each.
template <uint32_t V, uint32_t ROW, uint32_t KEEP, uint32_t THREADS>
__device__ __forceinline__ void norm_grad_part(const NormGradParams& p, const float (&acc)[KEEP][V], float* all) {
    constexpr uint32_t kRows = THREADS / ROW, kStep = ROW * V;
    const uint32_t first = threadIdx.x % ROW * V;
    float* part = p.part + (size_t)blockIdx.x * p.cols;
    if constexpr (kRows > 1u) {  // the rows' sums, in order
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i) {
            __syncthreads();
#pragma unroll
            for (uint32_t j = 0; j < V; ++j) all[threadIdx.x / ROW * kStep + first + j] = acc[i][j];
            __syncthreads();
            for (uint32_t c = threadIdx.x; c < kStep && i * kStep + c < p.cols; c += THREADS) {
                float v = all[c];
#pragma unroll
                for (uint32_t k = 1; k < kRows; ++k) v += all[k * kStep + c];
                part[i * kStep + c] = v;
            }
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i)
#pragma unroll
            for (uint32_t j = 0; j < V; ++j)
                if (first + i * kStep + j < p.cols) part[first + i * kStep + j] = acc[i][j];
    }
}

// Rows that registers hold whole, in one pass: a CTA takes every gridDim.x-th row and adds up dy n of its rows
// in registers, a column always in the same thread; it leaves one part.
template <typename T, typename R, uint32_t V, uint32_t ROW, uint32_t KEEP>
__global__ void __launch_bounds__(ROW) norm_grad_kernel(const NormGradParams p) {
    constexpr uint32_t kStep = ROW * V;
    __shared__ float scratch[2][2][ROW / 32u];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    RowReduce<ROW> reduce{scratch[0]}, reduce2{scratch[1]};
    const uint32_t first = threadIdx.x % ROW * V;
    const auto left = [&](uint32_t c) { return c < p.cols ? p.cols - c : 0u; };
    float acc[KEEP][V] = {}, w[KEEP][V];
    row_weights<V, ROW, KEEP>(p.weight, p.cols, w);
    for (size_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        Pack<T, V> dy[KEEP];
        Pack<R, V> h[KEEP], dh[KEEP];
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i) {
            const uint32_t c = first + i * kStep;
            dy[i] = load_pack<V>(static_cast<const T*>(p.dy) + r * p.dy_stride + c, left(c));
            h[i] = load_pack<V>(static_cast<const R*>(p.h) + r * p.h_stride + c, left(c));
            if (p.dh) dh[i] = load_pack<V>(static_cast<const R*>(p.dh) + r * p.dh_stride + c, left(c));
        }
        norm_grad_row<T, R, V, ROW, KEEP>(
            p, r, [&](uint32_t i) { return dy[i]; }, [&](uint32_t i) { return h[i]; }, [&](uint32_t i) { return dh[i]; }, w,
            acc, reduce, reduce2);
    }
    if (p.dw) norm_grad_part<V, ROW, KEEP, ROW>(p, acc, nullptr);
}

// The same with rows ahead on their way to shared memory, as add_norm_ring_kernel.
template <typename T, typename R, uint32_t ROW, uint32_t KEEP, uint32_t DEPTH>
__global__ void __launch_bounds__(kGradThreads, 1) norm_grad_ring_kernel(const NormGradParams p) {
    constexpr uint32_t V = 16u / sizeof(T), kThreads = kGradThreads, kRows = kThreads / ROW, kStep = ROW * V, kRes = sizeof(R) / sizeof(T);
    constexpr uint32_t kH = KEEP, kDh = KEEP * (1u + kRes), kPieces = KEEP * (1u + 2u * kRes);
    static_assert(DEPTH >= 1u, "a row has to fit");
    extern __shared__ uint4 ring_smem[];
    __shared__ float scratch[2][kRows][2][ROW / 32u];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    RowReduce<ROW, kThreads> reduce{scratch[0][threadIdx.x / ROW]}, reduce2{scratch[1][threadIdx.x / ROW]};
    RowRing<kThreads, kPieces, DEPTH> ring{ring_smem};
    const uint32_t first = threadIdx.x % ROW * V;
    const size_t step = (size_t)gridDim.x * kRows;
    size_t ahead = (size_t)blockIdx.x * kRows + threadIdx.x / ROW;
    const auto ask = [&](uint32_t st) {
        if (ahead < p.rows) {
            const T* dy = static_cast<const T*>(p.dy) + ahead * p.dy_stride;
            const R* h = static_cast<const R*>(p.h) + ahead * p.h_stride;
            const R* dh = static_cast<const R*>(p.dh) + ahead * p.dh_stride;
#pragma unroll
            for (uint32_t i = 0; i < KEEP; ++i) {
                const uint32_t c = first + i * kStep, left = c < p.cols ? p.cols - c : 0u, at = left ? c : 0u;
                ring.template ask<V>(st, i, dy + at, left);
                ring.template ask<V>(st, kH + i * kRes, h + at, left);
                if (p.dh) ring.template ask<V>(st, kDh + i * kRes, dh + at, left);
            }
        }
        tc::cp_async_commit();
        ahead += step;
    };
    size_t r = ahead;
#pragma unroll
    for (uint32_t i = 0; i + 1u < DEPTH; ++i) ask(i);
    float acc[KEEP][V] = {}, w[KEEP][V];
    row_weights<V, ROW, KEEP>(p.weight, p.cols, w);
    for (; r < p.rows; r += step) {
        ask(ring.stage ? ring.stage - 1u : DEPTH - 1u);
        ring.wait();
        norm_grad_row<T, R, V, ROW, KEEP>(
            p, r, [&](uint32_t i) { return ring.template get<V, T>(i); },
            [&](uint32_t i) { return ring.template get<V, R>(kH + i * kRes); },
            [&](uint32_t i) { return ring.template get<V, R>(kDh + i * kRes); }, w, acc, reduce, reduce2);
        if (++ring.stage == DEPTH) ring.stage = 0;
    }
    tc::cp_async_wait_all();
    if (p.dw) norm_grad_part<V, ROW, KEEP, kThreads>(p, acc, reinterpret_cast<float*>(ring_smem));
}

// dw[c] = sum of the parts, in order: 32 columns by 32 shares of the parts a CTA.
__global__ void __launch_bounds__(1024) norm_grad_sum_kernel(const NormGradParams p, uint32_t parts) {
    __shared__ float at[32][32];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    const uint32_t lane = threadIdx.x & 31u, share = threadIdx.x >> 5, c = blockIdx.x * 32u + lane;
    float acc = 0.f;
    if (c < p.cols)
#pragma unroll 8
        for (uint32_t i = share; i < parts; i += 32u) acc += p.part[(size_t)i * p.cols + c];
    at[share][lane] = acc;
    __syncthreads();
    if (share || c >= p.cols) return;
#pragma unroll
    for (uint32_t i = 1; i < 32u; ++i) acc += at[i][lane];
    p.dw[c] = acc;
}

bool on16(const void* p, size_t stride_bytes) { return reinterpret_cast<uintptr_t>(p) % 16u == 0 && stride_bytes % 16u == 0; }

// Calls f with the pieces a thread takes of a row, as types: of V elements, ROW threads, KEEP pieces.
template <uint32_t V_, uint32_t ROW_, uint32_t KEEP_>
struct Shape {
    static constexpr uint32_t V = V_, ROW = ROW_, KEEP = KEEP_;
};

constexpr uint32_t ring_depth(uint32_t pieces, uint32_t ctas) {
    return kRingSmem / ctas / (pieces * 256u * 16u) < 6u ? kRingSmem / ctas / (pieces * 256u * 16u) : 6u;
}
uint32_t ring_blocks(uint32_t ctas, uint32_t rows) {
    const uint32_t all = ctas * sm_count();
    return rows < all ? rows : all;
}
template <typename K, typename P>
cudaError_t launch_ring(K* kernel, uint32_t pieces, uint32_t threads, uint32_t blocks, cudaStream_t s, const P& p) {
    const size_t smem = (size_t)pieces * threads * 16u;
    const cudaError_t e = smem_once(kernel, smem);
    if (e != cudaSuccess) return e;
    return launch_chained(kernel, dim3(blocks), threads, smem, 0, s, p);
}

template <typename T, typename R>
cudaError_t norm_typed(const NormParams& p, cudaStream_t s) {
    constexpr uint32_t N = 16u / sizeof(T);
    const auto run = [&](auto shape) {
        using S = decltype(shape);
        const bool whole = p.cols <= S::V * S::ROW * S::KEEP;
        return launch_chained(whole ? add_norm_kernel<T, R, S::V, S::ROW, S::KEEP, false>
                                    : add_norm_kernel<T, R, S::V, S::ROW, S::KEEP, true>,
                              dim3(p.rows < 65535u ? p.rows : 65535u), S::ROW, 0, 0, s, p);
    };
    const auto run_ring = [&](auto shape) {
        using S = decltype(shape);
        constexpr uint32_t kPieces = S::KEEP * (1u + sizeof(R) / sizeof(T)), kCtas = norm_ctas(S::KEEP), kRows = kNormThreads / S::ROW;
        constexpr uint32_t kDepth = ring_depth(kPieces, kNormThreads, kCtas);
        return launch_ring(add_norm_ring_kernel<T, R, S::ROW, S::KEEP, kDepth>, kPieces * kDepth, kNormThreads,
                           ring_blocks(kCtas, (p.rows + kRows - 1u) / kRows), s, p);
    };
    const bool vec = on16(p.x, p.x_stride * sizeof(T)) && on16(p.residual, p.residual_stride * sizeof(R)) &&
                     on16(p.h, p.h_stride * sizeof(R)) && on16(p.y, p.y_stride * sizeof(T)) && on16(p.weight, 0) &&
                     reinterpret_cast<uintptr_t>(p.q) % N == 0 && p.q_stride % N == 0;
    if (!vec) {
        if (p.cols <= 256u * 4u) return run(Shape<1, 256, 4>{});
        return run(Shape<1, 512, 8>{});
    }
    const uint32_t packs = (p.cols + N - 1u) / N;
    if (p.rows >= kRingRows) {
        if (packs <= 32u) return run_ring(Shape<N, 32, 1>{});
        if (packs <= 64u) return run_ring(Shape<N, 32, 2>{});
        if (packs <= 128u) return run_ring(Shape<N, 64, 2>{});
        if (packs <= 256u) return run_ring(Shape<N, 128, 2>{});
        if (packs <= 512u) return run_ring(Shape<N, 256, 2>{});
        if (packs <= 1024u) return run_ring(Shape<N, 256, 4>{});
    }
    if (packs <= 256u) return run(Shape<N, 256, 1>{});
    if (packs <= 512u) return run(Shape<N, 512, 1>{});
    if (packs <= 1024u) return run(Shape<N, 512, 2>{});
    return run(Shape<N, 512, 4>{});
}

template <typename T, typename R>
cudaError_t grad_typed(const NormGradParams& p, cudaStream_t s) {
    constexpr uint32_t N = 16u / sizeof(T);
    const auto sum = [&](uint32_t parts) {
        return launch_chained(norm_grad_sum_kernel, dim3((p.cols + 31u) / 32u), 1024, 0, 0, s, p, parts);
    };
    const auto run = [&](auto shape) {
        using S = decltype(shape);
        const uint32_t blocks = p.rows < kNormParts ? p.rows : kNormParts;
        const cudaError_t e = launch_chained(norm_grad_kernel<T, R, S::V, S::ROW, S::KEEP>, dim3(blocks), S::ROW, 0, 0, s, p);
        return e != cudaSuccess || !p.dw ? e : sum(blocks);
    };
    const bool vec = on16(p.dy, p.dy_stride * sizeof(T)) && on16(p.h, p.h_stride * sizeof(R)) &&
                     on16(p.dh, p.dh_stride * sizeof(R)) && on16(p.dx, p.dx_stride * sizeof(T)) &&
                     on16(p.dres, p.dres_stride * sizeof(R)) && on16(p.weight, 0);
    const auto run_ring = [&](auto shape) {
        using S = decltype(shape);
        constexpr uint32_t kPieces = S::KEEP * (1u + 2u * sizeof(R) / sizeof(T)), kRows = kGradThreads / S::ROW;
        constexpr uint32_t kDepth = ring_depth(kPieces, kGradThreads, 1);
        const uint32_t all = ring_blocks(1, (p.rows + kRows - 1u) / kRows), blocks = all < kNormParts ? all : kNormParts;
        const cudaError_t e =
            launch_ring(norm_grad_ring_kernel<T, R, S::ROW, S::KEEP, kDepth>, kPieces * kDepth, kGradThreads, blocks, s, p);
        return e != cudaSuccess || !p.dw ? e : sum(blocks);
    };
    if (vec) {
        const uint32_t packs = (p.cols + N - 1u) / N;
        if (p.rows >= kRingRows) {
            if (packs <= 32u) return run_ring(Shape<N, 32, 1>{});
            if (packs <= 64u) return run_ring(Shape<N, 32, 2>{});
            if (packs <= 128u) return run_ring(Shape<N, 64, 2>{});
            if (packs <= 256u) return run_ring(Shape<N, 128, 2>{});
            if (packs <= 512u) return run_ring(Shape<N, 128, 4>{});
            if (packs <= 1024u) return run_ring(Shape<N, 256, 4>{});
        }
        if (packs <= 256u) return run(Shape<N, 256, 1>{});
        if (packs <= 512u) return run(Shape<N, 256, 2>{});
        if (packs <= 1024u) return run(Shape<N, 512, 2>{});
        if (packs <= 2048u) return run(Shape<N, 1024, 2>{});
    } else {
        if (p.cols <= 256u * 4u) return run(Shape<1, 256, 4>{});
        if (p.cols <= 512u * 8u) return run(Shape<1, 512, 8>{});
    }
    cudaError_t e = launch_chained(norm_grad_rows_kernel<T, R, 256>, dim3(p.rows < 65535u ? p.rows : 65535u), 256, 0, 0, s, p);
    if (e != cudaSuccess || !p.dw) return e;
    const uint32_t each = (p.rows + kNormParts - 1u) / kNormParts, parts = (p.rows + each - 1u) / each;
    e = launch_chained(norm_grad_cols_kernel<T, R>, dim3((p.cols + 255u) / 256u, parts), 256, 0, 0, s, p, each);
    return e != cudaSuccess ? e : sum(parts);
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
