// The residual's addition and RMS norm, with rows in the activations' type and in 8 bits, and its gradient.
//
//   forward    h = x + residual,  s = 1 / sqrt(mean h^2 + eps),  y = h s w;  a = max |y|,
//              q = rint(y * (127 / a)), scale = a / 127
//   gradient   n = h s,  g = dy w,  d = s (g - n mean(g n)) + dh,  dw = sum over rows of dy n
//
// Both move every element once and do a dozen operations on it: HBM bounds them. The sums are in 32 bits.
// Where the squares pass them (h above 1.8e19) the row is taken again with h lifted by 2^-100.
//
// Rows come as pieces of V neighbouring elements (16 bytes of the wider type), ROW threads a row, KEEP pieces
// a thread. A matrix whose stride is no multiple of V has its rows at V different offsets from a 16-byte
// boundary: pieces then start on the boundary before the row, and a thread takes only rows of one offset,
// so that its columns, their weights and their sums stay its own.
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

// Holds over the whole range: the largest h becomes 2^28, and 2^30 such squares stay below 2^86; a row that gets
// here has a sum of 2^128 at least, lifted 2^-72 and its mean 2^-102, far above the subnormals (eps, where lifted it
// underflows, is below 2^-45 of the mean). s itself is subnormal once the mean passes 2^252: within 2^-22 then.
constexpr float kNormLift = 0x1p-100f;

// The rings' shared memory an SM, threads and CTAs an SM, and depth: as many rows as a CTA's share holds of
// `bytes` a thread, at most 6.
constexpr uint32_t kRingSmem = 216u * 1024u, kGradThreads = 512;
__host__ __device__ constexpr uint32_t norm_threads(uint32_t row) { return row > 256u ? row : 256u; }
__host__ __device__ constexpr uint32_t norm_ctas(uint32_t row, uint32_t elements, bool shifted) {
    return (elements > 16u ? 512u : shifted ? 768u : 1024u) / norm_threads(row);
}
__host__ __device__ constexpr uint32_t ring_depth(uint32_t bytes, uint32_t threads, uint32_t ctas) {
    return kRingSmem / ctas / (bytes * threads) < 6u ? kRingSmem / ctas / (bytes * threads) : 6u;
}

// 1 / sqrt(mean + eps) of a row's sum of lifted squares; share: 1 / cols.
__device__ __forceinline__ float norm_step(float sum, float share, float eps, float lift) {
    return __frsqrt_rn(fmaf(sum, share, eps * lift * lift));
}

// A ring of rows in shared memory, filled by cp.async: thread by thread, each reading back what it asked for
// itself, so that waiting for its own copies is all the synchronisation there is. BYTES of a row a thread,
// DEPTH rows; `before`: the bytes a thread has of the operands in front.
template <uint32_t THREADS, uint32_t BYTES, uint32_t DEPTH>
struct RowRing {
    static_assert(DEPTH >= 1u, "a row has to fit");
    char* at;
    uint32_t stage = 0;
    template <uint32_t SIZE>
    __device__ __forceinline__ char* slot(uint32_t st, uint32_t before, uint32_t piece) const {
        return at + (st * BYTES + before) * THREADS + (piece * THREADS + threadIdx.x) * SIZE;
    }
    // piece `piece` at p, columns c .. c + V - 1 of cols: zeros behind the row, what lies before it as it is
    template <uint32_t V, typename E>
    __device__ __forceinline__ void ask(uint32_t st, uint32_t before, uint32_t piece, const E* p, int32_t c, uint32_t cols) const {
        constexpr uint32_t kSize = V * sizeof(E);
        const int32_t left = (int32_t)cols - c;
        const uint32_t have = left <= 0 ? 0u : min((uint32_t)left, V) * (uint32_t)sizeof(E);
        char* to = slot<kSize>(st, before, piece);
        if (have == 0) {  // no address of this row's
            if constexpr (kSize == 16) *reinterpret_cast<uint4*>(to) = make_uint4(0u, 0u, 0u, 0u);
            else *reinterpret_cast<uint2*>(to) = make_uint2(0u, 0u);
        } else if constexpr (kSize == 16) {
            tc::cp_async16(to, p, have);
        } else {
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(tc::smem_u32(to)), "l"(p), "r"(have) : "memory");
        }
    }
    template <uint32_t V, typename E>
    __device__ __forceinline__ Pack<E, V> get(uint32_t before, uint32_t piece) const {
        return *reinterpret_cast<const Pack<E, V>*>(slot<V * sizeof(E)>(stage, before, piece));
    }
    __device__ __forceinline__ uint32_t behind() const { return stage ? stage - 1u : DEPTH - 1u; }
    __device__ __forceinline__ void next() {
        if (++stage == DEPTH) stage = 0;
    }
    __device__ __forceinline__ void wait() const { asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory"); }
};

// The weights of a thread's columns from c0 on (zeros outside the row), the same in every row it takes.
template <uint32_t V, uint32_t ROW, uint32_t KEEP>
__device__ __forceinline__ void row_weights(const float* weight, int32_t c0, uint32_t cols, float (&w)[KEEP][V]) {
    const bool wide = V % 4 == 0 && weight && reinterpret_cast<uintptr_t>(weight + c0) % 16u == 0;
#pragma unroll
    for (uint32_t i = 0; i < KEEP; ++i) {
        const int32_t c = c0 + (int32_t)(i * ROW * V);
        if (wide && inside(c, V, cols)) {
            const Pack<float, V> a = *reinterpret_cast<const Pack<float, V>*>(weight + c);
            unpack(a, w[i]);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < V; ++j)
                w[i][j] = (uint32_t)(c + (int32_t)j) >= cols ? 0.f : weight ? __ldg(weight + c + (int32_t)j) : 1.f;
        }
    }
}

// Bytes of y: V of them from column c on, where they are inside [0, cols), in one store where they lie on V bytes.
template <uint32_t V>
__device__ __forceinline__ void store_row_bytes(int8_t* q, float (&y)[V], const RowStep& st, int32_t c, uint32_t cols) {
    if (st.lift != 1.f) {  // a row of zeros, of tiny values, or not finite
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) y[i] = st.inv == 0.f ? 0.f : y[i] * st.lift;
    }
    if constexpr (V % 4 == 0) {
        if (inside(c, V, cols) && reinterpret_cast<uintptr_t>(q) % V == 0) {
            store_bytes<V>(q, y, st, V);
            return;
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < V; ++i)
        if ((uint32_t)(c + (int32_t)i) < cols)
            q[i] = (int8_t)__float_as_uint(__fadd_rn(__fmul_rn(y[i], st.inv), 12582912.f));
}

// ---- forward ---------------------------------------------------------------------------------

// What is done with row r once its pieces h are in registers (zeros outside the row), the thread's first from
// column c0 on, the others ROW * V apart. LONG: the row goes on behind them; that is read again in each step.
// Every element is read and written by one thread: outputs may lie over inputs.
// weight multiplies piece i by its columns' weights.
template <typename T, typename R, uint32_t V, uint32_t ROW, uint32_t KEEP, bool LONG, typename W, typename REDUCE>
__device__ __forceinline__ void norm_row(const NormParams& p, size_t r, int32_t c0, float (&h)[KEEP][V], W&& weight,
                                         REDUCE& reduce) {
    constexpr int32_t kStep = ROW * V;
    const int32_t rest = c0 + (int32_t)KEEP * kStep, end = LONG ? (int32_t)p.cols : rest;
    R* to_h = static_cast<R*>(p.h) + r * p.h_stride;
    T* to_y = static_cast<T*>(p.y) + r * p.y_stride;
    int8_t* to_q = p.q + r * p.q_stride;
    const auto again = [&](int32_t c, float (&f)[V]) {
        unpack(load_piece<V>(static_cast<const T*>(p.x) + r * p.x_stride + c, c, p.cols), f);
        if (!p.residual) return;
        float more[V];
        unpack(load_piece<V>(static_cast<const R*>(p.residual) + r * p.residual_stride + c, c, p.cols), more);
#pragma unroll
        for (uint32_t j = 0; j < V; ++j) f[j] += more[j];
    };
    const auto squares = [&](float lift) {
        float sum = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i)
#pragma unroll
            for (uint32_t j = 0; j < V; ++j) sum = fmaf(h[i][j] * lift, h[i][j] * lift, sum);
        for (int32_t c = rest; c < end; c += kStep) {
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
    const auto norm = [&](int32_t c, float (&f)[V]) {  // of the columns behind the pieces
        float more[1][V];
        row_weights<V, ROW, 1>(p.weight, c, p.cols, more);
#pragma unroll
        for (uint32_t j = 0; j < V; ++j) f[j] = f[j] * s * more[0][j];
    };
#pragma unroll
    for (uint32_t i = 0; i < KEEP; ++i) {
        const int32_t c = c0 + (int32_t)i * kStep;
        if (p.h) store_piece<V>(to_h + c, h[i], c, p.cols);
#pragma unroll
        for (uint32_t j = 0; j < V; ++j) h[i][j] *= s;
        weight(i, h[i]);
        if (p.y) store_piece<V>(to_y + c, h[i], c, p.cols);
    }
    RowStep st{};
    if (p.q) {
        uint32_t most = 0;
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i)  // outside the row 0, or NaN where the row is
#pragma unroll
            for (uint32_t j = 0; j < V; ++j) most = max(most, __float_as_uint(h[i][j]) & 0x7fffffffu);
        for (int32_t c = rest; c < end; c += kStep) {
            float f[V];
            again(c, f);
            norm(c, f);
#pragma unroll
            for (uint32_t j = 0; j < V; ++j) most = max(most, __float_as_uint(f[j]) & 0x7fffffffu);
        }
        st = row_step(reduce.most(most));
        if (threadIdx.x % ROW == 0) p.scale[r] = st.scale;
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i) {
            const int32_t c = c0 + (int32_t)i * kStep;
            store_row_bytes<V>(to_q + c, h[i], st, c, p.cols);
        }
    }
    for (int32_t c = rest; c < end; c += kStep) {
        float f[V];
        again(c, f);
        if (p.h) store_piece<V>(to_h + c, f, c, p.cols);
        norm(c, f);
        if (p.y) store_piece<V>(to_y + c, f, c, p.cols);
        if (p.q) store_row_bytes<V>(to_q + c, f, st, c, p.cols);
    }
}

// Few rows, rows whose operands lie at different offsets (V 1), rows longer than the pieces: a CTA a row, loads
// straight to registers.
template <typename T, typename R, uint32_t V, uint32_t ROW, uint32_t KEEP, bool LONG>
__global__ void __launch_bounds__(ROW) add_norm_kernel(const NormParams p) {
    constexpr uint32_t kStep = ROW * V;
    __shared__ float scratch[2][ROW / 32u];
    const int32_t c0 = threadIdx.x * V;
    float w[KEEP][V];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    RowReduce<ROW> reduce{scratch};
    for (size_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(p.x) + r * p.x_stride + c0;
        Pack<T, V> a[KEEP];  // all loads first
        Pack<R, V> b[KEEP];
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i) a[i] = load_piece<V>(x + i * kStep, c0 + (int32_t)(i * kStep), p.cols);
        if (p.residual) {
            const R* res = static_cast<const R*>(p.residual) + r * p.residual_stride + c0;
#pragma unroll
            for (uint32_t i = 0; i < KEEP; ++i) b[i] = load_piece<V>(res + i * kStep, c0 + (int32_t)(i * kStep), p.cols);
        }
        if (r == blockIdx.x) row_weights<V, ROW, KEEP>(p.weight, c0, p.cols, w);
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
        norm_row<T, R, V, ROW, KEEP, LONG>(p, r, c0, h, [&](uint32_t i, float (&f)[V]) {
#pragma unroll
            for (uint32_t j = 0; j < V; ++j) f[j] *= w[i][j];
        }, reduce);
    }
}

// Many rows: persistent CTAs, DEPTH - 1 rows ahead on their way to shared memory, since the registers that h and w
// take leave too few threads to hold enough loads in flight themselves. 16,384 x 4096 bf16, h and y written:
// a CTA a row from registers 126 us, rings 85 (6.3 TB/s). Rows of f32 past 8192 columns fill a ring (DEPTH 1) and none
// is ahead; it still reads each row once, which registers do not: 2048 x 12,288 f32 76 us for 90, 2048 x 16,384 95 for
// 131 (5.3 and 5.7 TB/s).
template <typename T, typename R, uint32_t ROW, uint32_t KEEP, uint32_t DEPTH, bool SHIFTED>
__global__ void __launch_bounds__(norm_threads(ROW), norm_ctas(ROW, KEEP * 16u / sizeof(R), SHIFTED)) add_norm_ring_kernel(const NormParams p) {
    constexpr uint32_t V = 16u / sizeof(R), kThreads = norm_threads(ROW), kRows = kThreads / ROW, kStep = ROW * V;
    constexpr uint32_t kX = KEEP * V * sizeof(T);
    extern __shared__ uint4 ring_smem[];
    __shared__ float scratch[kRows][2][ROW / 32u];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    RowReduce<ROW, kThreads> reduce{scratch[threadIdx.x / ROW]};
    RowRing<kThreads, kX + KEEP * 16u, DEPTH> ring{reinterpret_cast<char*>(ring_smem)};
    const size_t step = (size_t)gridDim.x * kRows, row0 = (size_t)blockIdx.x * kRows + threadIdx.x / ROW;
    const int32_t c0 = (int32_t)(threadIdx.x % ROW * V) - (int32_t)(row0 * p.x_stride % V);  // of every row: V divides step
    const T* x = static_cast<const T*>(p.x) + row0 * p.x_stride + c0;
    const R* res = static_cast<const R*>(p.residual) + row0 * p.residual_stride + c0;
    size_t ahead = row0;
    const auto ask = [&](uint32_t st) {
        if (ahead < p.rows) {
#pragma unroll
            for (uint32_t i = 0; i < KEEP; ++i) {
                const int32_t c = c0 + (int32_t)(i * kStep);
                ring.template ask<V>(st, 0, i, x + i * kStep, c, p.cols);
                if (p.residual) ring.template ask<V>(st, kX, i, res + i * kStep, c, p.cols);
            }
        }
        tc::cp_async_commit();
        ahead += step;
        x += step * p.x_stride;
        res += step * p.residual_stride;
    };
#pragma unroll
    for (uint32_t i = 0; i + 1u < DEPTH; ++i) ask(i);
    // SHIFTED, the weights do not lie on 16 bytes: they stay in registers. Else they are loaded again, from L1, and
    // the registers they would take hold a CTA more (16,384 x 4096 bf16: 99 us in registers, 86 from L1)
    float w[SHIFTED ? KEEP : 1u][V];
    if constexpr (SHIFTED) row_weights<V, ROW, KEEP>(p.weight, c0, p.cols, w);
    for (size_t r = row0; r < p.rows; r += step) {
        ask(ring.behind());
        ring.wait();
        float h[KEEP][V];
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i) {
            unpack(ring.template get<V, T>(0, i), h[i]);
            if (p.residual) {
                float more[V];
                unpack(ring.template get<V, R>(kX, i), more);
#pragma unroll
                for (uint32_t j = 0; j < V; ++j) h[i][j] += more[j];
            }
            if constexpr (SHIFTED) clip(h[i], c0 + (int32_t)(i * kStep), p.cols);
        }
        norm_row<T, R, V, ROW, KEEP, false>(p, r, c0, h, [&](uint32_t i, float (&f)[V]) {
            if constexpr (SHIFTED) {
#pragma unroll
                for (uint32_t j = 0; j < V; ++j) f[j] *= w[i][j];
            } else if (p.weight) {
                const int32_t c = c0 + (int32_t)(i * kStep);
                const Pack<float, V> v = load_piece<V>(p.weight + c, c, p.cols);
#pragma unroll
                for (uint32_t j = 0; j < V; ++j) f[j] *= v.v[j];
            }
        }, reduce);
        ring.next();
    }
    tc::cp_async_wait_all();
}

// ---- gradient --------------------------------------------------------------------------------

// Row r; adds dy n to acc. dy, h and dh give piece i (from registers, or again from shared memory: holding all
// three beside the weights and the sums would take more registers than there are).
template <typename T, typename R, uint32_t V, uint32_t ROW, uint32_t KEEP, bool SHIFTED, typename DY, typename H, typename DH, typename REDUCE>
__device__ __forceinline__ void norm_grad_row(const NormGradParams& p, size_t r, int32_t c0, DY&& dy, H&& h, DH&& dh,
                                              const float (&w)[KEEP][V], float (&acc)[KEEP][V], REDUCE& reduce, REDUCE& reduce2) {
    constexpr int32_t kStep = ROW * V;
    float sum, along;
    const auto sums = [&](float lift) {
        sum = along = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i) {
            float g[V], v[V];
            unpack(dy(i), g);
            unpack(h(i), v);
            if constexpr (SHIFTED) {
                clip(v, c0 + (int32_t)i * kStep, p.cols);
                clip(g, c0 + (int32_t)i * kStep, p.cols);
            }
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
        const int32_t c = c0 + (int32_t)i * kStep;
        float g[V], v[V], d[V];
        unpack(dy(i), g);
        unpack(h(i), v);
#pragma unroll
        for (uint32_t j = 0; j < V; ++j) {
            const float n = v[j] * s;
            d[j] = fmaf(-n, mean, g[j] * w[i][j]) * s;
            acc[i][j] = fmaf(g[j], n, acc[i][j]);  // outside the row: of columns that are not stored
        }
        if (p.dh) {
            unpack(dh(i), v);
#pragma unroll
            for (uint32_t j = 0; j < V; ++j) d[j] += v[j];
        }
        if (p.dx) store_piece<V>(static_cast<T*>(p.dx) + r * p.dx_stride + c, d, c, p.cols);
        if (p.dres) store_piece<V>(static_cast<R*>(p.dres) + r * p.dres_stride + c, d, c, p.cols);
    }
}

// The CTA's part of the weight's gradient: its rows' sums side by side in shared memory, added in order column by
// column (rows at different offsets have a column in different threads). all: for each row room for its columns and
// a 32nd, less than the ring holds of a row.
template <uint32_t V, uint32_t ROW, uint32_t KEEP, uint32_t THREADS>
__device__ __forceinline__ void norm_grad_part(const NormGradParams& p, int32_t c0, const float (&acc)[KEEP][V], float* all) {
    constexpr uint32_t kRows = THREADS / ROW, kStep = ROW * V;
    float* part = p.part + (size_t)blockIdx.x * p.cols;
    const auto place = [](uint32_t c) { return c + c / 32u; };  // lanes V columns apart on banks of their own
    const uint32_t pitch = place(p.cols) + 1u;
    if constexpr (kRows > 1u) __syncthreads();  // the ring is read
#pragma unroll
    for (uint32_t i = 0; i < KEEP; ++i)
#pragma unroll
        for (uint32_t j = 0; j < V; ++j) {
            const uint32_t c = (uint32_t)(c0 + (int32_t)(i * kStep + j));
            if (c >= p.cols) continue;
            if constexpr (kRows == 1u) part[c] = acc[i][j];
            else all[threadIdx.x / ROW * pitch + place(c)] = acc[i][j];
        }
    if constexpr (kRows > 1u) {
        __syncthreads();
        for (uint32_t c = threadIdx.x; c < p.cols; c += THREADS) {
            float v = all[place(c)];
#pragma unroll
            for (uint32_t k = 1; k < kRows; ++k) v += all[k * pitch + place(c)];
            part[c] = v;
        }
    }
}

// Few rows, rows whose operands lie at different offsets (V 1): a CTA takes every gridDim.x-th row and adds up
// dy n of its rows in registers; it leaves one part.
template <typename T, typename R, uint32_t V, uint32_t ROW, uint32_t KEEP>
__global__ void __launch_bounds__(ROW) norm_grad_kernel(const NormGradParams p) {
    constexpr uint32_t kStep = ROW * V;
    __shared__ float scratch[2][2][ROW / 32u];
    const int32_t c0 = threadIdx.x * V;
    float acc[KEEP][V] = {}, w[KEEP][V];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    RowReduce<ROW> reduce{scratch[0]}, reduce2{scratch[1]};
    for (size_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        Pack<T, V> dy[KEEP];
        Pack<R, V> h[KEEP], dh[KEEP];
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i) {
            const int32_t c = c0 + (int32_t)(i * kStep);
            dy[i] = load_piece<V>(static_cast<const T*>(p.dy) + r * p.dy_stride + c, c, p.cols);
            h[i] = load_piece<V>(static_cast<const R*>(p.h) + r * p.h_stride + c, c, p.cols);
            if (p.dh) dh[i] = load_piece<V>(static_cast<const R*>(p.dh) + r * p.dh_stride + c, c, p.cols);
        }
        if (r == blockIdx.x) row_weights<V, ROW, KEEP>(p.weight, c0, p.cols, w);
        norm_grad_row<T, R, V, ROW, KEEP, false>(
            p, r, c0, [&](uint32_t i) { return dy[i]; }, [&](uint32_t i) { return h[i]; }, [&](uint32_t i) { return dh[i]; }, w,
            acc, reduce, reduce2);
    }
    if (p.dw) norm_grad_part<V, ROW, KEEP, ROW>(p, c0, acc, nullptr);
}

// Many rows, as add_norm_ring_kernel (rows past 8192 columns with an f32 residual fill a ring too: 2048 x 16,384 f32 93 us,
// read again 220); a CTA an SM, so that few parts are left. 8192 x 4096 bf16 with dh and dw: from registers 156 us,
// rings 48 with the sum of the parts (5.6 TB/s).
template <typename T, typename R, uint32_t ROW, uint32_t KEEP, uint32_t DEPTH, bool SHIFTED>
__global__ void __launch_bounds__(kGradThreads, 1) norm_grad_ring_kernel(const NormGradParams p) {
    constexpr uint32_t V = 16u / sizeof(R), kThreads = kGradThreads, kRows = kThreads / ROW, kStep = ROW * V;
    constexpr uint32_t kH = KEEP * V * sizeof(T), kDh = kH + KEEP * 16u;
    extern __shared__ uint4 ring_smem[];
    __shared__ float scratch[2][kRows][2][ROW / 32u];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    RowReduce<ROW, kThreads> reduce{scratch[0][threadIdx.x / ROW]}, reduce2{scratch[1][threadIdx.x / ROW]};
    RowRing<kThreads, kDh + KEEP * 16u, DEPTH> ring{reinterpret_cast<char*>(ring_smem)};
    const size_t step = (size_t)gridDim.x * kRows, row0 = (size_t)blockIdx.x * kRows + threadIdx.x / ROW;
    const int32_t c0 = (int32_t)(threadIdx.x % ROW * V) - (int32_t)(row0 * p.dy_stride % V);  // of every row: V divides step
    const T* dy = static_cast<const T*>(p.dy) + row0 * p.dy_stride + c0;
    const R* h = static_cast<const R*>(p.h) + row0 * p.h_stride + c0;
    const R* dh = static_cast<const R*>(p.dh) + row0 * p.dh_stride + c0;
    size_t ahead = row0;
    const auto ask = [&](uint32_t st) {
        if (ahead < p.rows) {
#pragma unroll
            for (uint32_t i = 0; i < KEEP; ++i) {
                const int32_t c = c0 + (int32_t)(i * kStep);
                ring.template ask<V>(st, 0, i, dy + i * kStep, c, p.cols);
                ring.template ask<V>(st, kH, i, h + i * kStep, c, p.cols);
                if (p.dh) ring.template ask<V>(st, kDh, i, dh + i * kStep, c, p.cols);
            }
        }
        tc::cp_async_commit();
        ahead += step;
        dy += step * p.dy_stride;
        h += step * p.h_stride;
        dh += step * p.dh_stride;
    };
#pragma unroll
    for (uint32_t i = 0; i + 1u < DEPTH; ++i) ask(i);
    float acc[KEEP][V] = {}, w[KEEP][V];
    row_weights<V, ROW, KEEP>(p.weight, c0, p.cols, w);
    for (size_t r = row0; r < p.rows; r += step) {
        ask(ring.behind());
        ring.wait();
        norm_grad_row<T, R, V, ROW, KEEP, SHIFTED>(
            p, r, c0, [&](uint32_t i) { return ring.template get<V, T>(0, i); },
            [&](uint32_t i) { return ring.template get<V, R>(kH, i); },
            [&](uint32_t i) { return ring.template get<V, R>(kDh, i); }, w, acc, reduce, reduce2);
        ring.next();
    }
    tc::cp_async_wait_all();
    if (p.dw) norm_grad_part<V, ROW, KEEP, kThreads>(p, c0, acc, reinterpret_cast<float*>(ring_smem));
}

// Rows too long for registers, read again for dx and dresidual; with dw only a row's s and mean(g n), and the next
// kernel does the rest.
template <typename T, typename R, uint32_t ROW>
__global__ void __launch_bounds__(ROW) norm_grad_rows_kernel(const NormGradParams p) {
    __shared__ float scratch[2][2][ROW / 32u];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    RowReduce<ROW> reduce{scratch[0]}, reduce2{scratch[1]};
    for (size_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* dy = static_cast<const T*>(p.dy) + r * p.dy_stride;
        const R* h = static_cast<const R*>(p.h) + r * p.h_stride;
        float lift = 1.f, sum, along;
        const auto sums = [&] {
            sum = along = 0.f;
#pragma unroll 4
            for (uint32_t c = threadIdx.x; c < p.cols; c += ROW) {
                const float v = to_float(h[c]) * lift;
                sum = fmaf(v, v, sum);
                along = fmaf(to_float(dy[c]) * (p.weight ? p.weight[c] : 1.f), v, along);
            }
            reduce_two(reduce, reduce2, sum, along);
        };
        sums();
        if (!(sum < INFINITY)) {
            lift = kNormLift;
            sums();
        }
        const float step = norm_step(sum, p.share, p.eps, lift);
        const float s = step * lift, mean = along * step * p.share;
        if (p.dw) {
            if (threadIdx.x == 0) p.row[r] = make_float2(s, mean);
            continue;
        }
        const R* dh = p.dh ? static_cast<const R*>(p.dh) + r * p.dh_stride : nullptr;
#pragma unroll 4
        for (uint32_t c = threadIdx.x; c < p.cols; c += ROW) {
            const float d = fmaf(-to_float(h[c]) * s, mean, to_float(dy[c]) * (p.weight ? p.weight[c] : 1.f)) * s +
                            (dh ? to_float(dh[c]) : 0.f);
            if (p.dx) static_cast<T*>(p.dx)[r * p.dx_stride + c] = from_float<T>(d);
            if (p.dres) static_cast<R*>(p.dres)[r * p.dres_stride + c] = from_float<R>(d);
        }
    }
}

// A thread a column of the rows of part blockIdx.y.
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
        const float2 row = p.row[r];
        const float dy = to_float(static_cast<const T*>(p.dy)[r * p.dy_stride + c]);
        const float n = to_float(static_cast<const R*>(p.h)[r * p.h_stride + c]) * row.x;
        const float d = fmaf(-n, row.y, dy * w) * row.x +
                        (p.dh ? to_float(static_cast<const R*>(p.dh)[r * p.dh_stride + c]) : 0.f);
        if (p.dx) static_cast<T*>(p.dx)[r * p.dx_stride + c] = from_float<T>(d);
        if (p.dres) static_cast<R*>(p.dres)[r * p.dres_stride + c] = from_float<R>(d);
        acc = fmaf(dy, n, acc);
    }
    p.part[(size_t)blockIdx.y * p.cols + c] = acc;
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

// ---- hosts -----------------------------------------------------------------------------------

// Whether the operands' rows all lie at one offset from a boundary of V elements, `stride` giving it: every
// base on a boundary, every stride the same modulo V. A null operand has none.
struct Offsets {
    uint64_t stride;
    uint32_t v;
    bool fit;
    void add(const void* p, uint64_t s, size_t size) {
        if (p && (reinterpret_cast<uintptr_t>(p) % (v * size) || s % v != stride % v)) fit = false;
    }
    bool shifted() const { return stride % v != 0; }
};

// Persistent CTAs of `rows_each` rows: at most `most`, and rows at several offsets taken V at a time.
uint32_t ring_blocks(uint32_t most, uint32_t rows, uint32_t rows_each, uint32_t v, bool shifted) {
    const uint32_t need = (rows + rows_each - 1u) / rows_each, blocks = need < most ? need : most;
    const uint32_t whole = shifted && v > rows_each ? v / rows_each : 1u;
    return blocks / whole * whole;
}
template <typename K, typename P>
cudaError_t launch_ring(K* kernel, size_t smem, uint32_t threads, uint32_t blocks, cudaStream_t s, const P& p) {
    const cudaError_t e = smem_once(kernel, smem);
    if (e != cudaSuccess) return e;
    return launch_chained(kernel, dim3(blocks), threads, smem, 0, s, p);
}

template <uint32_t V_, uint32_t ROW_, uint32_t KEEP_>
struct Shape {
    static constexpr uint32_t V = V_, ROW = ROW_, KEEP = KEEP_;
};

// Rows from which rings are taken. Below, a CTA of more threads a row is over sooner (registers / ring: 32 x 2048 f32 1.9 /
// 2.2 us, gradient 3.8 / 5.5); at 64 that still holds for short rows (64 x 2048 f32 2.0 / 2.3, gradient 4.0 / 5.6; 64 x
// 4096 bf16 2.4 / 2.4, 7.0 / 7.1) and no longer for long ones (64 x 16,384 f32 8.9 / 7.5, 23.6 / 12.7; 64 x 8192 bf16
// 4.3 / 3.9, 11.9 / 8.3). From 512 rows on rings are ahead or within a tenth at every width from 256 to 16,384.
constexpr uint32_t kNormRingRows = 64, kGradRingRows = 64;

template <typename T, typename R>
cudaError_t norm_typed(const NormParams& p, cudaStream_t s) {
    constexpr uint32_t V = 16u / sizeof(R);
    const auto run = [&](auto shape) {
        using S = decltype(shape);
        const bool whole = p.cols <= S::V * S::ROW * S::KEEP;
        return launch_chained(whole ? add_norm_kernel<T, R, S::V, S::ROW, S::KEEP, false>
                                    : add_norm_kernel<T, R, S::V, S::ROW, S::KEEP, true>,
                              dim3(p.rows < 65535u ? p.rows : 65535u), S::ROW, 0, 0, s, p);
    };
    Offsets at{p.x_stride, V, true};
    at.add(p.x, p.x_stride, sizeof(T));
    at.add(p.residual, p.residual_stride, sizeof(R));
    at.add(p.h, p.h_stride, sizeof(R));
    at.add(p.y, p.y_stride, sizeof(T));
    const auto run_ring = [&](auto shape) {
        using S = decltype(shape);
        constexpr uint32_t kBytes = S::KEEP * V * (sizeof(T) + sizeof(R)), kThreads = norm_threads(S::ROW);
        const auto launch = [&](auto shifted) {
            constexpr bool kShifted = decltype(shifted)::value;
            constexpr uint32_t kCtas = norm_ctas(S::ROW, S::KEEP * V, kShifted), kDepth = ring_depth(kBytes, kThreads, kCtas);
            return launch_ring(add_norm_ring_kernel<T, R, S::ROW, S::KEEP, kDepth, kShifted>, kBytes * kDepth * kThreads,
                               kThreads, ring_blocks(kCtas * sm_count(), p.rows, kThreads / S::ROW, V, kShifted), s, p);
        };
        // int8 rows from 16-bit ones: with the second reduction the rows ahead count for more than a CTA (16,384 x
        // 4096 bf16 86 us with the weights from L1, 77 in registers; f32 142 and 157)
        const bool apart = at.shifted() || reinterpret_cast<uintptr_t>(p.weight) % 16u || (p.q && sizeof(R) == 2u);
        return apart ? launch(std::true_type{}) : launch(std::false_type{});
    };
    // pieces of a row, one more where it may begin inside one
    const uint32_t pieces = (p.cols + V - 1u) / V + (at.shifted() ? 1u : 0u);
    if (at.fit && p.rows >= kNormRingRows) {
        if (pieces <= 32u) return run_ring(Shape<V, 32, 1>{});
        if (pieces <= 64u) return run_ring(Shape<V, 32, 2>{});
        if (pieces <= 128u) return run_ring(Shape<V, 64, 2>{});
        if (pieces <= 256u) return run_ring(Shape<V, 128, 2>{});
        if (pieces <= 512u) return run_ring(Shape<V, 256, 2>{});
        if (pieces <= 1024u) return run_ring(Shape<V, 256, 4>{});
        if (pieces <= 2048u) return run_ring(Shape<V, 512, 4>{});
        if constexpr (V == 4u) {
            if (pieces <= 4096u) return run_ring(Shape<V, 512, 8>{});
        }
    }
    if (at.fit && !at.shifted()) {
        if (pieces <= 256u) return run(Shape<V, 256, 1>{});
        if (pieces <= 512u) return run(Shape<V, 512, 1>{});
        if (pieces <= 1024u) return run(Shape<V, 512, 2>{});
        return run(Shape<V, 512, 4>{});
    }
    if (p.cols <= 256u * 4u) return run(Shape<1, 256, 4>{});
    return run(Shape<1, 512, 8>{});
}

template <typename T, typename R>
cudaError_t grad_typed(const NormGradParams& p, cudaStream_t s) {
    constexpr uint32_t V = 16u / sizeof(R);
    const auto sum = [&](uint32_t parts) {
        return launch_chained(norm_grad_sum_kernel, dim3((p.cols + 31u) / 32u), 1024, 0, 0, s, p, parts);
    };
    const auto run = [&](auto shape) {
        using S = decltype(shape);
        const uint32_t blocks = p.rows < kNormParts ? p.rows : kNormParts;
        const cudaError_t e = launch_chained(norm_grad_kernel<T, R, S::V, S::ROW, S::KEEP>, dim3(blocks), S::ROW, 0, 0, s, p);
        return e != cudaSuccess || !p.dw ? e : sum(blocks);
    };
    Offsets at{p.dy_stride, V, true};
    at.add(p.dy, p.dy_stride, sizeof(T));
    at.add(p.h, p.h_stride, sizeof(R));
    at.add(p.dh, p.dh_stride, sizeof(R));
    at.add(p.dx, p.dx_stride, sizeof(T));
    at.add(p.dres, p.dres_stride, sizeof(R));
    const auto run_ring = [&](auto shape) {
        using S = decltype(shape);
        constexpr uint32_t kBytes = S::KEEP * V * (sizeof(T) + 2u * sizeof(R)), kDepth = ring_depth(kBytes, kGradThreads, 1);
        const uint32_t most = sm_count() < kNormParts ? sm_count() : kNormParts;  // a part each
        const uint32_t blocks = ring_blocks(most, p.rows, kGradThreads / S::ROW, V, at.shifted());
        const cudaError_t e = launch_ring(at.shifted() ? norm_grad_ring_kernel<T, R, S::ROW, S::KEEP, kDepth, true>
                                                       : norm_grad_ring_kernel<T, R, S::ROW, S::KEEP, kDepth, false>,
                                          kBytes * kDepth * kGradThreads, kGradThreads, blocks, s, p);
        return e != cudaSuccess || !p.dw ? e : sum(blocks);
    };
    const uint32_t pieces = (p.cols + V - 1u) / V + (at.shifted() ? 1u : 0u);
    if (at.fit && p.rows >= kGradRingRows) {
        if (pieces <= 32u) return run_ring(Shape<V, 32, 1>{});
        if (pieces <= 64u) return run_ring(Shape<V, 32, 2>{});
        // 16 elements a thread or more: what a row costs a thread besides is then less of it (65,536 x 512 f32, 8 a thread 90
        // us, 16 86)
        constexpr uint32_t kKeep = 16u / V;
        if (pieces <= 128u) return run_ring(Shape<V, 128 / kKeep, kKeep>{});
        if (pieces <= 256u) return run_ring(Shape<V, 256 / kKeep, kKeep>{});
        if (pieces <= 512u) return run_ring(Shape<V, 128, 4>{});
        if (pieces <= 1024u) return run_ring(Shape<V, 256, 4>{});
        if (pieces <= 2048u) return run_ring(Shape<V, 512, 4>{});
        if constexpr (V == 4u) {
            if (pieces <= 4096u) return run_ring(Shape<V, 512, 8>{});
        }
    }
    if (at.fit && !at.shifted()) {
        if (pieces <= 256u) return run(Shape<V, 256, 1>{});
        if (pieces <= 512u) return run(Shape<V, 256, 2>{});
        if (pieces <= 1024u) return run(Shape<V, 512, 2>{});
    } else {
        if (p.cols <= 256u * 4u) return run(Shape<1, 256, 4>{});
        if (p.cols <= 512u * 8u) return run(Shape<1, 512, 8>{});
    }
    cudaError_t e = launch_chained(norm_grad_rows_kernel<T, R, 512>, dim3(p.rows < 65535u ? p.rows : 65535u), 512, 0, 0, s, p);
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
