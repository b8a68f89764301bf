// Products on 8-bit integers with a scale for each token and each output channel.
//
//   quantize   row r of x (plain, gathered, or SwiGLU of two operands):
//                a = max_c |x_rc|,  s_r = a / 127,  q_rc = rint(x_rc * (127 / a))
//   linear     y_rn = (sum_k q_rk w_nk) * s_r * t_n, the sum exact in 32-bit integers
//              (cols <= 131,071: 128 * 128 * cols < 2^31), for one matrix or grouped: row r uses
//              the matrix of the group whose range [offsets[g], offsets[g + 1]) holds it;
//              with an epilogue y_rn = rw_r act(y_rn + b_n) + residual_rn, act also SwiGLU of channel pairs.
//
// The reference has no 8-bit integer path; the row scheme follows from the formulas above.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <mutex>
#include <type_traits>

#include "vlb_launch.h"
#include "vlb_math.cuh"
#include "vlb_rows.cuh"
#include "vlb_tcgen05.cuh"

namespace vlb {
namespace {

// silu(g) * u with the clamp of the layer's experts (gate from above, up on both sides). The
// comparisons keep a NaN, which fminf / fmaxf would drop. The exponential takes the gate inside
// [-88, 1000]: beyond, its reciprocal is 0 (silu's true value is under 1e-35) and 1.
__device__ __forceinline__ float swiglu(float g, float u, float limit) {
    if (limit > 0.f) {
        g = g > limit ? limit : g;
        u = u > limit ? limit : (u < -limit ? -limit : u);
    }
    return g * fast_rcp(1.f + fast_exp(fmaxf(fminf(-g, 88.f), -1000.f))) * u;
}

// ---- the products' epilogue ------------------------------------------------------------------
//
// z = sum * x_scale * w_scale + bias, y = row_weight * act(z) + residual, the same operations in the same
// order in every form of the product.

// Added where there is no residual: it leaves every value as it is, a -0 too, as the tiles' plain product does.
constexpr float kNoResidual = -0.f;

template <bool EPI>
using LinearParams = std::conditional_t<EPI, Int8ActParams, Int8LinearParams>;

__device__ __forceinline__ float epi_sum(int32_t sum, float x_scale, float w_scale, float bias) {
    return fmaf((float)sum * x_scale, w_scale, bias);
}

// z Phi(z) with erfc by Abramowitz and Stegun's 7.1.26 (|error| <= 1.5e-7): erfc(x) = (a1 t + .. + a5 t^5)
// e^(-x^2), t = 1 / (1 + p x), x = |z| / sqrt(2) >= 0. In 32 bits the polynomial adds up to 10 units of 2^-24
// (its terms' magnitudes sum to 4.5): z Phi(z) within 2^-20 |z|. CUDA's erfcf takes five times the
// instructions, which a tile's epilogue does not have.
__device__ __forceinline__ float gelu(float z) {
    const float x = fabsf(z) * 0.707106781f;
    const float t = fast_rcp(fmaf(0.3275911f, x, 1.f));
    float c = fmaf(t, 1.061405429f, -1.453152027f);
    c = fmaf(t, c, 1.421413741f);
    c = fmaf(t, c, -0.284496736f);
    c = fmaf(t, c, 0.254829592f);
    const float tail = 0.5f * (c * t) * fast_exp(fmaxf(-x * x, -1000.f));  // Phi(-|z|)
    return z * (z > 0.f ? 1.f - tail : tail);
}

// sigmoid(v): of SiLU, and of GELU's tanh form, (1 + tanh(u)) / 2 = sigmoid(2 u).
__device__ __forceinline__ float sigmoid_of(float v) { return fast_rcp(1.f + fast_exp(fmaxf(fminf(-v, 88.f), -1000.f))); }

template <int ACT>
__device__ __forceinline__ float activate(float z) {
    if constexpr (ACT == VLB_ACT_RELU) return z < 0.f ? 0.f : z;  // keeps a NaN
    else if constexpr (ACT == VLB_ACT_SILU) return z * sigmoid_of(z);
    else if constexpr (ACT == VLB_ACT_GELU) return gelu(z);
    else if constexpr (ACT == VLB_ACT_GELU_TANH)
        return z * sigmoid_of(1.59576912f * fmaf(0.044715f * z * z, z, z));  // 2 sqrt(2 / pi)
    else return z;
}
__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case VLB_ACT_RELU: return activate<VLB_ACT_RELU>(z);
        case VLB_ACT_SILU: return activate<VLB_ACT_SILU>(z);
        case VLB_ACT_GELU: return activate<VLB_ACT_GELU>(z);
        case VLB_ACT_GELU_TANH: return activate<VLB_ACT_GELU_TANH>(z);
        default: return z;
    }
}

// ---- row quantizer ---------------------------------------------------------------------------

template <typename T, bool SWIGLU>
__device__ __forceinline__ float row_value(const Int8QuantParams& p, size_t at) {
    const float x = to_float(static_cast<const T*>(p.x)[at]);
    if (!SWIGLU) return x;
    return swiglu(x, to_float(static_cast<const T*>(p.up)[at]), p.limit);
}

// Rows at any alignment: neighbouring lanes take neighbouring elements, a thread up to KEEP of them in
// registers between the row's maximum and its rounding (the rest is read twice); bytes are written
// one a lane. ROW: threads of a row (32 or the CTA's 256).
template <typename T, bool SWIGLU, uint32_t ROW, uint32_t KEEP>
__global__ void __launch_bounds__(256) int8_quantize_kernel(const Int8QuantParams p) {
    __shared__ uint32_t top[8];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    const uint32_t tid = threadIdx.x % ROW;
    for (size_t r = (size_t)blockIdx.x * (256u / ROW) + threadIdx.x / ROW; r < p.rows;
         r += (size_t)gridDim.x * (256u / ROW)) {
        const uint64_t src = p.row_index ? p.row_index[r] : r;
        const uint32_t have = src < p.x_rows ? p.cols : 0u;
        const size_t base = src * p.x_stride;
        const T* x = static_cast<const T*>(p.x) + base + tid;
        const T* up = SWIGLU ? static_cast<const T*>(p.up) + base + tid : nullptr;
        float v[KEEP];
        uint32_t m = 0;
        {
            T a[KEEP], b[SWIGLU ? KEEP : 1];  // all loads first
#pragma unroll
            for (uint32_t i = 0; i < KEEP; ++i) {
                a[i] = from_float<T>(0.f);
                if (tid + i * ROW < have) a[i] = x[i * ROW];
                if constexpr (SWIGLU) {
                    b[i] = from_float<T>(0.f);
                    if (tid + i * ROW < have) b[i] = up[i * ROW];
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < KEEP; ++i) {
                v[i] = to_float(a[i]);
                if constexpr (SWIGLU) v[i] = swiglu(v[i], to_float(b[i]), p.limit);
                m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
            }
        }
#pragma unroll 4
        for (uint32_t c = tid + KEEP * ROW; c < have; c += ROW)
            m = max(m, __float_as_uint(row_value<T, SWIGLU>(p, base + c)) & 0x7fffffffu);
        m = __reduce_max_sync(0xffffffffu, m);
        if constexpr (ROW == 256) {
            __syncthreads();
            if ((tid & 31u) == 0) top[tid >> 5] = m;
            __syncthreads();
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) m = max(m, top[i]);
        }
        const RowStep st = row_step(m);
        if (tid == 0) p.scale[r] = st.scale;
        int8_t* q = p.q + r * p.q_stride;
        if (st.lift != 1.f) {  // a row of zeros, of tiny values, or not finite
#pragma unroll
            for (uint32_t i = 0; i < KEEP; ++i) v[i] = st.inv == 0.f ? 0.f : v[i] * st.lift;
        }
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i)
            if (tid + i * ROW < p.fill_cols)
                q[tid + i * ROW] = (int8_t)__float_as_uint(__fadd_rn(__fmul_rn(v[i], st.inv), 12582912.f));
#pragma unroll 4
        for (uint32_t c = tid + KEEP * ROW; c < p.fill_cols; c += ROW)
            q[c] = (int8_t)(c < have ? quant_byte(row_value<T, SWIGLU>(p, base + c), st) : 0u);
    }
}

// ---- row quantizer, rows on 16-byte boundaries ---------------------------------------------------
//
// HBM-bound: every element is read once (16 bytes a load) and kept in registers between the row's
// maximum and its rounding; rows longer than the registers hold are read twice, the second time
// mostly from L2. A warp takes a row of up to 16 loads a lane (8 rows a CTA: no barrier, all loads
// in flight at once, and what a row costs beside its elements paid by one warp); longer rows, and calls of too few rows to fill the GPU with warps, take a
// CTA a row.

template <typename T>
struct RowVec {
    static constexpr uint32_t kN = 16u / sizeof(T);
    uint4 raw;
    __device__ __forceinline__ void load(const T* p) { raw = __ldg(reinterpret_cast<const uint4*>(p)); }
    __device__ __forceinline__ void clear() { raw = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ float get(uint32_t i) const {
        const uint32_t w = (&raw.x)[i * sizeof(T) / 4u];
        if constexpr (sizeof(T) == 4) return __uint_as_float(w);
        else if constexpr (std::is_same<T, __half>::value)
            return __half2float(__ushort_as_half((unsigned short)(i & 1u ? w >> 16 : w & 0xffffu)));
        else
            return __uint_as_float(i & 1u ? w & 0xffff0000u : w << 16);
    }
    // the last vector of a row that ends inside it
    __device__ __forceinline__ void load_part(const T* p, uint32_t n) {
        clear();
#pragma unroll
        for (uint32_t i = 0; i < kN; ++i)
            if (i < n) {
                if constexpr (sizeof(T) == 4) (&raw.x)[i] = __float_as_uint(p[i]);
                else {
                    const uint32_t v = reinterpret_cast<const unsigned short*>(p)[i];
                    (&raw.x)[i / 2u] |= i & 1u ? v << 16 : v;
                }
            }
    }
};

// Largest |x| of vectors, as float bits, a NaN above all. 16-bit types compare two magnitudes an
// instruction.
template <typename T>
struct RowMax {
    uint32_t m = 0;
    __device__ __forceinline__ void add(const RowVec<T>& v) {
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            const uint32_t w = (&v.raw.x)[i];
            if constexpr (sizeof(T) == 4) {
                m = max(m, w & 0x7fffffffu);
            } else {
                const uint32_t a = w & 0x7fff7fffu;
                if constexpr (std::is_same<T, __half>::value)
                    asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(m) : "r"(a));
                else
                    asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(a));
            }
        }
    }
    __device__ __forceinline__ uint32_t bits() const {
        if constexpr (sizeof(T) == 4) return m;
        const uint32_t top = max(m & 0xffffu, m >> 16);
        if constexpr (std::is_same<T, __half>::value)
            return __float_as_uint(__half2float(__ushort_as_half((unsigned short)top)));
        return top << 16;
    }
};

// ROW: threads of a row (32 or the CTA's 256); KEEP: vectors a thread keeps.
template <typename T, bool SWIGLU, uint32_t ROW, uint32_t KEEP>
__global__ void __launch_bounds__(256, KEEP > (SWIGLU ? 4 : 8) ? 2 : SWIGLU || KEEP > 4 ? 3 : 5) int8_quantize_vec_kernel(const Int8QuantParams p) {
    constexpr uint32_t N = RowVec<T>::kN;
    __shared__ uint32_t top[8];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    const uint32_t tid = threadIdx.x % ROW;
    const uint32_t vecs = (p.cols + N - 1u) / N, all = (p.fill_cols + N - 1u) / N;  // of x; of q
    for (size_t r = (size_t)blockIdx.x * (256u / ROW) + threadIdx.x / ROW; r < p.rows;
         r += (size_t)gridDim.x * (256u / ROW)) {
        const uint64_t src = p.row_index ? p.row_index[r] : r;
        const uint32_t have = src < p.x_rows ? vecs : 0u;
        const T* x = static_cast<const T*>(p.x) + src * p.x_stride;
        const T* up = SWIGLU ? static_cast<const T*>(p.up) + src * p.x_stride : nullptr;
        auto fetch = [&](const T* row, uint32_t v) {
            RowVec<T> a;
            if (v >= have) a.clear();
            else if ((v + 1u) * N <= p.cols) a.load(row + (size_t)v * N);
            else a.load_part(row + (size_t)v * N, p.cols - v * N);
            return a;
        };
        RowVec<T> a[SWIGLU ? 1 : KEEP];
        float f[SWIGLU ? KEEP : 1][N];
        uint32_t m = 0;
        if constexpr (SWIGLU) {
            constexpr uint32_t kAtOnce = KEEP < 4u ? KEEP : 4u;  // loads of both operands in flight
#pragma unroll
            for (uint32_t i0 = 0; i0 < KEEP; i0 += kAtOnce) {
                RowVec<T> a[kAtOnce], b[kAtOnce];
#pragma unroll
                for (uint32_t i = 0; i < kAtOnce; ++i) {
                    a[i] = fetch(x, tid + (i0 + i) * ROW);
                    b[i] = fetch(up, tid + (i0 + i) * ROW);
                }
#pragma unroll
                for (uint32_t i = 0; i < kAtOnce; ++i)
#pragma unroll
                    for (uint32_t j = 0; j < N; ++j) {
                        f[i0 + i][j] = swiglu(a[i].get(j), b[i].get(j), p.limit);
                        m = max(m, __float_as_uint(f[i0 + i][j]) & 0x7fffffffu);
                    }
            }
            for (uint32_t v = tid + KEEP * ROW; v < have; v += ROW) {
                const RowVec<T> c = fetch(x, v), d = fetch(up, v);
#pragma unroll
                for (uint32_t j = 0; j < N; ++j)
                    m = max(m, __float_as_uint(swiglu(c.get(j), d.get(j), p.limit)) & 0x7fffffffu);
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < KEEP; ++i) a[i] = fetch(x, tid + i * ROW);
            RowMax<T> t;
#pragma unroll
            for (uint32_t i = 0; i < KEEP; ++i) t.add(a[i]);
            for (uint32_t v = tid + KEEP * ROW; v < have; v += ROW) t.add(fetch(x, v));
            m = t.bits();
        }
        m = __reduce_max_sync(0xffffffffu, m);
        if constexpr (ROW == 256) {
            __syncthreads();
            if ((tid & 31u) == 0) top[tid >> 5] = m;
            __syncthreads();
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) m = max(m, top[i]);
        }
        const RowStep st = row_step(m);
        if (tid == 0) p.scale[r] = st.scale;
        int8_t* q = p.q + r * p.q_stride;
        auto put = [&](uint32_t v, float (&y)[N]) {
            if (st.lift != 1.f) {  // a row of zeros, of tiny values, or not finite
#pragma unroll
                for (uint32_t j = 0; j < N; ++j) y[j] = st.inv == 0.f ? 0.f : y[j] * st.lift;
            }
            store_bytes<N>(q + (size_t)v * N, y, st, min(N, p.fill_cols - v * N));
        };
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i) {
            const uint32_t v = tid + i * ROW;
            if (v < all) {
                float y[N];
#pragma unroll
                for (uint32_t j = 0; j < N; ++j) {
                    if constexpr (SWIGLU) y[j] = f[i][j];
                    else y[j] = a[i].get(j);
                }
                put(v, y);
            }
        }
        for (uint32_t v = tid + KEEP * ROW; v < all; v += ROW) {
            const RowVec<T> c = fetch(x, v);
            RowVec<T> d = c;
            if constexpr (SWIGLU) d = fetch(up, v);
            float y[N];
#pragma unroll
            for (uint32_t j = 0; j < N; ++j) y[j] = SWIGLU ? swiglu(c.get(j), d.get(j), p.limit) : c.get(j);
            put(v, y);
        }
    }
}

// Quantized rows by index: a warp a row, 16 bytes a lane.
__global__ void __launch_bounds__(256) int8_gather_kernel(const Int8GatherParams p) {
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    const uint32_t lane = threadIdx.x & 31u, vecs = (uint32_t)(p.pitch / 16u);
    for (size_t r = (size_t)blockIdx.x * 8u + (threadIdx.x >> 5); r < p.rows; r += (size_t)gridDim.x * 8u) {
        const uint32_t src = p.row_index[r];
        const bool have = src < p.x_rows;
        const uint4* from = reinterpret_cast<const uint4*>(p.x + (size_t)(have ? src : 0u) * p.pitch);
        uint4* to = reinterpret_cast<uint4*>(p.q + r * p.pitch);
        if (lane == 0) p.scale[r] = have ? p.x_scale[src] : 0.f;
        for (uint32_t v0 = lane; v0 < vecs; v0 += 128u) {
            uint4 a[4];
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i)
                a[i] = have && v0 + 32u * i < vecs ? from[v0 + 32u * i] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i)
                if (v0 + 32u * i < vecs) to[v0 + 32u * i] = a[i];
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

template <typename TY, bool EPI>
__global__ void __launch_bounds__(256) int8_linear_kernel(const LinearParams<EPI> p) {
    __shared__ uint32_t xs[kGenTile][kGenK / 4 + 1], ws[kGenTile][kGenK / 4 + 1];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
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
                if constexpr (EPI) {
                    const bool pairs = p.act == VLB_ACT_SWIGLU, have = r < hi;
                    const float s = have ? p.x_scale[r] : 0.f, rw = have && p.row_weight ? p.row_weight[r] : 1.f;
#pragma unroll
                    for (uint32_t j = 0; j < 4u; ++j) {
                        const uint32_t n = n0 + tc + 16u * j;
                        const size_t at = (size_t)g * p.out_cols + n;
                        const bool in = n < p.out_cols;
                        const float z = epi_sum(acc[i][j], s, in ? p.w_scale[at] : 0.f, in && p.bias ? p.bias[at] : 0.f);
                        const float up = __shfl_xor_sync(0xffffffffu, z, 1);  // of a pair's gate: channel n + 1
                        if (!have || !in || (pairs && (n & 1u))) continue;
                        const uint32_t c = pairs ? n / 2u : n;
                        const float a = pairs ? swiglu(z, up, p.act_limit) : activate(z, p.act);
                        const float res = p.residual
                                              ? to_float(static_cast<const TY*>(p.residual)[(size_t)r * p.residual_stride + c])
                                              : kNoResidual;
                        static_cast<TY*>(p.y)[(size_t)r * p.y_stride + c] = from_float<TY>(fmaf(rw, a, res));
                    }
                    continue;
                }
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

// ---- product of few rows ------------------------------------------------------------------------
//
// One launch from the float rows on: for a handful of rows a call is as long as its launches and the
// latency of its loads, and the weights are its bytes. A block quantizes the rows into shared memory
// while its warps' first weights are on their way; then a warp takes two channels at a time, a lane
// 16 bytes of each every 512, two or four such pieces of both in flight, dp4a against the rows. A call with
// groups (GROUPED) takes one row a block and that row's matrix (two rows of one group read it twice, from L2).

constexpr uint32_t kFewThreads = 256, kFewWarps = kFewThreads / 32u;
// Pieces of a channel in flight, and blocks an SM. A group's row has registers for twice the blocks, whose set-up then
// overlaps (16 rows of 64 experts' 2048 x 2048: 4 pieces and 2 blocks 19.2 us, 2 and 4 14.8); one row of one matrix fills
// no more than two an SM (int8 rows, 2 pieces and 4 blocks / 4 and 2: 512 x 512 2.0 / 1.9 us, 2048 x 2048 3.4 / 2.9, 4096 x
// 4096 6.0 / 5.2, 8192 x 8192 13.8 / 13.8). 128 registers are short of 4 and 8 rows with an epilogue: 56 to 92 bytes
// a thread spill.
__host__ __device__ constexpr uint32_t few_pieces(bool grouped) { return grouped ? 2u : 4u; }
__host__ __device__ constexpr uint32_t few_blocks(bool grouped) { return grouped ? 4u : 2u; }
constexpr uint32_t kFewSmem = 64u * 1024u;
// Dynamic shared memory a launch may ask for without an opt-in: the default 48 KB hold the kernel's
// static arrays too (up to 1 KB as the compiler lays them out).
constexpr uint32_t kFewDefaultSmem = 47u * 1024u;

// 16 bytes of a weight row from byte k on, zeros past K.
__device__ __forceinline__ uint4 few_load(const int8_t* row, uint32_t k, uint32_t cols) {
    if (k + 16u <= cols) return __ldg(reinterpret_cast<const uint4*>(row + k));
    if (k >= cols) return make_uint4(0u, 0u, 0u, 0u);
    return make_uint4(load_word(row, k, cols), load_word(row, k + 4u, cols), load_word(row, k + 8u, cols),
                      load_word(row, k + 12u, cols));
}

__device__ __forceinline__ float load_typed(const void* y, size_t at, int type) {
    if (type == VLB_DTYPE_F32) return static_cast<const float*>(y)[at];
    if (type == VLB_DTYPE_F16) return __half2float(static_cast<const __half*>(y)[at]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(y)[at]);
}
__device__ __forceinline__ void store_typed(void* y, size_t at, float v, int type) {
    if (type == VLB_DTYPE_F32) static_cast<float*>(y)[at] = v;
    else if (type == VLB_DTYPE_F16) static_cast<__half*>(y)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(y)[at] = __float2bfloat16_rn(v);
}

// T: the rows' type, int8_t for rows that are integers already. ROWS: rows of a block.
template <typename T, uint32_t ROWS, bool EPI, bool GROUPED>
__global__ void __launch_bounds__(kFewThreads, few_blocks(GROUPED)) int8_few_kernel(const LinearParams<EPI> l, const Int8QuantParams q, int y_type,
                                                               uint32_t channels) {
    constexpr uint32_t kFewPieces = few_pieces(GROUPED);
    extern __shared__ __align__(16) unsigned char few_smem[];
    __shared__ uint32_t top[ROWS], group_s;
    __shared__ float scale[ROWS];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t pitch = (l.cols + 15u) / 16u * 16u;
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    uint32_t row0 = 0, rows = l.rows, g = 0;
    if constexpr (GROUPED) {
        row0 = blockIdx.y;
        rows = 1;
        if (tid == 0) group_s = l.groups;
        __syncthreads();
        for (uint32_t i = tid; i < l.groups; i += kFewThreads) {
            uint32_t lo, hi;
            group_range(l, i, lo, hi);
            if (row0 >= lo && row0 < hi) atomicMin(&group_s, i);
        }
        __syncthreads();
        g = group_s;
        if (g == l.groups) return;
    }
    const uint32_t n_end = min(l.out_cols, (blockIdx.x + 1u) * channels);
    const int8_t* w = l.w + (size_t)g * l.out_cols * l.w_stride;
    uint32_t n = blockIdx.x * channels + 2u * warp;
    uint4 a[kFewPieces], b[kFewPieces];
    const auto fetch = [&](uint32_t n, uint32_t k0) {
        const int8_t *wa = w + (size_t)n * l.w_stride, *wb = w + (size_t)min(n + 1u, l.out_cols - 1u) * l.w_stride;
#pragma unroll
        for (uint32_t i = 0; i < kFewPieces; ++i) {
            // no piece behind the row (of the whole block; none is multiplied below): one row of 512 x 512 int8 2.14 -> 1.89
            // us. Two pieces in 64 registers would spill for it (24 rows of 64 groups 30.3 -> 34.6)
            if (!GROUPED && k0 + 512u * i >= l.cols) break;
            a[i] = few_load(wa, k0 + 512u * i + 16u * lane, l.cols);
            b[i] = few_load(wb, k0 + 512u * i + 16u * lane, l.cols);
        }
    };
    if (n < n_end) fetch(n, 0);
    // with an epilogue the channels' scales and biases come beside their weights too (lane j those of channel n + j / ROWS,
    // of a SwiGLU pair both), not after the sums
    [[maybe_unused]] float ws[2] = {}, bs[2] = {};
    [[maybe_unused]] const auto fetch_scales = [&](uint32_t n) {
        if constexpr (EPI) {
            const bool pairs = l.act == VLB_ACT_SWIGLU;
            const uint32_t c = n + (pairs ? 0u : lane / ROWS);
            const size_t at = (size_t)g * l.out_cols + c;
#pragma unroll
            for (uint32_t i = 0; i < 2u; ++i) {
                if (lane >= 2u * ROWS || c + i >= l.out_cols || (i && !pairs)) continue;
                ws[i] = l.w_scale[at + i];
                if (l.bias) bs[i] = l.bias[at + i];
            }
        }
    };
    if (EPI && n < n_end) fetch_scales(n);
    // the rows: warps share them out, each row's warps its columns
    if (tid < ROWS) top[tid] = 0;
    __syncthreads();
    const uint32_t row_warps = kFewWarps / ROWS, m = warp / row_warps, part = (warp % row_warps) * 32u + lane;
    const uint32_t r = row0 + m;
    int8_t* xs = reinterpret_cast<int8_t*>(few_smem);
    if constexpr (std::is_same<T, int8_t>::value) {
        if (m < rows && part == 0) scale[m] = !EPI && l.row_weight ? l.x_scale[r] * l.row_weight[r] : l.x_scale[r];
        for (uint32_t c = part * 16u; c < pitch; c += row_warps * 512u)
            *reinterpret_cast<uint4*>(xs + m * pitch + c) =
                m < rows ? few_load(l.x + (size_t)r * l.x_stride, c, l.cols) : make_uint4(0u, 0u, 0u, 0u);
    } else {
        const uint64_t src = m < rows ? q.row_index ? q.row_index[r] : r : ~0ull;
        const bool have = src < q.x_rows;
        const size_t base = have ? src * q.x_stride : 0;
        const auto value = [&](uint32_t c) {
            return q.up ? row_value<T, true>(q, base + c) : row_value<T, false>(q, base + c);
        };
        // a lane's first kFewKeep elements stay in registers between the row's maximum and its rounding, four at a time
        // as far as the row goes (all sixteen for a row of 512 took a lone one 2.7 -> 2.8 us, of SwiGLU 3.0 -> 3.5)
        constexpr uint32_t kFewKeep = 16;
        float kept[kFewKeep];
        const uint32_t step = row_warps * 32u;
        const auto each = [&](auto&& f) {
#pragma unroll
            for (uint32_t i0 = 0; i0 < kFewKeep; i0 += 4u) {
                if (i0 * step >= pitch) break;
#pragma unroll
                for (uint32_t i = i0; i < i0 + 4u; ++i) f(i);
            }
        };
        uint32_t most = 0;
        {
            T a[kFewKeep], b[kFewKeep];  // all loads first
            const auto load = [&](const void* from, uint32_t i) {
                const uint32_t c = part + i * step;
                return have && c < l.cols ? static_cast<const T*>(from)[base + c] : from_float<T>(0.f);
            };
            each([&](uint32_t i) { a[i] = load(q.x, i); });
            if (q.up) {
                each([&](uint32_t i) { b[i] = load(q.up, i); });
                each([&](uint32_t i) { kept[i] = swiglu(to_float(a[i]), to_float(b[i]), q.limit); });
            } else {
                each([&](uint32_t i) { kept[i] = to_float(a[i]); });
            }
        }
        each([&](uint32_t i) { most = max(most, __float_as_uint(kept[i]) & 0x7fffffffu); });
        if (have)
#pragma unroll 8
            for (uint32_t c = part + kFewKeep * step; c < l.cols; c += step)
                most = max(most, __float_as_uint(value(c)) & 0x7fffffffu);
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) atomicMax(top + m, most);
        __syncthreads();
        const RowStep st = row_step(top[m]);
        if (m < rows && part == 0) scale[m] = !EPI && l.row_weight ? st.scale * l.row_weight[r] : st.scale;
        each([&](uint32_t i) {
            if (part + i * step < pitch) xs[m * pitch + part + i * step] = (int8_t)quant_byte(kept[i], st);
        });
#pragma unroll 8
        for (uint32_t c = part + kFewKeep * step; c < pitch; c += step)
            xs[m * pitch + c] = (int8_t)(have && c < l.cols ? quant_byte(value(c), st) : 0u);
    }
    __syncthreads();
    for (; n < n_end; n += 2u * kFewWarps) {
        int32_t sum[2][ROWS] = {};
        for (uint32_t k0 = 0; k0 < l.cols; k0 += 512u * kFewPieces) {
            uint4 va[kFewPieces], vb[kFewPieces];
#pragma unroll
            for (uint32_t i = 0; i < kFewPieces; ++i) va[i] = a[i], vb[i] = b[i];
            // the next pieces, of these channels or the next two
            if (k0 + 512u * kFewPieces < l.cols) fetch(n, k0 + 512u * kFewPieces);
            else if (n + 2u * kFewWarps < n_end) fetch(n + 2u * kFewWarps, 0);
#pragma unroll
            for (uint32_t i = 0; i < kFewPieces; ++i) {
                const uint32_t k = k0 + 512u * i + 16u * lane;
                if (k >= pitch) break;
#pragma unroll
                for (uint32_t j = 0; j < ROWS; ++j) {
                    const uint4 x = *reinterpret_cast<const uint4*>(xs + j * pitch + k);
                    sum[0][j] = __dp4a((int)va[i].x, (int)x.x, sum[0][j]);
                    sum[1][j] = __dp4a((int)vb[i].x, (int)x.x, sum[1][j]);
                    sum[0][j] = __dp4a((int)va[i].y, (int)x.y, sum[0][j]);
                    sum[1][j] = __dp4a((int)vb[i].y, (int)x.y, sum[1][j]);
                    sum[0][j] = __dp4a((int)va[i].z, (int)x.z, sum[0][j]);
                    sum[1][j] = __dp4a((int)vb[i].z, (int)x.z, sum[1][j]);
                    sum[0][j] = __dp4a((int)va[i].w, (int)x.w, sum[0][j]);
                    sum[1][j] = __dp4a((int)vb[i].w, (int)x.w, sum[1][j]);
                }
            }
        }
        // lane c * ROWS + j stores row j of channel c; of a SwiGLU pair, lane j
        int32_t mine = 0, second = 0;
#pragma unroll
        for (uint32_t c = 0; c < 2u; ++c)
#pragma unroll
            for (uint32_t j = 0; j < ROWS; ++j) {
                const int32_t v = __reduce_add_sync(0xffffffffu, sum[c][j]);
                if (lane == c * ROWS + j) mine = v;
                if (EPI && c == 1u && lane == j) second = v;
            }
        const uint32_t c = n + lane / ROWS, j = lane % ROWS;
        if constexpr (EPI) {
            const bool pairs = l.act == VLB_ACT_SWIGLU;
            if (lane < (pairs ? 1u : 2u) * ROWS && j < rows && c < n_end) {
                const size_t r = row0 + j;
                float a = epi_sum(mine, scale[j], ws[0], bs[0]);
                if (pairs)
                    a = swiglu(a, epi_sum(second, scale[j], ws[1], bs[1]), l.act_limit);
                else
                    a = activate(a, l.act);
                const uint32_t to = pairs ? c / 2u : c;
                const float res = l.residual ? load_typed(l.residual, r * l.residual_stride + to, y_type) : kNoResidual;
                store_typed(l.y, r * l.y_stride + to, fmaf(l.row_weight ? l.row_weight[r] : 1.f, a, res), y_type);
            }
            if (n + 2u * kFewWarps < n_end) fetch_scales(n + 2u * kFewWarps);
            continue;
        }
        if (lane < 2u * ROWS && j < rows && c < n_end)
            store_typed(l.y, (size_t)(row0 + j) * l.y_stride + c,
                        (float)mine * scale[j] * l.w_scale[(size_t)g * l.out_cols + c], y_type);
    }
}

// ---- product on the tensor cores ---------------------------------------------------------------
//
// D[channel][token] = W X^T by tcgen05.mma kind::i8: a tile is 128 channels (the TMEM lanes) by up
// to 256 tokens of one group (the columns), so a lane of the epilogue holds one channel's scale and
// a warp's stores are 32 neighbouring channels of one token; few tokens cost few columns.
// K runs in chunks of 128 bytes (one 128-byte swizzle row) through a ring of TMA stages.
// Roles: warps 0-7 (with an epilogue 12 or 16 of them) the sums to memory, the next three TMA, MMA, and the tiles' places and scales for the
// epilogue, a tile or two ahead (behind an epilogue's stores their lookup took 3,000 to 5,000 cycles
// of a tile's 8,000); two accumulators, so a tile's epilogue runs beside the next tile's products.
// Persistent CTAs, tiles in order, a group's token tiles innermost (its weights come from HBM once).
// PAIR: two CTAs share a tile of 256 channels (cta_group::2): each loads its own 128 channels and half
// the tokens, which is two thirds of the operand bytes a CTA alone takes from L2 for the same products.
// SPLIT: a cluster shares a tile, each CTA a part of K; the partial sums are integers, so their
// order does not matter, and are added through distributed shared memory.

enum class Mm { kOne, kSplit, kPair };
constexpr uint32_t kMmChannels = 128, kMmMaxTokens = 256, kMmKc = 128;
// Warps that take the sums to memory: more where an epilogue's operations come on top (elements of 2 bytes 16, of 4 12;
// what 8 warps hold in flight does not cover the operations' latency: 4096 x 4096 x 4096 f16 with GELU 96 us with 8, 67
// with 16). The registers that leaves are enough where rows of y lie on 16 bytes (up to 8 bytes a thread spill); off
// them 2-byte elements spill 204 bytes a thread, in pairs 156.
__host__ __device__ constexpr uint32_t mm_epi_warps(Mm mode, bool epi, size_t element) {
    return !epi || mode == Mm::kSplit ? 8u : element == 2u ? 16u : 12u;
}
__host__ __device__ constexpr uint32_t mm_threads(Mm mode, bool epi, size_t element) {
    return (mm_epi_warps(mode, epi, element) + 3u) * 32u;
}
constexpr uint32_t kMmWStage = kMmChannels * kMmKc;
constexpr uint32_t kMmMaxStages = 12;
constexpr uint32_t kMmSmemLimit = 227u * 1024u;
constexpr uint64_t kMmWaitNs = 2000000000ull;

template <bool EPI>
struct Int8MmaParams {
    CUtensorMap wmap, xmap;
    LinearParams<EPI> l;
    uint32_t width;     // most tokens a tile takes (a multiple of 16)
    uint32_t box;       // rows of the token operand's TMA box
    uint32_t stages, x_stage;
    uint32_t channels;  // of a tile: 128, a pair's 256
    uint32_t ct, nk;    // channel tiles, K chunks
    uint32_t tmem_cols, acc_cols;
    uint32_t split;
    uint32_t early;     // the kernel ahead quantizes the tokens: weights may be loaded beside it
};

struct MmTile {
    uint32_t g, row0, count, channel0;
};

struct MmShared {
    uint32_t* first;  // [groups + 1] token tiles before group g
    uint32_t* lo;     // [groups] first row
    uint32_t* cnt;    // [groups] rows
    float* scale;     // [2][256] the tile's token scales
    float* channel;   // [2][128] its channels'
    float* weight;    // with an epilogue: [2][256] the tokens' row weights,
    float* bias;      // [2][128] the channels' biases
    float* out;       // [turns of four warps][16][128] act(z) on its way to rows of y
    MmTile* tile;     // [2]
    uint64_t *full, *empty, *acc_full, *acc_empty, *tile_full, *tile_empty;
    uint32_t* tmem;
    volatile uint32_t* abort;
};

__host__ __device__ constexpr uint32_t mm_table_bytes(uint32_t groups) { return (3u * groups + 1u) * 4u; }
__host__ __device__ constexpr uint32_t mm_out_bytes(Mm mode, bool epi, size_t element) {
    return epi && mode != Mm::kSplit ? mm_epi_warps(mode, epi, element) / 4u * 16u * kMmChannels * 4u : 0u;
}
__host__ __device__ constexpr uint32_t mm_fixed_bytes(uint32_t groups, Mm mode, bool epi, size_t element) {
    return mm_out_bytes(mode, epi, element) + (epi ? 4u : 2u) * (kMmMaxTokens + kMmChannels) * 4u + 2u * 16u + (2u * kMmMaxStages + 8u) * 8u + 16u + mm_table_bytes(groups) +
           16u;
}

// Columns of a tile's products: the shapes' steps are 16 for one CTA, 32 for a pair.
template <bool PAIR>
__device__ __forceinline__ uint32_t mm_columns(uint32_t count) {
    return PAIR ? (count + 31u) & ~31u : (count + 15u) & ~15u;
}

// Bounded: false once the time limit has passed or another role has given up. CLUSTER: the arrivals
// come from the peer CTA too.
template <bool CLUSTER = false>
__device__ __forceinline__ bool mm_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* abort) {
    auto done = [&] { return CLUSTER ? tc::mbar_try_cluster(bar, parity) : tc::mbar_try(bar, parity); };
    if (done()) return true;
    const uint64_t t0 = tc::global_ns();
    for (;;) {
        for (uint32_t i = 0; i < 64u; ++i) {
            if (done()) return true;
            if (*abort) return false;
        }
        if (tc::global_ns() - t0 > kMmWaitNs) return false;
    }
}

// A wait that ran out (a fault of this code: every wait's event is this CTA's own copies or
// products) is told to the call's handle: its word in host memory holds 1 until it is read.
__device__ __forceinline__ void mm_report(const Int8LinearParams& l) {
    *static_cast<volatile uint32_t*>(l.error) = 1u;
    __threadfence_system();
}
__device__ __forceinline__ void mm_fail(volatile uint32_t* abort, const Int8LinearParams& l) {
    *abort = 1u;
    mm_report(l);
}

template <bool EPI>
__device__ __forceinline__ MmTile mm_tile(const MmShared& sh, const Int8MmaParams<EPI>& p, uint32_t t) {
    const uint32_t u = t / p.ct;
    uint32_t a = 0, b = p.l.groups;  // last g with first[g] <= u; groups without rows have no tiles
    while (b - a > 1u) {
        const uint32_t mid = (a + b) / 2u;
        if (sh.first[mid] <= u) a = mid;
        else b = mid;
    }
    const uint32_t tt = sh.first[a + 1] - sh.first[a], local = t - sh.first[a] * p.ct;
    const uint32_t c = local / tt, j = local - c * tt;
    // balanced: the first `more` of the group's tiles have one row more than the others
    const uint32_t each = sh.cnt[a] / tt, more = sh.cnt[a] - each * tt;
    return MmTile{a, sh.lo[a] + j * each + min(j, more), each + (j < more ? 1u : 0u), c * p.channels};
}

// A tile's way out with an epilogue (functions of their own: as lambdas of the kernel, which without an epilogue does
// not call them, they cost that form 0.2 us a launch).

// Whether `ok` holds in the four warps of a turn; each of them comes here once a tile, its waits behind it.
__device__ __forceinline__ bool all_of_turn(bool ok, uint32_t warp) {
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 q, %1, 0;\n\t"
        "barrier.cta.red.and.pred p, %2, 128, q;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(all)
        : "r"(ok ? 1u : 0u), "r"(1u + (warp >> 2))
        : "memory");
    return all != 0;
}

// 16 tokens from c on of the CTA's 128 channels (64 columns of y for SwiGLU), with an epilogue: the four warps of a
// turn. act(z) goes to shared memory, and comes back in rows of y: 16 bytes a thread of neighbouring columns, with
// the residual's loaded before. (Stored from where the sums are, a channel a lane, the tokens' rows are 64 bytes a
// store: 4096 x 4096 x 4096 f16 with GELU and a residual 88 us, so 68.)
template <typename TY, bool PAIR, bool WIDE_Y>
__device__ __forceinline__ void finish(const Int8ActParams& l, float* out, const float (&v)[16], const MmTile& tile, uint32_t c,
                                       uint32_t warp, uint32_t rank, const float* ts, const float* rw, float cs, float bias) {
    constexpr uint32_t E = 16u / sizeof(TY);
    const uint32_t lane = threadIdx.x & 31u, quad = warp & 3u, turn = warp >> 2, t = threadIdx.x & 127u, count = min(tile.count - c, 16u);
    const auto put = [&](auto act, auto whole) {
        constexpr int ACT = decltype(act)::value;
        // WIDE: 16 bytes a thread; rows of y at any offset: neighbouring lanes on neighbouring columns
        constexpr bool PAIRS = ACT == VLB_ACT_SWIGLU, WIDE = decltype(whole)::value;
        constexpr uint32_t kEach = WIDE ? E : 1u, kCols = PAIRS ? 64u : 128u;
        constexpr uint32_t kPitch = PAIRS ? 80u : 128u;  // the pitch keeps pairs off each other's banks
        constexpr uint32_t kAcross = kCols / kEach, kRows = 128u / kAcross, kPasses = 16u / kRows;
        float* at = out + turn * (16u * kMmChannels);
        const uint32_t y_cols = PAIRS ? l.out_cols / 2u : l.out_cols;
        const uint32_t col = (tile.channel0 + (PAIR ? rank * kMmChannels : 0u)) / (PAIRS ? 2u : 1u) + t % kAcross * kEach;
        const uint32_t n_cols = col < y_cols ? min(kEach, y_cols - col) : 0u;
        const uint32_t row0 = t / kAcross, rows = n_cols ? count : 0u;  // of this thread: row0, row0 + kRows, ..
        const size_t r0 = tile.row0 + c + row0;
        Pack<TY, kEach> res[kPasses];
        if (l.residual) {
            const TY* from = static_cast<const TY*>(l.residual) + r0 * l.residual_stride + col;
#pragma unroll
            for (uint32_t i = 0; i < kPasses; ++i) {
                if (row0 + i * kRows < rows) {
                    if (n_cols == kEach) {
                        res[i] = *reinterpret_cast<const Pack<TY, kEach>*>(from);
                    } else {
#pragma unroll
                        for (uint32_t j = 0; j < kEach; ++j)
                            if (j < n_cols) res[i].v[j] = from[j];
                    }
                }
                from += kRows * l.residual_stride;
            }
        }
        const float4* t4 = reinterpret_cast<const float4*>(ts + c);
        const uint32_t odd = lane & 1u;  // of a pair's lanes the even one takes the even tokens
#pragma unroll
        for (uint32_t i0 = 0; i0 < 16u; i0 += 4u) {
            const float4 s4 = t4[i0 / 4u];
            float z[4];
#pragma unroll
            for (uint32_t j = 0; j < 4u; ++j) z[j] = epi_sum(__float_as_int(v[i0 + j]), (&s4.x)[j], cs, bias);
            if constexpr (PAIRS) {
#pragma unroll
                for (uint32_t j = 0; j < 4u; j += 2u) {  // one exchange for two tokens
                    const float other = __shfl_xor_sync(0xffffffffu, odd ? z[j] : z[j + 1u], 1);
                    at[(i0 + j + odd) * kPitch + 16u * quad + lane / 2u] =
                        swiglu(odd ? other : z[j], odd ? z[j + 1u] : other, l.act_limit);
                }
            } else {
#pragma unroll
                for (uint32_t j = 0; j < 4u; ++j) at[(i0 + j) * kPitch + 32u * quad + lane] = activate<ACT>(z[j]);
            }
        }
        asm volatile("bar.sync %0, 128;" ::"r"(1u + turn) : "memory");
        TY* y = static_cast<TY*>(l.y) + r0 * l.y_stride + col;
#pragma unroll
        for (uint32_t i = 0; i < kPasses; ++i) {
            const uint32_t row = row0 + i * kRows;
            float f[kEach];
            const Pack<float, kEach> sums = *reinterpret_cast<const Pack<float, kEach>*>(at + row * kPitch + t % kAcross * kEach);
            unpack(sums, f);
            const float w = rw[c + row];
            if (l.residual) {
                float g[kEach];
                unpack(res[i], g);
#pragma unroll
                for (uint32_t j = 0; j < kEach; ++j) f[j] = fmaf(w, f[j], g[j]);
            } else {
#pragma unroll
                for (uint32_t j = 0; j < kEach; ++j) f[j] *= w;
            }
            const Pack<TY, kEach> row_y = pack<TY>(f);
            if (row < rows) {
                if (n_cols == kEach) {
                    *reinterpret_cast<Pack<TY, kEach>*>(y) = row_y;
                } else {
#pragma unroll
                    for (uint32_t j = 0; j < kEach; ++j)
                        if (j < n_cols) y[j] = row_y.v[j];
                }
            }
            y += kRows * l.y_stride;
        }
        asm volatile("bar.sync %0, 128;" ::"r"(1u + turn) : "memory");
    };
    // one branch for all of them, whose chains then run side by side
    const auto by_act = [&](auto whole) {
        switch (l.act) {
            case VLB_ACT_RELU: return put(std::integral_constant<int, VLB_ACT_RELU>{}, whole);
            case VLB_ACT_SILU: return put(std::integral_constant<int, VLB_ACT_SILU>{}, whole);
            case VLB_ACT_GELU: return put(std::integral_constant<int, VLB_ACT_GELU>{}, whole);
            case VLB_ACT_GELU_TANH: return put(std::integral_constant<int, VLB_ACT_GELU_TANH>{}, whole);
            case VLB_ACT_SWIGLU: return put(std::integral_constant<int, VLB_ACT_SWIGLU>{}, whole);
            default: return put(std::integral_constant<int, VLB_ACT_NONE>{}, whole);
        }
    };
    by_act(std::integral_constant<bool, WIDE_Y>{});
}

// WIDE_Y: with an epilogue, rows of y and of the residual lie on 16-byte boundaries (a kernel of its own: the other form's
// registers would spill into it).
template <typename TY, Mm MODE, bool EPI, bool WIDE_Y>
__global__ void __launch_bounds__(mm_threads(MODE, EPI, sizeof(TY)), 1) int8_mma_kernel(const __grid_constant__ Int8MmaParams<EPI> p) {
    constexpr bool SPLIT = MODE == Mm::kSplit, PAIR = MODE == Mm::kPair;
    constexpr uint32_t kEpi = mm_epi_warps(MODE, EPI, sizeof(TY));
    extern __shared__ __align__(1024) unsigned char mm_smem[];
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31u;
    const uint32_t smem = tc::smem_u32(mm_smem), stage_bytes = kMmWStage + p.x_stage;
    const LinearParams<EPI>& l = p.l;
    MmShared sh;
    {
        unsigned char* at = mm_smem + p.stages * stage_bytes;
        sh.out = reinterpret_cast<float*>(at);
        sh.scale = sh.out + mm_out_bytes(MODE, EPI, sizeof(TY)) / 4u;
        sh.channel = sh.scale + 2u * kMmMaxTokens;
        sh.weight = sh.channel + 2u * kMmChannels;
        sh.bias = sh.weight + 2u * kMmMaxTokens;
        sh.tile = reinterpret_cast<MmTile*>(EPI ? sh.bias + 2u * kMmChannels : sh.weight);
        sh.full = reinterpret_cast<uint64_t*>(sh.tile + 2);
        sh.empty = sh.full + kMmMaxStages;
        sh.acc_full = sh.empty + kMmMaxStages;
        sh.acc_empty = sh.acc_full + 2;
        sh.tile_full = sh.acc_empty + 2;
        sh.tile_empty = sh.tile_full + 2;
        sh.tmem = reinterpret_cast<uint32_t*>(sh.tile_empty + 2);
        sh.abort = sh.tmem + 1;
        sh.first = sh.tmem + 4;
        sh.lo = sh.first + l.groups + 1;
        sh.cnt = sh.lo + l.groups;
    }
    if (!p.early) tc::grid_dependency_wait();
    if (smem & 1023u) {  // the swizzle atoms need it; the same in every CTA of the launch
        tc::grid_dependency_wait();
        if (tid == 0) mm_report(l);
        return;
    }
    if (warp == kEpi) {
        if (PAIR) tc::tmem_alloc_pair(sh.tmem, p.tmem_cols);
        else tc::tmem_alloc(sh.tmem, p.tmem_cols);
    }
    if (warp == kEpi + 1u && lane < 2u)
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(lane ? &p.xmap : &p.wmap)) : "memory");
    if (tid == 0) {
        for (uint32_t i = 0; i < p.stages; ++i) {
            tc::mbar_init(sh.full + i, 1);
            tc::mbar_init(sh.empty + i, 1);
        }
        for (uint32_t i = 0; i < 2u; ++i) {
            tc::mbar_init(sh.acc_full + i, 1);
            tc::mbar_init(sh.acc_empty + i, PAIR ? 2u * kEpi : kEpi);
            tc::mbar_init(sh.tile_full + i, 1);
            tc::mbar_init(sh.tile_empty + i, kEpi);
        }
        *sh.abort = 0;
        tc::mbar_fence_init();
    }
    for (uint32_t g = tid; g < l.groups; g += mm_threads(MODE, EPI, sizeof(TY))) {
        uint32_t lo, hi;
        group_range(l, g, lo, hi);
        sh.lo[g] = lo;
        sh.cnt[g] = hi - lo;
    }
    __syncthreads();
    if (warp == kEpi + 1u) {
        // token tiles before each group, 32 groups a step
        uint32_t run = 0;
        for (uint32_t g0 = 0; g0 < l.groups; g0 += 32u) {
            const uint32_t g = g0 + lane;
            const uint32_t tiles = g < l.groups ? (sh.cnt[g] + p.width - 1u) / p.width : 0u;
            uint32_t incl = tiles;
#pragma unroll
            for (uint32_t d = 1; d < 32u; d <<= 1) {
                const uint32_t v = __shfl_up_sync(0xffffffffu, incl, d);
                if (lane >= d) incl += v;
            }
            if (g < l.groups) sh.first[g] = run + incl - tiles;
            run += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) sh.first[l.groups] = run;
    }
    tc::fence_before_sync();
    __syncthreads();
    if (PAIR) tc::cluster_sync();  // the peer's barriers and TMEM are ready too
    tc::fence_after_sync();
    const uint32_t tmem = *sh.tmem;
    const uint32_t total = sh.first[l.groups] * p.ct;
    const uint32_t rank = MODE != Mm::kOne ? tc::cluster_rank() : 0u, in_cluster = SPLIT ? p.split : PAIR ? 2u : 1u;
    const uint32_t step = gridDim.x / in_cluster, begin = blockIdx.x / in_cluster;
    const uint32_t k_lo = SPLIT ? p.nk * rank / p.split : 0u, k_hi = SPLIT ? p.nk * (rank + 1u) / p.split : p.nk;
    const uint32_t nk = k_hi - k_lo;
    bool dirty = false, pending = false;  // copies / products under way when a role gave up
    uint32_t pending_bar = 0, pending_parity = 0;

    tc::grid_launch_dependents();
    // ---- roles; in SPLIT mode each returns to the common tile loop after one tile -------------
    uint32_t stage = 0, phase = 0, it = 0;
    bool waited = false;  // on the kernel ahead
    auto next_stage = [&] {
        if (++stage == p.stages) stage = 0, phase ^= 1u;
    };
    // One K chunk's operands: 128 rows of w, and the tile's tokens (a pair: this CTA's half of them) in
    // boxes. Rows past the tile's are loaded and not used; past the matrix, also past K, the TMA unit
    // fills zeros. A pair's bytes all complete on the first CTA's barrier. One lane of a warp in step
    // runs these, as the products.
    struct Source {
        int32_t w_row, x_row;
        uint32_t boxes;
    };
    const uint32_t full0 = PAIR ? tc::cluster_map(tc::smem_u32(sh.full), 0) : tc::smem_u32(sh.full);
    auto load_w = [&](uint32_t st, const Source& src, uint32_t kc) {
        if (!PAIR || rank == 0)
            tc::mbar_arrive_expect_tx(sh.full + st, (PAIR ? 2u : 1u) * (src.boxes * p.box * kMmKc + kMmWStage));
        if (PAIR) tc::tma_load_2d_pair(smem + st * stage_bytes, &p.wmap, (int32_t)(kc * kMmKc), src.w_row, full0 + st * 8u);
        else tc::tma_load_2d(smem + st * stage_bytes, &p.wmap, (int32_t)(kc * kMmKc), src.w_row, sh.full + st);
    };
    auto load_x = [&](uint32_t st, const Source& src, uint32_t kc) {
        const uint32_t dst = smem + st * stage_bytes + kMmWStage;
        for (uint32_t b = 0; b < src.boxes; ++b) {
            const int32_t x = (int32_t)(kc * kMmKc), y = src.x_row + (int32_t)(b * p.box);
            if (PAIR) tc::tma_load_2d_pair(dst + b * p.box * kMmKc, &p.xmap, x, y, full0 + st * 8u);
            else tc::tma_load_2d(dst + b * p.box * kMmKc, &p.xmap, x, y, sh.full + st);
        }
    };
    auto produce = [&](uint32_t t) -> bool {
        const MmTile tile = mm_tile(sh, p, t);
        const uint32_t own = PAIR ? mm_columns<PAIR>(tile.count) / 2u : tile.count;
        Source src;
        src.w_row = (int32_t)(tile.g * l.out_cols + tile.channel0 + (PAIR ? rank * kMmChannels : 0u));
        src.x_row = (int32_t)(tile.row0 + (PAIR ? rank * own : 0u));
        src.boxes = (own + p.box - 1u) / p.box;
        dirty = true;
        uint32_t done = 0;
        if (!waited) {
            // the weights are no kernel's output: the first stages' are on their way while the
            // kernel ahead still quantizes the tokens
            done = nk < p.stages ? nk : p.stages;
            if (tc::elect_lane())
                for (uint32_t i = 0; i < done; ++i) load_w(i, src, k_lo + i);
            __syncwarp();
            tc::grid_dependency_wait();
            waited = true;
            if (tc::elect_lane())
                for (uint32_t i = 0; i < done; ++i) load_x(i, src, k_lo + i);
            __syncwarp();
            for (uint32_t i = 0; i < done; ++i) next_stage();
        }
        for (uint32_t i = done; i < nk; ++i) {
            if (!__all_sync(0xffffffffu, mm_wait(sh.empty + stage, phase ^ 1u, sh.abort))) return false;
            if (tc::elect_lane()) {
                load_w(stage, src, k_lo + i);
                load_x(stage, src, k_lo + i);
            }
            __syncwarp();
            next_stage();
        }
        dirty = false;
        return true;
    };
    auto commit = [&](uint64_t* bar) {
        if (PAIR) tc::mma_commit_pair(bar);
        else tc::mma_commit(bar);
    };
    // the whole warp, in step
    auto multiply = [&](uint32_t t) -> bool {
        const MmTile tile = mm_tile(sh, p, t);
        const uint32_t buf = SPLIT ? 0u : it & 1u, use = SPLIT ? it : it >> 1;
        if (!SPLIT && !__all_sync(0xffffffffu, mm_wait<PAIR>(sh.acc_empty + buf, (use & 1u) ^ 1u, sh.abort))) return false;
        tc::fence_after_sync();
        const uint32_t idesc = tc::idesc_i8(PAIR ? 2u * kMmChannels : kMmChannels, mm_columns<PAIR>(tile.count));
        const uint32_t acc = tmem + buf * p.acc_cols;
        pending_bar = buf;
        pending_parity = use & 1u;
        for (uint32_t i = 0; i < nk; ++i) {
            if (!__all_sync(0xffffffffu, mm_wait(sh.full + stage, phase, sh.abort))) return false;
            tc::fence_after_sync();
            pending = true;
            if (tc::elect_lane()) {
                const uint64_t wd = tc::sw128_desc(smem + stage * stage_bytes);
                const uint64_t xd = tc::sw128_desc(smem + stage * stage_bytes + kMmWStage);
#pragma unroll
                for (uint32_t ks = 0; ks < kMmKc / 32u; ++ks) {  // 32 bytes on: 2 of the descriptor's 16-byte units
                    if (PAIR) tc::mma_i8_pair(acc, wd + 2u * ks, xd + 2u * ks, idesc, (i | ks) ? 1u : 0u);
                    else tc::mma_i8(acc, wd + 2u * ks, xd + 2u * ks, idesc, (i | ks) ? 1u : 0u);
                }
                commit(sh.empty + stage);
                if (i + 1u == nk) commit(sh.acc_full + buf);
            }
            __syncwarp();
            next_stage();
        }
        pending = false;
        ++it;
        return true;
    };
    const uint32_t quad = warp & 3u, half = warp >> 2;
    // the whole warp
    auto place = [&](uint32_t t) -> bool {
        const uint32_t buf = it & 1u, use = it >> 1;
        const MmTile tile = mm_tile(sh, p, t);
        if (!waited) {
            tc::grid_dependency_wait();
            waited = true;
        }
        float ts[kMmMaxTokens / 32u], cs[kMmChannels / 32u], rw[EPI ? kMmMaxTokens / 32u : 1u], bs[EPI ? kMmChannels / 32u : 1u];
#pragma unroll
        for (uint32_t i = 0; i < kMmMaxTokens / 32u; ++i) {
            const uint32_t j = lane + 32u * i;
            ts[i] = j < tile.count ? l.x_scale[tile.row0 + j] : 0.f;
            if constexpr (EPI) rw[i] = l.row_weight && j < tile.count ? l.row_weight[tile.row0 + j] : 1.f;
            else if (l.row_weight && j < tile.count) ts[i] *= l.row_weight[tile.row0 + j];
        }
#pragma unroll
        for (uint32_t i = 0; i < kMmChannels / 32u; ++i) {
            const uint32_t n = tile.channel0 + (PAIR ? rank * kMmChannels : 0u) + lane + 32u * i;
            cs[i] = n < l.out_cols ? l.w_scale[(size_t)tile.g * l.out_cols + n] : 0.f;
            if constexpr (EPI) bs[i] = l.bias && n < l.out_cols ? l.bias[(size_t)tile.g * l.out_cols + n] : 0.f;
        }
        if (!__all_sync(0xffffffffu, mm_wait(sh.tile_empty + buf, (use & 1u) ^ 1u, sh.abort))) return false;
#pragma unroll
        for (uint32_t i = 0; i < kMmMaxTokens / 32u; ++i) sh.scale[buf * kMmMaxTokens + lane + 32u * i] = ts[i];
#pragma unroll
        for (uint32_t i = 0; i < kMmChannels / 32u; ++i) sh.channel[buf * kMmChannels + lane + 32u * i] = cs[i];
        if constexpr (EPI) {
#pragma unroll
            for (uint32_t i = 0; i < kMmMaxTokens / 32u; ++i) sh.weight[buf * kMmMaxTokens + lane + 32u * i] = rw[i];
#pragma unroll
            for (uint32_t i = 0; i < kMmChannels / 32u; ++i) sh.bias[buf * kMmChannels + lane + 32u * i] = bs[i];
        }
        if (lane == 0) sh.tile[buf] = tile;
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(sh.tile_full + buf);
        ++it;
        return true;
    };
    auto epilogue = [&]() -> bool {
        const uint32_t buf = it & 1u, use = it >> 1;
        const float* ts = sh.scale + buf * kMmMaxTokens;
        bool ok = __all_sync(0xffffffffu, mm_wait(sh.tile_full + buf, use & 1u, sh.abort));
        const MmTile tile = sh.tile[buf];
        const float cs = sh.channel[buf * kMmChannels + 32u * quad + lane];
        const uint32_t n = tile.channel0 + (PAIR ? rank * kMmChannels : 0u) + 32u * quad + lane;
        ok = ok && __all_sync(0xffffffffu, mm_wait(sh.acc_full + buf, use & 1u, sh.abort));
        if constexpr (EPI) ok = all_of_turn(ok, warp);  // the four warps go on to their barriers, or give up, together
        if (ok) {
            tc::fence_after_sync();
            const uint32_t src = tmem + buf * p.acc_cols + ((32u * quad) << 16);
            if constexpr (EPI) {
                const float bias = sh.bias[buf * kMmChannels + 32u * quad + lane];
                for (uint32_t c = 16u * half; c < tile.count; c += 4u * kEpi) {
                    float v[16];
                    tc::tmem_ld16(src + c, v);
                    tc::tmem_wait_ld();
                    finish<TY, PAIR, WIDE_Y>(l, sh.out, v, tile, c, warp, rank, ts, sh.weight + buf * kMmMaxTokens, cs, bias);
                }
            }
            // 32 columns (tokens) at a time, the warps of a lane quarter taking turns
            for (uint32_t c = 32u * half; !EPI && c < tile.count; c += 64u) {
                uint32_t v[32];
                tc::tmem_ld32(src + c, v);
                tc::tmem_wait_ld();
                TY* y = static_cast<TY*>(l.y) + (size_t)(tile.row0 + c) * l.y_stride + n;
                const float4* t4 = reinterpret_cast<const float4*>(ts + c);
                if (tile.count - c >= 32u && n - lane + 32u <= l.out_cols) {
#pragma unroll
                    for (uint32_t i = 0; i < 32u; i += 4u) {
                        const float4 t = t4[i / 4u];
                        y[0] = from_float<TY>((float)(int32_t)v[i] * t.x * cs);
                        y += l.y_stride;
                        y[0] = from_float<TY>((float)(int32_t)v[i + 1] * t.y * cs);
                        y += l.y_stride;
                        y[0] = from_float<TY>((float)(int32_t)v[i + 2] * t.z * cs);
                        y += l.y_stride;
                        y[0] = from_float<TY>((float)(int32_t)v[i + 3] * t.w * cs);
                        y += l.y_stride;
                    }
                } else if (n < l.out_cols) {
#pragma unroll
                    for (uint32_t i = 0; i < 32u; ++i)
                        if (c + i < tile.count) y[i * l.y_stride] = from_float<TY>((float)(int32_t)v[i] * ts[c + i] * cs);
                }
            }
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                tc::mbar_arrive(sh.tile_empty + buf);
                if (PAIR) tc::mbar_arrive_cluster(tc::cluster_map(tc::smem_u32(sh.acc_empty + buf), 0));
                else tc::mbar_arrive(sh.acc_empty + buf);
            }
            ++it;
        }
        return ok;
    };

    if (!SPLIT) {
        if (warp < kEpi) {
            for (uint32_t t = begin; t < total; t += step)
                if (!epilogue()) {
                    if (lane == 0) mm_fail(sh.abort, l);
                    break;
                }
        } else if (warp == kEpi) {
            for (uint32_t t = begin; t < total; t += step)
                if (!produce(t)) {
                    if (lane == 0) mm_fail(sh.abort, l);
                    break;
                }
        } else if (warp == kEpi + 2u) {
            for (uint32_t t = begin; t < total; t += step)
                if (!place(t)) {
                    if (lane == 0) mm_fail(sh.abort, l);
                    break;
                }
        } else if (!PAIR || rank == 0) {
            for (uint32_t t = begin; t < total; t += step)
                if (!multiply(t)) {
                    if (lane == 0) mm_fail(sh.abort, l);
                    break;
                }
        }
    } else {
        int32_t* part = reinterpret_cast<int32_t*>(mm_smem);  // [token][128], over the idle ring
        for (uint32_t t = begin; t < total; t += step) {
            // every CTA of the cluster takes part in both barriers of every tile, also after a
            // role has given up
            const MmTile tile = mm_tile(sh, p, t);
            bool ok = true;
            float cs[4] = {}, bs[4] = {};
            float* ts = sh.scale;
            if (warp == kEpi) {
                ok = __all_sync(0xffffffffu, *sh.abort == 0) && produce(t);
            } else if (warp == kEpi + 1u) {
                ok = __all_sync(0xffffffffu, *sh.abort == 0) && multiply(t);
            } else if (warp < kEpi) {
                if (!waited) {
                    tc::grid_dependency_wait();
                    waited = true;
                }
                if (tid < tile.count) {
                    const uint32_t r = tile.row0 + tid;
                    ts[tid] = !EPI && l.row_weight ? l.x_scale[r] * l.row_weight[r] : l.x_scale[r];
                    if constexpr (EPI) sh.weight[tid] = l.row_weight ? l.row_weight[r] : 1.f;
                }
                ok = __all_sync(0xffffffffu, *sh.abort == 0 && mm_wait(sh.acc_full, it & 1u, sh.abort));
                ++it;
#pragma unroll
                for (uint32_t i = 0; i < 4u; ++i) {
                    const uint32_t n = tile.channel0 + 4u * lane + i;
                    cs[i] = n < l.out_cols ? l.w_scale[(size_t)tile.g * l.out_cols + n] : 0.f;
                    if constexpr (EPI) bs[i] = l.bias && n < l.out_cols ? l.bias[(size_t)tile.g * l.out_cols + n] : 0.f;
                }
                if (ok) {
                    tc::fence_after_sync();
                    const uint32_t src = tmem + ((32u * quad) << 16);
                    for (uint32_t c = 16u * half; c < tile.count; c += 32u) {
                        float v[16];
                        tc::tmem_ld16(src + c, v);
                        tc::tmem_wait_ld();
#pragma unroll
                        for (uint32_t i = 0; i < 16u; ++i)
                            part[(c + i) * kMmChannels + 32u * quad + lane] = __float_as_int(v[i]);
                    }
                    tc::fence_before_sync();
                }
            }
            if (!ok && lane == 0) mm_fail(sh.abort, l);
            __syncwarp();
            tc::cluster_sync();
            if (warp < kEpi) {
                // a warp takes every split-th token, a lane four neighbouring channels: the loads of two
                // tokens from all peers are in flight together
                const uint32_t pace = kEpi * p.split, c = 4u * lane, n = tile.channel0 + c;
                for (uint32_t j = rank + p.split * warp; j < tile.count; j += 2u * pace) {
                    uint4 v[2][8];
#pragma unroll
                    for (uint32_t u = 0; u < 2u; ++u)
#pragma unroll
                        for (uint32_t r = 0; r < 8u; ++r)
                            v[u][r] = r < p.split && j + u * pace < tile.count
                                          ? tc::cluster_ld16(smem + ((j + u * pace) * kMmChannels + c) * 4u, r)
                                          : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                    for (uint32_t u = 0; u < 2u; ++u) {
                        if (j + u * pace >= tile.count) break;
                        uint4 sum = v[u][0];
#pragma unroll
                        for (uint32_t r = 1; r < 8u; ++r)
                            sum.x += v[u][r].x, sum.y += v[u][r].y, sum.z += v[u][r].z, sum.w += v[u][r].w;
                        const float s = ts[j + u * pace];
                        if constexpr (EPI) {
                            const bool pairs = l.act == VLB_ACT_SWIGLU;
                            const size_t r = tile.row0 + j + u * pace;
                            const float rw = sh.weight[j + u * pace];
                            const TY* from = static_cast<const TY*>(l.residual);
                            float z[4];
#pragma unroll
                            for (uint32_t i = 0; i < 4u; ++i) z[i] = epi_sum((int32_t)(&sum.x)[i], s, cs[i], bs[i]);
#pragma unroll
                            for (uint32_t i = 0; i < 4u; ++i) {
                                if (n + i >= l.out_cols || (pairs && (i & 1u))) continue;
                                const uint32_t to = pairs ? (n + i) / 2u : n + i;
                                const float a = pairs ? swiglu(z[i], z[i | 1u], l.act_limit) : activate(z[i], l.act);
                                const float res = from ? to_float(from[r * l.residual_stride + to]) : kNoResidual;
                                static_cast<TY*>(l.y)[r * l.y_stride + to] = from_float<TY>(fmaf(rw, a, res));
                            }
                            continue;
                        }
                        TY* y = static_cast<TY*>(l.y) + (size_t)(tile.row0 + j + u * pace) * l.y_stride + n;
#pragma unroll
                        for (uint32_t i = 0; i < 4u; ++i)
                            if (n + i < l.out_cols) y[i] = from_float<TY>((float)(int32_t)(&sum.x)[i] * s * cs[i]);
                    }
                }
            }
            tc::fence_proxy_async();
            tc::fence_after_sync();
            tc::cluster_sync();
        }
    }
    if (!waited) tc::grid_dependency_wait();  // also a CTA without a tile
    __syncthreads();
    if (warp == kEpi && lane == 0 && dirty) {
        // after giving up: copies already issued land before the CTA's shared memory goes away
        const uint64_t t0 = tc::global_ns();
        while (tc::global_ns() - t0 < 1000000ull) {
        }
    }
    if (warp == kEpi + 1u && pending && tc::elect_lane()) {
        commit(sh.acc_full + pending_bar);
        const uint64_t t0 = tc::global_ns();
        while (!tc::mbar_try(sh.acc_full + pending_bar, pending_parity) && tc::global_ns() - t0 < kMmWaitNs) {
        }
    }
    __syncthreads();
    if (PAIR) {
        // the peer may still be read by products or signal this CTA's barriers
        tc::fence_before_sync();
        tc::cluster_sync();
    }
    if (warp == kEpi) {
        tc::fence_after_sync();
        if (PAIR) tc::tmem_dealloc_pair(tmem, p.tmem_cols);
        else tc::tmem_dealloc(tmem, p.tmem_cols);
    }
}

template <typename T, bool SWIGLU>
cudaError_t quantize_rows(const Int8QuantParams& p, cudaStream_t s) {
    constexpr uint32_t N = RowVec<T>::kN;
    auto on = [](const void* at, size_t stride_bytes, size_t n) {
        return reinterpret_cast<uintptr_t>(at) % n == 0 && stride_bytes % n == 0;
    };
    const uint32_t by_block = p.rows < 65535u ? p.rows : 65535u, by_warp = (p.rows + 7u) / 8u;
    const auto launch = [&](auto* kernel, uint32_t grid) { return launch_chained(kernel, dim3(grid), 256, 0, 0, s, p); };
    // a warp a row where that fills the GPU (with a product of 16 channels, a warp / a CTA a row: 512
    // rows of 1024 bf16 8.4 / 8.6 us, 1024 8.6 / 10.2, 4096 10.9 / 15.9)
    const bool many = p.rows >= 1024u;
    if (!on(p.x, p.x_stride * sizeof(T), 16) || !on(p.up, 0, 16) || !on(p.q, p.q_stride, N)) {
        if (many && p.cols <= 32u * 16u) return launch(int8_quantize_kernel<T, SWIGLU, 32, 16>, by_warp);
        if (p.cols <= 256u * 4u) return launch(int8_quantize_kernel<T, SWIGLU, 256, 4>, by_block);
        return launch(int8_quantize_kernel<T, SWIGLU, 256, 16>, by_block);
    }
    if (many && p.cols <= 32u * 4u * N) return launch(int8_quantize_vec_kernel<T, SWIGLU, 32, 4>, by_warp);
    if (many && p.cols <= 32u * 8u * N) return launch(int8_quantize_vec_kernel<T, SWIGLU, 32, 8>, by_warp);
    if constexpr (!SWIGLU) {
        if (many && p.cols <= 32u * 16u * N) return launch(int8_quantize_vec_kernel<T, SWIGLU, 32, 16>, by_warp);
    }
    if (p.cols <= 256u * 2u * N) return launch(int8_quantize_vec_kernel<T, SWIGLU, 256, 2>, by_block);
    return launch(int8_quantize_vec_kernel<T, SWIGLU, 256, 4>, by_block);
}

template <typename T>
cudaError_t quantize_type(const Int8QuantParams& p, cudaStream_t s) {
    return p.up ? quantize_rows<T, true>(p, s) : quantize_rows<T, false>(p, s);
}

template <typename TY, bool EPI>
cudaError_t general_type(const LinearParams<EPI>& p, cudaStream_t s) {
    const uint32_t tiles_n = (p.out_cols + kGenTile - 1u) / kGenTile, tiles_r = (p.rows + kGenTile - 1u) / kGenTile;
    const dim3 grid(tiles_n, tiles_r < 1024u ? tiles_r : 1024u, p.groups < 1024u ? p.groups : 1024u);
    return launch_chained(int8_linear_kernel<TY, EPI>, grid, 256, 0, 0, s, p);
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(f);
    });
    return fn;
}

// Rows of bytes read as boxes of 128 columns x box_rows with the 128-byte swizzle.
bool encode_rows(CUtensorMap* map, const int8_t* base, uint64_t rows, uint64_t cols, uint64_t stride, uint32_t box_rows) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    const cuuint64_t dims[2] = {cols, rows};
    const cuuint64_t strides[1] = {stride};
    const cuuint32_t box[2] = {kMmKc, box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool tma_rows(const int8_t* p, size_t stride) {
    return reinterpret_cast<uintptr_t>(p) % 16u == 0 && stride % 16u == 0;
}

// Tile width, split or pairs of a product on the tensor cores. Returns the mode.
template <bool EPI>
Mm mma_plan(Int8MmaParams<EPI>& p, uint32_t sms, size_t y_size) {
    const Int8LinearParams& l = p.l;
    p.nk = (l.cols + kMmKc - 1u) / kMmKc;
    const auto split_of = [&](uint64_t tiles) {
        // clusters of 8 only while they are few: more of them do not fit the GPU at once (16 tiles of
        // 2048 x 2048 x 64 rows: 14 us in eights, 9 in fours)
        uint32_t split = 1;
        while (split < 8u && tiles * split * 2u <= (split < 4u ? sms : 64u) && p.nk >= split * 2u) split *= 2u;
        return split;
    };
    const auto up = [](uint32_t v, uint32_t step) { return (v + step - 1u) / step * step; };
    Mm mode = Mm::kOne;
    if (l.groups == 1) {
        // One CTA a tile (K split over a cluster where the tiles are few) or pairs, and the tiles'
        // width: what takes the least cycles by what was measured - a K chunk its columns + 240 (424
        // at 128 columns, 525 at 256; a tenth more for CTAs alone, which draw more from L2), an
        // epilogue 1,500 and 18 a column, a split's sums 4,000 and 32 a column, a pair's start 1,500.
        // (4096 x 4096, int8 rows, split or alone / pairs: 130 rows 9.8 / 11.2 us, 300 12.4 / 11.8,
        // 2048 28.8 / 26.5; 1024 -> 4096: 130 rows 8.9 / 6.9, 1024 8.1 / 9.1.)
        uint64_t best = ~0ull;
        for (uint32_t pair = 0; pair < 2u; ++pair) {
            const uint32_t step = pair ? 32u : 16u, most = up(l.rows < kMmMaxTokens ? l.rows : kMmMaxTokens, step);
            const uint64_t ct = (l.out_cols + kMmChannels * (1u + pair) - 1u) / (kMmChannels * (1u + pair));
            for (uint32_t w = most; w >= 64u || w == most; w -= step) {
                const uint64_t n = (l.rows + w - 1u) / w, tiles = n * ct;
                const uint32_t split = pair ? 1u : split_of(tiles);
                const uint64_t units = pair ? sms / 2u : sms / split, waves = (tiles + units - 1u) / units;
                const uint64_t columns = up((uint32_t)((l.rows + n - 1u) / n), step);
                uint64_t main = (p.nk + split - 1u) / split * (columns + 240u), cost;
                if (split > 1u) {
                    cost = waves * (main + 4000u + 32u * columns);
                } else {
                    if (!pair) main += main / 10u;
                    const uint64_t tail = 1500u + 18u * columns;
                    cost = (waves - 1u) * (main > tail ? main : tail) + main + tail + (pair ? 1500u : 0u);
                }
                if (cost < best) {
                    best = cost;
                    mode = pair ? Mm::kPair : split > 1u ? Mm::kSplit : Mm::kOne;
                    p.width = w;
                    p.split = split;
                }
                if (w <= step) break;
            }
        }
    } else {
        // The rows of each group are on the device only. Pairs from about 100 rows a group (64 groups
        // of 2048 x 2048: 64 rows 55.6 us alone / 56.9 in pairs, 96 60.0 / 60.5, 128 65.2 / 61.8, 512
        // 155 / 142); room for the usual spread around the mean, or a second tile would read the
        // group's weights again.
        const uint32_t used = l.groups < l.rows ? l.groups : l.rows, mean = (l.rows + used - 1u) / used;
        uint32_t spread = 1;
        while (spread * spread < mean) ++spread;
        if (mean >= 100u) mode = Mm::kPair;
        const uint32_t want = up(mean + 3u * spread, mode == Mm::kPair ? 32u : 16u);
        p.width = want < kMmMaxTokens ? want : kMmMaxTokens;
        p.split = 1;
        if (mode == Mm::kOne) {
            const uint64_t ct = (l.out_cols + kMmChannels - 1u) / kMmChannels;
            p.split = split_of((uint64_t)used * ((mean + p.width - 1u) / p.width) * ct);
            if (p.split > 1) mode = Mm::kSplit;
        }
    }
    p.channels = mode == Mm::kPair ? 2u * kMmChannels : kMmChannels;
    p.ct = (l.out_cols + p.channels - 1u) / p.channels;
    const uint32_t held = mode == Mm::kPair ? p.width / 2u : p.width;  // token rows in one CTA's stage
    p.box = held < 128u ? held : 128u;
    p.x_stage = (held + p.box - 1u) / p.box * p.box * kMmKc;
    p.acc_cols = p.width < 32u ? 32u : p.width;
    p.tmem_cols = 32;
    while (p.tmem_cols < (mode == Mm::kSplit ? 1u : 2u) * p.acc_cols) p.tmem_cols *= 2u;
    const uint32_t room = kMmSmemLimit - 1024u - mm_fixed_bytes(l.groups, mode, EPI, y_size);
    p.stages = room / (kMmWStage + p.x_stage);
    if (p.stages > kMmMaxStages) p.stages = kMmMaxStages;
    return mode;
}

template <typename TY, Mm MODE, bool EPI>
cudaError_t mma_launch(const Int8MmaParams<EPI>& p, uint32_t sms, bool wide, cudaStream_t s) {
    constexpr bool kForms = EPI && MODE != Mm::kSplit;  // a split's sums take another way out
    auto* kernel = wide && kForms ? int8_mma_kernel<TY, MODE, EPI, kForms> : int8_mma_kernel<TY, MODE, EPI, false>;
    const uint32_t in_cluster = MODE == Mm::kSplit ? p.split : MODE == Mm::kPair ? 2u : 1u;
    cudaError_t e = smem_once(kernel, kMmSmemLimit);
    if (e != cudaSuccess) return e;
    const size_t smem = p.stages * (kMmWStage + p.x_stage) + mm_fixed_bytes(p.l.groups, MODE, EPI, sizeof(TY));
    return launch_chained(kernel, dim3(sms / in_cluster * in_cluster), mm_threads(MODE, EPI, sizeof(TY)), smem, MODE == Mm::kOne ? 0 : in_cluster, s, p);
}

// What int8_few_kernel takes. Dense: up to kFewRows rows, from 3 on no more than kFewElements elements
// and kFewWork products; its dp4a work grows with the rows while the tensor cores' two launches do not
// (2048 x 2048: 3.6 us for one row, 6.1 for 4, 9.3 for 8, against about 6; 4096 x 4096: 5.7, 11.2, 21.9,
// against about 9), and every block quantizes all rows (5 rows of 3470: longer than the products).
// Grouped: up to kFewGroupedRows rows and no more than the groups, as each row reads its matrix and few
// then share one (2048 x 2048, few / tensor cores: 8, 24, 32 rows of 64 groups 8.8 / 10.7, 18.6 / 22.2,
// 25.3 / 23.6 us; 8, 16 rows of 8 groups 8.2 / 10.3, 12.9 / 10.5). Measured at these widths only.
constexpr uint32_t kFewRows = 8, kFewGroupedRows = 24, kFewElements = 8192;
constexpr uint64_t kFewWork = 1u << 24;

template <typename T, uint32_t ROWS, bool EPI, bool GROUPED = false>
cudaError_t few_launch(const LinearParams<EPI>& l, const Int8QuantParams& q, int y_type, uint32_t sms, cudaStream_t s) {
    auto* kernel = int8_few_kernel<T, ROWS, EPI, GROUPED>;
    const size_t smem = (size_t)ROWS * ((l.cols + 15u) / 16u * 16u);
    if (smem > kFewDefaultSmem) {
        const cudaError_t e = smem_once(kernel, kFewSmem);
        if (e != cudaSuccess) return e;
    }
    const uint32_t sets = GROUPED ? l.rows : 1u, slots = few_blocks(GROUPED) * sms;
    uint32_t channels = (uint32_t)(((uint64_t)l.out_cols * sets + slots - 1u) / slots);
    channels = (channels + 2u * kFewWarps - 1u) / (2u * kFewWarps) * (2u * kFewWarps);
    return launch_chained(kernel, dim3((l.out_cols + channels - 1u) / channels, sets), kFewThreads, smem, 0, s, l, q, y_type,
                          channels);
}

template <typename T, bool EPI>
cudaError_t few_rows(const LinearParams<EPI>& l, const Int8QuantParams& q, int y_type, cudaStream_t s) {
    const uint32_t rows = l.rows, sms = sm_count();
    if (l.offsets) return few_launch<T, 1, EPI, true>(l, q, y_type, sms, s);
    if (rows <= 1u) return few_launch<T, 1, EPI>(l, q, y_type, sms, s);
    if (rows <= 2u) return few_launch<T, 2, EPI>(l, q, y_type, sms, s);
    if (rows <= 4u) return few_launch<T, 4, EPI>(l, q, y_type, sms, s);
    return few_launch<T, 8, EPI>(l, q, y_type, sms, s);
}

template <typename TY, bool EPI>
cudaError_t linear_type(const LinearParams<EPI>& l, bool after_quantize, cudaStream_t s) {
    if (tma_rows(l.w, l.w_stride) && tma_rows(l.x, l.x_stride)) {
        Int8MmaParams<EPI> p{};
        p.l = l;
        p.early = after_quantize;
        const auto on16 = [](const void* at, size_t stride) {
            return reinterpret_cast<uintptr_t>(at) % 16u == 0 && stride * sizeof(TY) % 16u == 0;
        };
        bool wide = false;
        if constexpr (EPI) wide = on16(l.y, l.y_stride) && (!l.residual || on16(l.residual, l.residual_stride));
        const uint32_t sms = sm_count();
        const Mm mode = mma_plan(p, sms, sizeof(TY));
        if (encode_rows(&p.wmap, l.w, (uint64_t)l.groups * l.out_cols, l.cols, l.w_stride, kMmChannels) &&
            encode_rows(&p.xmap, l.x, l.rows, l.cols, l.x_stride, p.box))
            return mode == Mm::kPair    ? mma_launch<TY, Mm::kPair, EPI>(p, sms, wide, s)
                   : mode == Mm::kSplit ? mma_launch<TY, Mm::kSplit, EPI>(p, sms, wide, s)
                                        : mma_launch<TY, Mm::kOne, EPI>(p, sms, wide, s);
    }
    return general_type<TY, EPI>(l, s);
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

cudaError_t launch_int8_gather(const Int8GatherParams& p, cudaStream_t s) {
    return launch_chained(int8_gather_kernel, dim3((p.rows + 7u) / 8u), 256, 0, 0, s, p);
}

bool int8_few(const Int8LinearParams& l) {
    if (l.rows > (l.offsets ? kFewGroupedRows : kFewRows) || !tma_rows(l.w, l.w_stride)) return false;
    if (l.offsets && l.rows > l.groups) return false;
    if (!l.offsets && l.rows > 2u &&
        ((uint64_t)l.rows * l.cols > kFewElements || (uint64_t)l.rows * l.cols * l.out_cols > kFewWork))
        return false;
    uint32_t rows = 1;
    while (!l.offsets && rows < l.rows) rows *= 2u;
    return (size_t)rows * ((l.cols + 15u) / 16u * 16u) <= kFewSmem;
}

template <bool EPI>
static cudaError_t few_typed(const LinearParams<EPI>& l, const Int8QuantParams& q, int x_type, int y_type, cudaStream_t s) {
    switch (x_type) {
        case VLB_DTYPE_F32: return few_rows<float, EPI>(l, q, y_type, s);
        case VLB_DTYPE_F16: return few_rows<__half, EPI>(l, q, y_type, s);
        case VLB_DTYPE_BF16: return few_rows<__nv_bfloat16, EPI>(l, q, y_type, s);
        default: return few_rows<int8_t, EPI>(l, q, y_type, s);
    }
}
cudaError_t launch_int8_few(const Int8ActParams& l, const Int8QuantParams& q, int x_type, int y_type, cudaStream_t s) {
    return l.act == kInt8NoEpilogue ? few_typed<false>(l, q, x_type, y_type, s) : few_typed<true>(l, q, x_type, y_type, s);
}

template <bool EPI>
static cudaError_t linear_typed(const LinearParams<EPI>& p, int y_type, bool after_quantize, cudaStream_t s) {
    switch (y_type) {
        case VLB_DTYPE_F32: return linear_type<float, EPI>(p, after_quantize, s);
        case VLB_DTYPE_F16: return linear_type<__half, EPI>(p, after_quantize, s);
        case VLB_DTYPE_BF16: return linear_type<__nv_bfloat16, EPI>(p, after_quantize, s);
        default: return cudaErrorInvalidValue;
    }
}
cudaError_t launch_int8_linear(const Int8ActParams& p, int y_type, bool after_quantize, cudaStream_t s) {
    return p.act == kInt8NoEpilogue ? linear_typed<false>(p, y_type, after_quantize, s)
                                    : linear_typed<true>(p, y_type, after_quantize, s);
}

}  // namespace vlb
