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
// The counts carry no gradient, so they are taken first (they read the routes alone) and one pass
// over the logits then gives both the loss (the sum of d_t) and the gradient: HBM-bound, logits
// read once and gradient written once. Two launches: each sequence's routes are counted in parts,
// without atomics on memory or zeroed buffers; the blocks of the second kernel sum the parts they
// need, take tokens warp by warp with a row in registers, and the last block adds the blocks' losses
// in a fixed order. Calls of few tokens take one launch of one block. The reference routes only (it
// does not train): the scores are its routers' (deepseek_v4_reference.cpp:65-69,
// olmoe_runtime.cpp:1120-1137).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "vlb_launch.h"
#include "vlb_tcgen05.cuh"

namespace vlb {
namespace {

template <typename T>
__device__ __forceinline__ float bl_float(T v);
template <>
__device__ __forceinline__ float bl_float(float v) {
    return v;
}
template <>
__device__ __forceinline__ float bl_float(__half v) {
    return __half2float(v);
}
template <>
__device__ __forceinline__ float bl_float(__nv_bfloat16 v) {
    return __bfloat162float(v);
}
__device__ __forceinline__ void bl_set(float& p, float v) { p = v; }
__device__ __forceinline__ void bl_set(__half& p, float v) { p = __float2half_rn(v); }
__device__ __forceinline__ void bl_set(__nv_bfloat16& p, float v) { p = __float2bfloat16_rn(v); }

constexpr uint32_t kBalThreads = 512, kBalWarps = kBalThreads / 32u;

// The first sequence that ends after token t (S: none does).
__device__ __forceinline__ uint32_t sequence_after(const BalanceParams& p, uint32_t t) {
    if (!p.seq_offsets) return 0;
    uint32_t lo = 0, hi = p.S;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2u;
        if (p.seq_offsets[mid + 1] > t) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}
// Whether sequence s holds token t.
__device__ __forceinline__ bool holds(const BalanceParams& p, uint32_t s, uint32_t t) {
    return sequence_after(p, t) == s && (!p.seq_offsets || p.seq_offsets[s] <= t);
}

// Adds the routes of the live tokens in [lo, hi) to hist[E] (shared) and returns this thread's
// share of the live tokens.
__device__ __forceinline__ uint32_t count_routes(const BalanceParams& p, uint32_t lo, uint32_t hi, uint32_t* hist) {
    uint32_t live = 0;
    for (uint32_t t = lo + threadIdx.x; t < hi; t += blockDim.x) live += !p.mask || p.mask[t];
    const uint32_t end = hi * p.k;
    for (uint32_t i = lo * p.k + threadIdx.x; i < end; i += blockDim.x) {
        const uint32_t e = p.idx[i];
        if (e < p.E && (!p.mask || p.mask[i / p.k])) atomicAdd(hist + e, 1u);
    }
    return live;
}

// Part blockIdx.x % parts of sequence blockIdx.x / parts: its counts and, behind them, its live tokens.
__global__ void __launch_bounds__(kBalThreads) balance_count_kernel(const BalanceParams p) {
    __shared__ uint32_t hist[512], range[2], live_s;
    tc::grid_launch_dependents();
    const uint32_t tid = threadIdx.x, s = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
    for (uint32_t e = tid; e < p.E; e += kBalThreads) hist[e] = 0;
    if (tid == 0) {
        uint32_t lo = 0, hi = p.T;
        if (p.seq_offsets) lo = min(p.seq_offsets[s], p.T), hi = max(lo, min(p.seq_offsets[s + 1], p.T));
        const uint32_t from = lo + (uint32_t)((uint64_t)(hi - lo) * part / p.parts);
        const uint32_t to = lo + (uint32_t)((uint64_t)(hi - lo) * (part + 1u) / p.parts);
        // offsets that fall: a range whose ends another sequence holds is empty
        const bool ours = from < to && holds(p, s, from) && holds(p, s, to - 1u);
        range[0] = from;
        range[1] = ours ? to : from;
        live_s = 0;
        if (blockIdx.x == 0) *p.ticket = 0;
    }
    __syncthreads();
    const uint32_t live = __reduce_add_sync(0xffffffffu, count_routes(p, range[0], range[1], hist));
    if ((tid & 31u) == 0 && live) atomicAdd(&live_s, live);
    __syncthreads();
    uint32_t* out = p.part + (size_t)blockIdx.x * (p.E + 1u);
    for (uint32_t e = tid; e < p.E; e += kBalThreads) out[e] = hist[e];
    if (tid == 0) out[p.E] = live_s;
}

// Entry e of sequence s (e == E: its live tokens), summed over the parts.
__device__ __forceinline__ uint32_t part_sum(const BalanceParams& p, uint32_t s, uint32_t e) {
    const uint32_t* at = p.part + (size_t)s * p.parts * (p.E + 1u) + e;
    uint32_t sum = 0;
#pragma unroll 8
    for (uint32_t i = 0; i < p.parts; ++i) sum += at[(size_t)i * (p.E + 1u)];
    return sum;
}

// log(1 + e) for e in [0, 1] as 2 artanh(e / (2 + e)): the series' next term is below 2^-26 of it,
// and small e keep their bits.
__device__ __forceinline__ float log1p_unit(float e) {
    const float s = __fdividef(e, 2.f + e), q = s * s;
    float v = fmaf(q, 1.f / 13.f, 1.f / 11.f);
    v = fmaf(q, v, 1.f / 9.f);
    v = fmaf(q, v, 1.f / 7.f);
    v = fmaf(q, v, 1.f / 5.f);
    v = fmaf(q, v, 1.f / 3.f);
    return 2.f * fmaf(s * q, v, s);
}

// u(z) / U and u(z) r(z) / U, U a power that only depends on m = min(0, largest z) (softmax: m the
// largest z): with it taken out the sums stay normal numbers however low a row's logits are.
// ZERO: m is 0, as in every row with a logit that is not negative.
template <int SCORE, bool ZERO>
__device__ __forceinline__ void balance_score(float z, float m, float& u, float& ur) {
    if (SCORE == VLB_SCORE_SOFTMAX) {
        u = expf(z - m);
        ur = u;
        return;
    }
    const float e = expf(-fabsf(z)), d = __fdividef(1.f, 1.f + e);
    if (SCORE == VLB_SCORE_SIGMOID) {
        const float low = ZERO ? e : expf(z - m);  // of a negative z; without ZERO all are
        u = (ZERO && z > 0.f ? 1.f : low) * d;
        ur = u * (z > 0.f ? e * d : d);
    } else if (ZERO && z > -80.f) {
        const float soft = fmaxf(z, 0.f) + log1p_unit(e), root = rsqrtf(soft);
        u = soft * root;
        ur = 0.5f * (z > 0.f ? d : e * d) * root;
    } else {
        // softplus(z) = e^z q
        const float q = e > 1e-30f ? __fdividef(log1p_unit(e), e) : 1.f, root = rsqrtf(q), x = expf(0.5f * (z - m));
        u = q * root * x;
        ur = 0.5f * d * root * x;
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

template <typename T, uint32_t VEC>
struct alignas(sizeof(T) * VEC) BalVec {
    T v[VEC];
};

// Expert of value j of a lane: runs of VEC neighbours.
template <uint32_t VEC>
__device__ __forceinline__ uint32_t expert_of(uint32_t lane, uint32_t j) {
    return (j / VEC) * (32u * VEC) + lane * VEC + j % VEC;
}

// One token by a warp: returns weight * d_t and writes the row's gradient.
template <typename T, int SCORE, uint32_t NV, uint32_t VEC>
__device__ __forceinline__ float balance_row(const BalanceParams& p, uint32_t t, const float (&f)[NV], float weight,
                                             float up) {
    const uint32_t lane = threadIdx.x & 31u;
    const T* z = static_cast<const T*>(p.logits) + (size_t)t * p.stride;
    float u[NV], ur[NV];
    float m = -INFINITY;
#pragma unroll
    for (uint32_t j = 0; j < NV; j += VEC) {
        const uint32_t e = expert_of<VEC>(lane, j);
        if (e < p.E) {
            const BalVec<T, VEC> v = *reinterpret_cast<const BalVec<T, VEC>*>(z + e);
#pragma unroll
            for (uint32_t i = 0; i < VEC; ++i) u[j + i] = bl_float(v.v[i]);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < VEC; ++i) u[j + i] = -INFINITY;
        }
#pragma unroll
        for (uint32_t i = 0; i < VEC; ++i) m = fmaxf(m, u[j + i]);
    }
    const bool zero = SCORE != VLB_SCORE_SOFTMAX && __any_sync(0xffffffffu, m >= 0.f);
    bool none = false;
    if (zero) {
        m = 0.f;
    } else {
        m = warp_max(m);
        if (m == -INFINITY) {
            // no expert left by the row's mask: it adds nothing and gets no gradient; but a row
            // that holds a NaN is no such row
            bool nan = false;
#pragma unroll
            for (uint32_t j = 0; j < NV; ++j) nan |= u[j] != u[j];
            none = !__any_sync(0xffffffffu, nan);
        }
    }
    float total = 0.f, dot = 0.f;
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) {
        const float zj = u[j];
        if (expert_of<VEC>(lane, j) >= p.E || none) u[j] = ur[j] = 0.f;
        else if (zero) balance_score<SCORE, true>(zj, 0.f, u[j], ur[j]);
        else balance_score<SCORE, false>(zj, m, u[j], ur[j]);
        total += u[j];
        dot = fmaf(u[j], f[j], dot);
    }
    total = warp_sum(total);
    dot = warp_sum(dot);
    const float inv = none ? 0.f : 1.f / total, d = dot * inv;
    if (p.dlogits) {
        T* grad = static_cast<T*>(p.dlogits) + (size_t)t * p.grad_stride;
        const float gw = up * weight * inv;
#pragma unroll
        for (uint32_t j = 0; j < NV; j += VEC) {
            const uint32_t e = expert_of<VEC>(lane, j);
            BalVec<T, VEC> v;
#pragma unroll
            for (uint32_t i = 0; i < VEC; ++i) bl_set(v.v[i], gw * ur[j + i] * (f[j + i] - d));
            if (e < p.E) *reinterpret_cast<BalVec<T, VEC>*>(grad + e) = v;
        }
    }
    return weight * d;
}

template <typename T, uint32_t NV, uint32_t VEC>
__device__ __forceinline__ void clear_row(const BalanceParams& p, uint32_t t) {
    if (!p.dlogits) return;
    T* grad = static_cast<T*>(p.dlogits) + (size_t)t * p.grad_stride;
    BalVec<T, VEC> v;
#pragma unroll
    for (uint32_t i = 0; i < VEC; ++i) bl_set(v.v[i], 0.f);
#pragma unroll
    for (uint32_t j = 0; j < NV; j += VEC) {
        const uint32_t e = expert_of<VEC>(threadIdx.x & 31u, j);
        if (e < p.E) *reinterpret_cast<BalVec<T, VEC>*>(grad + e) = v;
    }
}

// A block takes a run of tokens, sequence by sequence. ONE: one block is the whole call, with one
// sequence, and counts for itself.
template <typename T, int SCORE, uint32_t NV, uint32_t VEC, bool ONE>
__global__ void __launch_bounds__(kBalThreads) balance_kernel(const BalanceParams p) {
    __shared__ float f_s[512];
    __shared__ uint32_t hist[512], word[2];
    __shared__ double part[kBalWarps];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    if (!ONE) tc::grid_dependency_wait();
    if (tid < 2u) word[tid] = 0;
    if (ONE)
        for (uint32_t e = tid; e < p.E; e += kBalThreads) hist[e] = 0;
    __syncthreads();
    // the sequences with a live token; ONE: the live tokens
    uint32_t mine = 0;
    if (ONE) {
        uint32_t lo = 0, hi = p.T;
        if (p.seq_offsets) lo = min(p.seq_offsets[0], p.T), hi = max(lo, min(p.seq_offsets[1], p.T));
        mine = count_routes(p, lo, hi, hist);
    } else {
        for (uint32_t s = tid; s < p.S; s += kBalThreads) mine += part_sum(p, s, p.E) != 0;
        // the counts' own output, the sequences dealt over the blocks
        for (uint32_t s = blockIdx.x; s < p.S; s += gridDim.x)
            for (uint32_t e = tid; e < p.E; e += kBalThreads) p.counts[(size_t)s * p.E + e] = part_sum(p, s, e);
    }
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0 && mine) atomicAdd(word, mine);
    __syncthreads();
    const float up = p.upstream ? *p.upstream : 1.f;
    const uint32_t alive = ONE ? word[0] != 0 : word[0];
    const float base = alive ? p.coefficient / (float)alive : 0.f;
    double sum = 0.0;
    const uint32_t t0 = (uint32_t)((uint64_t)p.T * blockIdx.x / gridDim.x);
    const uint32_t t1 = (uint32_t)((uint64_t)p.T * (blockIdx.x + 1u) / gridDim.x);
    for (uint32_t t = t0; t < t1;) {
        // [t, end): tokens of sequence s, or of none
        uint32_t s = 0, end = t1;
        bool held = true;
        if (p.seq_offsets) {
            s = sequence_after(p, t);
            if (s == p.S) held = false;
            else if (p.seq_offsets[s] > t) held = false, end = min(t1, p.seq_offsets[s]);
            else end = min(t1, p.seq_offsets[s + 1]);
        }
        float weight = 0.f, f[NV];
        if (held) {
            __syncthreads();
            if (!ONE && tid == 0) word[1] = part_sum(p, s, p.E);
            for (uint32_t e = tid; e < p.E; e += kBalThreads) f_s[e] = (float)(ONE ? hist[e] : part_sum(p, s, e));
            __syncthreads();
            const uint32_t n = ONE ? word[0] : word[1];
            weight = n ? base / (float)n : 0.f;
            const float scale = n ? (float)p.E / ((float)p.k * (float)n) : 0.f;
#pragma unroll
            for (uint32_t j = 0; j < NV; ++j) {
                const uint32_t e = expert_of<VEC>(lane, j);
                f[j] = e < p.E ? f_s[e] * scale : 0.f;
            }
        }
        for (uint32_t r = t + warp; r < end; r += kBalWarps) {
            if (held && (!p.mask || p.mask[r])) sum += (double)balance_row<T, SCORE, NV, VEC>(p, r, f, weight, up);
            else clear_row<T, NV, VEC>(p, r);
        }
        t = end;
    }
    if (ONE)
        for (uint32_t e = tid; e < p.E; e += kBalThreads) p.counts[e] = hist[e];
    if (!p.loss) return;
    if (lane == 0) part[warp] = sum;
    __syncthreads();
    if (warp != 0) return;
    double v = lane < kBalWarps ? part[lane] : 0.0;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (ONE) {
        if (lane == 0) *p.loss = (float)v;
        return;
    }
    uint32_t last = 0;
    if (lane == 0) {
        p.partial[blockIdx.x] = v;
        __threadfence();
        last = atomicAdd(p.ticket, 1u) == gridDim.x - 1u;
    }
    if (!__shfl_sync(0xffffffffu, last, 0)) return;
    __threadfence();
    v = 0.0;
    for (uint32_t i = lane; i < gridDim.x; i += 32u) v += __ldcg(p.partial + i);
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) *p.loss = (float)v;
}

template <typename T, int SCORE, uint32_t NV, uint32_t VEC>
cudaError_t balance_launch(const BalanceParams& p, cudaStream_t s) {
    if (p.S == 1 && p.T <= kBalOneTokens) {
        balance_kernel<T, SCORE, NV, VEC, true><<<1, kBalThreads, 0, s>>>(p);
        return cudaGetLastError();
    }
    balance_count_kernel<<<p.S * p.parts, kBalThreads, 0, s>>>(p);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const uint32_t want = (p.T + kBalWarps - 1u) / kBalWarps;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(want < 1u ? 1u : want < kBalanceBlocks ? want : kBalanceBlocks);
    cfg.blockDim = dim3(kBalThreads);
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, balance_kernel<T, SCORE, NV, VEC, false>, p);
}

// NV: values of a row a lane holds; VEC: neighbours it loads at once, 1 where the rows do not start
// on such a boundary.
template <typename T, int SCORE>
cudaError_t balance_scored(const BalanceParams& p, cudaStream_t s) {
    const auto fits = [&](uint32_t n) {
        const auto on = [&](const void* at) { return reinterpret_cast<uintptr_t>(at) % (n * sizeof(T)) == 0; };
        return p.E % n == 0 && p.stride % n == 0 && p.grad_stride % n == 0 && on(p.logits) && on(p.dlogits);
    };
    constexpr uint32_t V = 16u / sizeof(T);
    if (p.E <= 64u)
        return fits(2) ? balance_launch<T, SCORE, 2, 2>(p, s) : balance_launch<T, SCORE, 2, 1>(p, s);
    if (p.E <= 256u)
        return fits(V) ? balance_launch<T, SCORE, 8, V>(p, s) : balance_launch<T, SCORE, 8, 1>(p, s);
    return fits(V) ? balance_launch<T, SCORE, 16, V>(p, s) : balance_launch<T, SCORE, 16, 1>(p, s);
}

template <typename T>
cudaError_t balance_typed(const BalanceParams& p, cudaStream_t s) {
    switch (p.score) {
        case VLB_SCORE_SQRT_SOFTPLUS: return balance_scored<T, VLB_SCORE_SQRT_SOFTPLUS>(p, s);
        case VLB_SCORE_SIGMOID: return balance_scored<T, VLB_SCORE_SIGMOID>(p, s);
        default: return balance_scored<T, VLB_SCORE_SOFTMAX>(p, s);
    }
}

}  // namespace

// Parts a sequence's routes are counted in: enough blocks to fill the GPU when the sequences are few,
// few enough that the second kernel's blocks sum them in little time (64: 1 us at 256 experts).
uint32_t balance_parts(uint32_t T, uint32_t S) {
    const uint32_t by_seqs = S >= 64u ? 1u : 64u / S, by_tokens = T / 256u + 1u;
    return by_seqs < by_tokens ? by_seqs : by_tokens;
}

cudaError_t launch_balance(const BalanceParams& p, cudaStream_t s) {
    switch (p.logits_type) {
        case VLB_DTYPE_F32: return balance_typed<float>(p, s);
        case VLB_DTYPE_F16: return balance_typed<__half>(p, s);
        default: return balance_typed<__nv_bfloat16>(p, s);
    }
}

}  // namespace vlb
