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
#include "vlb_math.cuh"
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
constexpr uint32_t kBalCluster = 8, kBalParts = 16;  // most blocks of a counting cluster, parts of a sequence
constexpr uint32_t kBalSeqs = 512;                  // offsets held in shared memory

// The first sequence that ends after token t (S: none does).
__device__ __forceinline__ uint32_t sequence_after(const uint32_t* offsets, uint32_t S, uint32_t t) {
    uint32_t lo = 0, hi = S;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2u;
        if (offsets[mid + 1] > t) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}
// The offsets from shared memory where they fit (a search in memory is one round trip a step).
__device__ __forceinline__ const uint32_t* near_offsets(const BalanceParams& p, uint32_t* shared) {
    if (!p.seq_offsets || p.S > kBalSeqs) return p.seq_offsets;
    for (uint32_t s = threadIdx.x; s <= p.S; s += kBalThreads) shared[s] = p.seq_offsets[s];
    __syncthreads();
    return shared;
}

// Adds the routes of the live tokens in [lo, hi) to hist[E] (shared), and the live tokens to hist[E]'s
// next entry: 16 bytes of routes a load, four loads a thread in flight.
__device__ __forceinline__ void count_routes(const BalanceParams& p, uint32_t lo, uint32_t hi, uint32_t* hist) {
    const uint32_t tid = threadIdx.x;
    uint32_t live = 0;
    if (p.mask)
        for (uint32_t t = lo + tid; t < hi; t += blockDim.x) live += p.mask[t] != 0;
    else if (tid == 0)
        live = hi - lo;
    live = __reduce_add_sync(0xffffffffu, live);
    if ((tid & 31u) == 0 && live) atomicAdd(hist + p.E, live);
    // the expert of pair i, or E when its token is not live
    const auto live_expert = [&](uint32_t i, uint32_t e) { return !p.mask || p.mask[i / p.k] ? e : p.E; };
    const auto add = [&](uint32_t e) {
        if (e < p.E) atomicAdd(hist + e, 1u);
    };
    const uint32_t first = lo * p.k, end = hi * p.k;
    const uint32_t head = min((4u - (uint32_t)(reinterpret_cast<uintptr_t>(p.idx + first) / 4u) % 4u) % 4u, end - first);
    const uint32_t body = first + head, quads = (end - body) / 4u, tail = body + 4u * quads;
    if (tid < head) add(live_expert(first + tid, p.idx[first + tid]));
    if (tid < end - tail) add(live_expert(tail + tid, p.idx[tail + tid]));
    const uint4* q = reinterpret_cast<const uint4*>(p.idx + body);
    for (uint32_t i0 = tid; i0 < quads; i0 += 4u * blockDim.x) {
        uint4 v[4];
#pragma unroll
        for (uint32_t u = 0; u < 4u; ++u)
            if (i0 + u * blockDim.x < quads) v[u] = __ldg(q + i0 + u * blockDim.x);
        if (p.mask) {
#pragma unroll
            for (uint32_t u = 0; u < 4u; ++u) {
                const uint32_t i = i0 + u * blockDim.x, at = body + 4u * i;
                if (i < quads)
                    v[u] = make_uint4(live_expert(at, v[u].x), live_expert(at + 1u, v[u].y), live_expert(at + 2u, v[u].z),
                                      live_expert(at + 3u, v[u].w));
            }
        }
#pragma unroll
        for (uint32_t u = 0; u < 4u; ++u) {
            if (i0 + u * blockDim.x >= quads) break;
            add(v[u].x);
            add(v[u].y);
            add(v[u].z);
            add(v[u].w);
        }
    }
}

// Block b counts piece b mod 2^log_pieces of sequence b >> log_pieces; the blocks of a cluster add theirs through
// distributed shared memory to one part: E counts and, behind them, the live tokens.
__global__ void __launch_bounds__(kBalThreads) balance_count_kernel(const BalanceParams p, uint32_t log_pieces, uint32_t cluster) {
    __shared__ uint32_t hist[513], foreign, offsets_s[kBalSeqs + 1];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    const uint32_t tid = threadIdx.x, s = blockIdx.x >> log_pieces;
    const uint32_t piece = blockIdx.x & ((1u << log_pieces) - 1u);
    uint32_t lo = 0, hi = p.T;
    if (p.seq_offsets) lo = min(p.seq_offsets[s], p.T), hi = max(lo, min(p.seq_offsets[s + 1], p.T));
    const uint32_t* offsets = near_offsets(p, offsets_s);
    for (uint32_t e = tid; e <= p.E; e += kBalThreads) hist[e] = 0;
    if (tid == 0) foreign = 0;
    if (blockIdx.x == 0 && tid == 0) *p.ticket = 0;
    const uint32_t from = lo + (uint32_t)(((uint64_t)(hi - lo) * piece) >> log_pieces);
    const uint32_t to = lo + (uint32_t)(((uint64_t)(hi - lo) * (piece + 1u)) >> log_pieces);
    __syncthreads();
    if ((tid == 0 || tid == 32u) && offsets && from < to) {
        // offsets that fall are outside the contract; a range whose ends another sequence holds counts
        // as empty, so that no count passes the tokens' pairs
        const uint32_t t = tid ? to - 1u : from;
        if (sequence_after(offsets, p.S, t) != s || offsets[s] > t) foreign = 1;
    }
    count_routes(p, from, to, hist);
    __syncthreads();
    if (foreign)
        for (uint32_t e = tid; e <= p.E; e += kBalThreads) hist[e] = 0;
    uint32_t* out = p.part + (size_t)(blockIdx.x / cluster) * (p.E + 1u);
    if (cluster == 1u) {
        for (uint32_t e = tid; e <= p.E; e += kBalThreads) out[e] = hist[e];  // entries this thread zeroed, or summed by all
        return;
    }
    tc::cluster_sync();
    const uint32_t base = tc::smem_u32(hist);
    for (uint32_t e = tc::cluster_rank() * kBalThreads + tid; e <= p.E; e += cluster * kBalThreads) {
        uint32_t v[kBalCluster], sum = 0;
#pragma unroll
        for (uint32_t r = 0; r < kBalCluster; ++r) v[r] = r < cluster ? tc::cluster_ld(base + e * 4u, r) : 0u;
#pragma unroll
        for (uint32_t r = 0; r < kBalCluster; ++r) sum += v[r];
        out[e] = sum;
    }
    tc::cluster_sync();  // no block leaves while its counts are read
}

// Entry e of sequence s (e == E: its live tokens), summed over the parts.
__device__ __forceinline__ uint32_t part_sum(const BalanceParams& p, uint32_t s, uint32_t e) {
    const uint32_t* at = p.part + (size_t)s * p.parts * (p.E + 1u) + e;
    uint32_t v[kBalParts], sum = 0;
#pragma unroll
    for (uint32_t i = 0; i < kBalParts; ++i) v[i] = i < p.parts ? at[(size_t)i * (p.E + 1u)] : 0u;
#pragma unroll
    for (uint32_t i = 0; i < kBalParts; ++i) sum += v[i];
    return sum;
}

// e^x for any x <= 0 (-inf: 0; a NaN stays).
__device__ __forceinline__ float exp_low(float x) { return x < -1000.f ? 0.f : fast_exp(x); }

// log(1 + e) / 2 for e in [0, 1] as artanh(e / (2 + e)): the series' next term is below 2^-26 of it,
// and small e keep their bits.
__device__ __forceinline__ float half_log1p(float e) {
    const float s = e * fast_rcp(2.f + e), q = s * s;
    float v = fmaf(q, 1.f / 13.f, 1.f / 11.f);
    v = fmaf(q, v, 1.f / 9.f);
    v = fmaf(q, v, 1.f / 7.f);
    v = fmaf(q, v, 1.f / 5.f);
    v = fmaf(q, v, 1.f / 3.f);
    return fmaf(s * q, v, s);
}

// u(z) / U and u(z) r(z) / U, U a power that only depends on m = min(0, largest z) (softmax: m the
// largest z): with it taken out the sums stay normal numbers however low a row's logits are.
// PLAIN: m is 0 and every z is in (-80, 900), as in nearly every row.
template <int SCORE, bool PLAIN>
__device__ __forceinline__ void balance_score(float z, float m, float& u, float& ur) {
    if (SCORE == VLB_SCORE_SOFTMAX) {
        u = exp_low(z - m);
        ur = u;
    } else if (SCORE == VLB_SCORE_SIGMOID && PLAIN) {
        const float t = fast_exp(-z);  // below e^80; r = 1 - u = t u
        u = fast_rcp(1.f + t);
        ur = t * u * u;
    } else if (SCORE == VLB_SCORE_SIGMOID) {
        const float e = exp_low(-fabsf(z)), d = fast_rcp(1.f + e);
        u = z > 0.f ? d : exp_low(z - m) * d;
        ur = u * (z > 0.f ? e * d : d);
    } else {
        const float e = PLAIN ? fast_exp(-fabsf(z)) : exp_low(-fabsf(z)), d = fast_rcp(1.f + e);
        if (PLAIN || z > 0.f) {
            const float soft = fmaf(2.f, half_log1p(e), fmaxf(z, 0.f)), root = fast_rsqrt(soft);
            u = soft * root;
            ur = (z > 0.f ? 0.5f : 0.5f * e) * d * root;
        } else {
            // softplus(z) = e^z q
            const float q = e > 1e-30f ? 2.f * half_log1p(e) * fast_rcp(e) : 1.f, root = fast_rsqrt(q);
            const float x = exp_low(0.5f * (z - m));
            u = q * root * x;
            ur = 0.5f * d * root * x;
        }
    }
}

// The rare rows' scores out of line: unrolled beside the others they would double the code every
// block first has to fetch.
template <int SCORE>
__device__ __noinline__ float2 balance_score_rare(float z, float m) {
    float2 v;
    balance_score<SCORE, false>(z, m, v.x, v.y);
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

template <typename T, uint32_t NV, uint32_t VEC, bool FULL>
struct BalRow {
    BalVec<T, VEC> v[NV / VEC];
    bool live;
    // A row that is not live is not read: its memory may not be there.
    __device__ __forceinline__ void load(const BalanceParams& p, uint32_t t, bool is_live) {
        live = is_live;
        if (!live) return;
        const T* z = static_cast<const T*>(p.logits) + (size_t)t * p.stride;
#pragma unroll
        for (uint32_t j = 0; j < NV; j += VEC) {
            const uint32_t e = expert_of<VEC>(threadIdx.x & 31u, j);
            if (FULL || e < p.E) v[j / VEC] = *reinterpret_cast<const BalVec<T, VEC>*>(z + e);
        }
    }
};

// One token by a warp: returns weight * d_t and writes the row's gradient.
template <typename T, int SCORE, uint32_t NV, uint32_t VEC, bool FULL>
__device__ __forceinline__ float balance_row(const BalanceParams& p, const BalRow<T, NV, VEC, FULL>& row, uint32_t t,
                                             const float (&f)[NV], float weight, float up) {
    const uint32_t lane = threadIdx.x & 31u;
    float u[NV], ur[NV];
    float m = -INFINITY;
    bool deep = false;
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) {
        const bool in = FULL || expert_of<VEC>(lane, j) < p.E;
        u[j] = in ? bl_float(row.v[j / VEC].v[j % VEC]) : SCORE == VLB_SCORE_SOFTMAX ? -INFINITY : -79.f;
        if (SCORE != VLB_SCORE_SOFTMAX) deep |= u[j] < -80.f;
        if (in) m = fmaxf(m, u[j]);
    }
    // (a place past the experts passes as -79: its score, under 2^-56 of the sum, leaves it as it is)
    const bool zero = SCORE != VLB_SCORE_SOFTMAX && __any_sync(0xffffffffu, m >= 0.f);
    const bool plain = zero && !__any_sync(0xffffffffu, deep || m > 900.f);
    bool none = false;
    if (zero) m = 0.f;
    if (!plain) {
        if (SCORE != VLB_SCORE_SOFTMAX) {
#pragma unroll
            for (uint32_t j = 0; j < NV; ++j)
                if (!FULL && expert_of<VEC>(lane, j) >= p.E) u[j] = -INFINITY;
        }
        if (!zero) m = warp_max(m);
        if (m == -INFINITY) {
            // no expert left by the row's mask: it adds nothing and gets no gradient; but a row
            // that holds a NaN is no such row
            bool nan = false;
#pragma unroll
            for (uint32_t j = 0; j < NV; ++j) nan |= u[j] != u[j];
            none = !__any_sync(0xffffffffu, nan);
            m = 0.f;  // its scores come out as 0
        }
    }
    float total = 0.f, dot = 0.f;
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) {
        const float zj = u[j];  // -inf (masked) scores 0
        if (SCORE == VLB_SCORE_SOFTMAX || plain) {
            balance_score<SCORE, true>(zj, m, u[j], ur[j]);
        } else {
            const float2 v = balance_score_rare<SCORE>(zj, m);
            u[j] = v.x;
            ur[j] = v.y;
        }
        total += u[j];
        dot = fmaf(u[j], f[j], dot);
    }
    // both sums at once: the lower half of the warp goes on with one, the upper with the other
    float half = (lane & 16u ? dot : total) + __shfl_xor_sync(0xffffffffu, lane & 16u ? total : dot, 16);
#pragma unroll
    for (int o = 8; o; o >>= 1) half += __shfl_xor_sync(0xffffffffu, half, o);
    total = __shfl_sync(0xffffffffu, half, 0);
    dot = __shfl_sync(0xffffffffu, half, 16);
    const float inv = none ? 0.f : fast_rcp(total), d = dot * inv;
    if (p.dlogits) {
        T* grad = static_cast<T*>(p.dlogits) + (size_t)t * p.grad_stride;
        const float gw = up * weight * inv, gd = gw * d;
#pragma unroll
        for (uint32_t j = 0; j < NV; j += VEC) {
            const uint32_t e = expert_of<VEC>(lane, j);
            BalVec<T, VEC> v;
#pragma unroll
            for (uint32_t i = 0; i < VEC; ++i) bl_set(v.v[i], ur[j + i] * fmaf(gw, f[j + i], -gd));
            if (FULL || e < p.E) *reinterpret_cast<BalVec<T, VEC>*>(grad + e) = v;
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

// A block takes a run of tokens, sequence by sequence; a warp reads its next row while it works on
// one, if that row is live. ONE: one block is the whole call, with one sequence, and counts for itself.
template <typename T, int SCORE, uint32_t NV, uint32_t VEC, bool FULL, bool ONE>
__global__ void __launch_bounds__(kBalThreads, NV > 8 ? 1 : 2) balance_kernel(const BalanceParams p) {
    __shared__ uint32_t hist[513], alive_s, offsets_s[kBalSeqs + 1];
    __shared__ double part[kBalWarps];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const uint32_t t0 = (uint32_t)((uint64_t)p.T * blockIdx.x / gridDim.x);
    const uint32_t t1 = (uint32_t)((uint64_t)p.T * (blockIdx.x + 1u) / gridDim.x);
    if (ONE) tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    // A token is live when the mask has it and some sequence holds it: [first, past), as the offsets
    // do not fall. `ahead`: whether the token after the one in `row` is, read a row early so that a
    // row's load waits for no flag.
    uint32_t first = 0, past = t1;
    if (p.seq_offsets) first = p.seq_offsets[0], past = min(t1, p.seq_offsets[p.S]);
    const auto is_live = [&](uint32_t t) { return t >= first && t < past && (!p.mask || p.mask[t]); };
    BalRow<T, NV, VEC, FULL> row;
    row.load(p, t0 + warp, is_live(t0 + warp));  // on its way while the counts are taken
    bool ahead = is_live(t0 + warp + kBalWarps);
    const uint32_t* offsets = near_offsets(p, offsets_s);
    if (tid == 0) alive_s = 0;
    if (ONE)
        for (uint32_t e = tid; e <= p.E; e += kBalThreads) hist[e] = 0;
    const float up = p.upstream ? *p.upstream : 1.f;
    // [t, end): tokens of sequence s, or of none
    uint32_t s = 0, end = t1;
    bool held = true;
    const auto segment = [&](uint32_t t) {
        if (!offsets) return;
        s = sequence_after(offsets, p.S, t);
        held = s < p.S && offsets[s] <= t;
        end = held ? min(t1, offsets[s + 1]) : s < p.S ? min(t1, offsets[s]) : t1;
    };
    // Counts in one part (short sequences): each warp takes its tokens' from memory when it meets a
    // new sequence. In several: the block adds them up in shared memory, a sequence at a time.
    const bool by_warp = !ONE && p.parts == 1u;
    const auto fetch_counts = [&] {
        if (held)
            for (uint32_t e = tid; e <= p.E; e += kBalThreads) hist[e] = part_sum(p, s, e);
    };
    if (t0 < t1 && !by_warp) segment(t0);
    if (!ONE) tc::grid_dependency_wait();
    __syncthreads();
    if (ONE) {
        uint32_t lo = 0, hi = p.T;
        if (offsets) lo = min(offsets[0], p.T), hi = max(lo, min(offsets[1], p.T));
        count_routes(p, lo, hi, hist);
    } else {
        uint32_t with = 0;  // sequences with a live token
        for (uint32_t i = tid; i < p.S; i += kBalThreads) with += part_sum(p, i, p.E) != 0;
        if (t0 < t1 && !by_warp) fetch_counts();
        // the counts' own output, the sequences dealt over the blocks
        for (uint32_t i = blockIdx.x; i < p.S; i += gridDim.x)
            for (uint32_t e = tid; e < p.E; e += kBalThreads) p.counts[(size_t)i * p.E + e] = part_sum(p, i, e);
        with = __reduce_add_sync(0xffffffffu, with);
        if (lane == 0 && with) atomicAdd(&alive_s, with);
    }
    __syncthreads();
    const uint32_t alive = ONE ? hist[p.E] != 0 : alive_s;
    const float base = alive ? p.coefficient / (float)alive : 0.f;
    double sum = 0.0;
    uint32_t mine = t0 + warp;  // this warp's next token, its logits in `row`
    float weight = 0.f, f[NV];
    const auto shares = [&](const uint32_t* counts) {
        const uint32_t n = counts[p.E];
        weight = n ? base / (float)n : 0.f;
        const float scale = n ? (float)p.E / ((float)p.k * (float)n) : 0.f;
#pragma unroll
        for (uint32_t j = 0; j < NV; ++j) {
            const uint32_t e = expert_of<VEC>(lane, j);
            f[j] = FULL || e < p.E ? (float)counts[e] * scale : 0.f;
        }
    };
    const auto next_token = [&] {
        const uint32_t r = mine;
        const BalRow<T, NV, VEC, FULL> now = row;
        mine += kBalWarps;
        row.load(p, mine, ahead);
        ahead = is_live(mine + kBalWarps);
        if (held && now.live) sum += (double)balance_row<T, SCORE, NV, VEC, FULL>(p, now, r, f, weight, up);
        else clear_row<T, NV, VEC>(p, r);
    };
    if (by_warp) {
        for (uint32_t upto = t0; mine < t1; next_token()) {
            if (mine < upto) continue;
            segment(mine);
            upto = end;
            if (held) shares(p.part + (size_t)s * (p.E + 1u));
        }
    } else {
        for (uint32_t t = t0; t < t1;) {
            if (held) shares(hist);
            while (mine < end) next_token();
            t = end;
            if (t >= t1) break;
            __syncthreads();  // hist is read by all
            segment(t);
            if (!ONE) fetch_counts();
            __syncthreads();
        }
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

// Blocks that count a sequence, a power of two: about 128 in all, but none for less than 256 tokens.
uint32_t balance_pieces(uint32_t T, uint32_t S) {
    uint32_t n = 1;
    while (n < kBalCluster * kBalParts && n * S < 128u && n * S * 256u < T) n *= 2u;
    return n;
}

template <typename T, int SCORE, uint32_t NV, uint32_t VEC, bool FULL>
cudaError_t balance_launch(const BalanceParams& p, cudaStream_t s) {
    if (p.S == 1 && p.T <= kBalOneTokens)
        return launch_chained(balance_kernel<T, SCORE, NV, VEC, FULL, true>, dim3(1), kBalThreads, 0, 0, s, p);
    const uint32_t pieces = balance_pieces(p.T, p.S), log_pieces = (uint32_t)__builtin_ctz(pieces);
    const uint32_t cluster = pieces / balance_parts(p.T, p.S);
    const cudaError_t e = launch_chained(balance_count_kernel, dim3(p.S * pieces), kBalThreads, 0, cluster, s, p, log_pieces, cluster);
    if (e != cudaSuccess) return e;
    const uint32_t want = (p.T + kBalWarps - 1u) / kBalWarps;
    const uint32_t blocks = want < 1u ? 1u : want < kBalanceBlocks ? want : kBalanceBlocks;
    return launch_chained(balance_kernel<T, SCORE, NV, VEC, FULL, false>, dim3(blocks), kBalThreads, 0, 0, s, p);
}

// NV: values of a row a lane holds; VEC: neighbours it loads at once, 1 where the rows do not start
// on such a boundary; FULL: the row fills the warp's values (64 to 512 experts by powers of two), no
// place is checked.
template <typename T, int SCORE>
cudaError_t balance_scored(const BalanceParams& p, cudaStream_t s) {
    const auto fits = [&](uint32_t n) {
        const auto on = [&](const void* at) { return reinterpret_cast<uintptr_t>(at) % (n * sizeof(T)) == 0; };
        return p.E % n == 0 && p.stride % n == 0 && p.grad_stride % n == 0 && on(p.logits) && on(p.dlogits);
    };
    constexpr uint32_t V = 16u / sizeof(T);
    if (p.E == 64u && fits(2)) return balance_launch<T, SCORE, 2, 2, true>(p, s);
    if (p.E == 128u && fits(4)) return balance_launch<T, SCORE, 4, 4, true>(p, s);
    if (p.E == 256u && fits(V)) return balance_launch<T, SCORE, 8, V, true>(p, s);
    if (p.E == 512u && fits(V)) return balance_launch<T, SCORE, 16, V, true>(p, s);
    if (p.E <= 64u)
        return fits(2) ? balance_launch<T, SCORE, 2, 2, false>(p, s) : balance_launch<T, SCORE, 2, 1, false>(p, s);
    if (p.E <= 256u)
        return fits(V) ? balance_launch<T, SCORE, 8, V, false>(p, s) : balance_launch<T, SCORE, 8, 1, false>(p, s);
    return fits(V) ? balance_launch<T, SCORE, 16, V, false>(p, s) : balance_launch<T, SCORE, 16, 1, false>(p, s);
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

uint32_t balance_parts(uint32_t T, uint32_t S) {
    const uint32_t pieces = balance_pieces(T, S);
    return pieces <= kBalParts ? pieces : pieces / kBalCluster;
}

// Parts of all sequences that any call of at most T tokens in at most S sequences has: it never falls
// as T or S rise, though balance_parts does where clusters begin. With n = balance_pieces > 1 pieces a
// sequence, half of them were too few: n / 2 * S < 128 and n / 2 * S < T / 256.
uint64_t balance_parts_bound(uint32_t T, uint32_t S) {
    const uint64_t tokens = ((uint64_t)T + 255u) / 256u, q = tokens < 128u ? tokens : 128u;
    const uint64_t pieces = q > 1u ? 2u * (q - 1u) : 0u, most = (uint64_t)S * kBalParts;
    const uint64_t split = pieces < most ? pieces : most;
    return split > S ? split : S;
}

cudaError_t launch_balance(const BalanceParams& p, cudaStream_t s) {
    switch (p.logits_type) {
        case VLB_DTYPE_F32: return balance_typed<float>(p, s);
        case VLB_DTYPE_F16: return balance_typed<__half>(p, s);
        default: return balance_typed<__nv_bfloat16>(p, s);
    }
}

}  // namespace vlb
