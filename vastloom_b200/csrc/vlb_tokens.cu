// Tokens sorted by expert and back: the (token, slot) pairs of a route in the dispatch's stable order
// (expert, then token, then slot; deepseek_v4_graph.cpp:2134-2223), each pair's row, the weighted sum of
// a token's rows, and its gradient.
//
//   sort      a stable counting sort by expert: each block counts its pairs' experts; with all blocks' counts
//             every block finds its first place for every expert, and each pair takes its place by the
//             pairs of its expert before it in its block. Few pairs: one launch, every block counts all
//   rows      rows[place(t, s)] = x[t]
//   combine   out[t] = sum_s w_ts rows[place(t, s)] + residual[t]
//   gradient  drows[place(t, s)] = w_ts dout[t],  dw_ts = <dout[t], rows[place(t, s)]>
//
// The order costs a few bytes a pair; moving the rows is what takes the time, and HBM bounds that. Rows move
// in 16-byte pieces of the row that is written. Where a row that is read lies at another offset from a
// 16-byte boundary (rows of no whole pieces), a piece of it is two aligned loads and a shift.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "vlb_launch.h"
#include "vlb_rows.cuh"
#include "vlb_tcgen05.cuh"

namespace vlb {
namespace {

// ---- pieces of rows at any offset ------------------------------------------------------------------

// A piece of V elements from column c of a row on, as it is loaded: its own word, or SHIFTED the two aligned words it
// lies across. No branch, and the shift is left for later: the loads of many rows go out together. SHIFTED reads
// on both sides of it, less than 32 bytes.
template <uint32_t V, bool SHIFTED, typename E>
struct Raw {
    static constexpr uint32_t kBytes = V * sizeof(E), kWords = kBytes / 4u;
    static_assert(kBytes == 8u || kBytes == 16u, "a piece is one access");
    using Word = Pack<uint32_t, kWords>;
    Word x, y;
    // bytes from the aligned word before them that pieces of the row begin at, the same for all of them
    __device__ __forceinline__ static uint32_t shift_of(const E* row, int32_t c) {
        return SHIFTED ? (uint32_t)(reinterpret_cast<uintptr_t>(row + c) % kBytes) : 0u;
    }
    __device__ __forceinline__ void load(const E* row, int32_t c, uint32_t shift) {
        const Word* at = reinterpret_cast<const Word*>(reinterpret_cast<uintptr_t>(row + c) - shift);
        x = at[0];
        if constexpr (SHIFTED) y = at[1];
    }
    __device__ __forceinline__ Pack<E, V> get(uint32_t shift) const {
        Pack<E, V> a;
        if constexpr (!SHIFTED) {
            *reinterpret_cast<Word*>(&a) = x;
        } else {
            uint32_t w[2u * kWords];
#pragma unroll
            for (uint32_t i = 0; i < kWords; ++i) w[i] = x.v[i], w[kWords + i] = y.v[i];
#pragma unroll
            for (uint32_t i = 0; i + 1u < 2u * kWords; ++i) w[i] = shift & 4u ? w[i + 1u] : w[i];
            if constexpr (kWords == 4u) {
#pragma unroll
                for (uint32_t i = 0; i + 2u < 2u * kWords; ++i) w[i] = shift & 8u ? w[i + 2u] : w[i];
            }
#pragma unroll
            for (uint32_t i = 0; i < kWords; ++i)
                reinterpret_cast<uint32_t*>(&a)[i] = __funnelshift_r(w[i], w[i + 1u], (shift & 3u) * 8u);
        }
        return a;
    }
};
// A piece of 16 bytes or less, or two halves of 32 bytes.
template <uint32_t V, bool SHIFTED, typename E>
struct Piece {
    static constexpr uint32_t kParts = V * sizeof(E) > 16u ? 2u : 1u, kPart = V / kParts;
    using Part = Raw<kPart, SHIFTED, E>;
    Part part[kParts];
    __device__ __forceinline__ static uint32_t shift_of(const E* row, int32_t c) { return Part::shift_of(row, c); }
    __device__ __forceinline__ void load(const E* row, int32_t c, uint32_t shift) {
        if constexpr (kParts == 2u && !SHIFTED) {  // one access: two of 16 bytes would each take half of every sector
            uint32_t *a = part[0].x.v, *b = part[1].x.v;
            asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(b[0]), "=r"(b[1]), "=r"(b[2]), "=r"(b[3])
                         : "l"(row + c)
                         : "memory");
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kParts; ++i) part[i].load(row, c + (int32_t)(i * kPart), shift);
        }
    }
    __device__ __forceinline__ void get(uint32_t shift, float (&f)[V]) const {
#pragma unroll
        for (uint32_t i = 0; i < kParts; ++i) {
            float g[kPart];
            unpack(part[i].get(shift), g);
#pragma unroll
            for (uint32_t j = 0; j < kPart; ++j) f[i * kPart + j] = g[j];
        }
    }
};
// Adds w times the columns from c on, element by element: where a piece does not lie inside the rows.
template <uint32_t V, typename E>
__device__ __forceinline__ void add_each(float w, const E* row, int32_t c, uint32_t H, float (&acc)[V]) {
#pragma unroll
    for (uint32_t i = 0; i < V; ++i)
        if ((uint32_t)(c + (int32_t)i) < H) acc[i] = fmaf(w, to_float(row[c + (int32_t)i]), acc[i]);
}
// Whether Raw::load of every column of row r of n stays inside the rows: those before and behind take its reach.
template <uint32_t V, bool SHIFTED, typename E>
__device__ __forceinline__ bool inside_rows(uint32_t r, uint32_t n, size_t stride, uint32_t H) {
    if constexpr (SHIFTED) return r > 0 && r + 1u < n && stride * sizeof(E) >= 64u;
    else return H % V == 0 || (r + 1u < n && stride >= V);
}
// Elements of a row from the boundary of V before its first one to that.
template <uint32_t V, typename E>
__device__ __forceinline__ int32_t row_offset(const E* row) {
    return (int32_t)(reinterpret_cast<uintptr_t>(row) / sizeof(E) % V);
}

// ---- the order -------------------------------------------------------------------------------------

constexpr uint32_t kSortBlocks = 256;    // counting blocks at most
constexpr uint32_t kSelfPairs = 16384;  // up to here the counts cost more as a launch than again in every block
constexpr uint32_t kSortThreads = 512, kSortWarps = kSortThreads / 32u;

// The expert of pair i; E where it was dropped.
__device__ __forceinline__ uint32_t pair_expert(const SortParams& p, uint32_t i) {
    const uint32_t e = p.idx[i];
    return e < p.E && (!p.mask || p.mask[i / p.k]) ? e : p.E;
}
// What is written of pair i besides its row.
__device__ __forceinline__ void put_pair(const SortParams& p, uint32_t i, uint32_t place) {
    p.elem_row[i] = place;
    if (place == VLB_NO_ROW) return;
    const uint32_t t = i / p.k;
    if (p.row_index) p.row_index[place] = t;
    if (p.row_weight) p.row_weight[place] = p.weights[i];
    if (p.row_scale) p.row_scale[place] = p.x_scale[t];
}

// The sum over a block's values before each thread's, at most 1024 threads; warps: 32 words of shared memory.
__device__ __forceinline__ uint32_t sum_before(uint32_t v, uint32_t* warps) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    uint32_t upto = v;
#pragma unroll
    for (uint32_t d = 1; d < 32u; d <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += u;
    }
    if (lane == 31u) warps[warp] = upto;
    __syncthreads();
    uint32_t before = upto - v;
    for (uint32_t w = 0; w < warp; ++w) before += warps[w];
    __syncthreads();
    return before;
}

// counts[b][e] = pairs of block b (`each` neighbours, a multiple of kSortThreads) on expert e.
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const SortParams p, uint32_t each) {
    __shared__ uint32_t hist[kSortMaxExperts];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    const uint32_t n = p.T * p.k, lo = blockIdx.x * each, hi = min(n, lo + each);
    for (uint32_t e = threadIdx.x; e < p.E; e += kSortThreads) hist[e] = 0;
    __syncthreads();
    for (uint32_t i = lo + threadIdx.x; i < hi; i += kSortThreads) {
        const uint32_t e = pair_expert(p, i);
        if (e < p.E) atomicAdd(hist + e, 1u);
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < p.E; e += kSortThreads) p.counts[(size_t)blockIdx.x * p.E + e] = hist[e];
}

// (Every placing block adding up all counts itself took 24.8 us for 16,384 x 8 over 256 experts, with this launch 9.1.)
// counts[b][e] becomes the pairs on expert e of the blocks before b, totals[e] those of all. 32 experts a block, a warp
// a 32nd of the counting blocks.
__global__ void __launch_bounds__(1024) sort_prefix_kernel(const SortParams p, uint32_t blocks) {
    constexpr uint32_t kEach = kSortBlocks / 32u;
    __shared__ uint32_t sums[32][33];
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, e = blockIdx.x * 32u + lane, b0 = warp * kEach;
    uint32_t v[kEach], sum = 0;
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) v[i] = e < p.E && b0 + i < blocks ? p.counts[(size_t)(b0 + i) * p.E + e] : 0u;
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) sum += v[i];
    sums[warp][lane] = sum;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < 32u; ++w) {
        if (w < warp) before += sums[w][lane];
        all += sums[w][lane];
    }
    if (e >= p.E) return;
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
        if (b0 + i < blocks) p.counts[(size_t)(b0 + i) * p.E + e] = before;
        before += v[i];
    }
    if (warp == 0) p.totals[e] = all;
}

// Every pair's place and what goes there of it. SELF: without the counts, every block goes through all pairs. Shared:
// base[E] the block's next place on each expert, by_warp[kSortWarps][E] the warps' pairs of each expert in a round of
// kSortThreads.
template <bool SELF>
__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(const SortParams p, uint32_t each) {
    extern __shared__ uint32_t sort_smem[];
    __shared__ uint32_t warps[32];
    uint32_t *base = sort_smem, *by_warp = sort_smem + p.E;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const uint32_t n = p.T * p.k, lo = blockIdx.x * each, hi = min(n, lo + each);
    for (uint32_t q = tid; q < kSortWarps * p.E; q += kSortThreads) by_warp[q] = 0;
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    __syncthreads();
    // by_warp[0]: all pairs on an expert; [1]: those of the blocks before this one
    if constexpr (SELF) {
#pragma unroll 4
        for (uint32_t i = tid; i < n; i += kSortThreads) {
            const uint32_t e = pair_expert(p, i);
            if (e >= p.E) continue;
            atomicAdd(by_warp + e, 1u);
            if (i < lo) atomicAdd(by_warp + p.E + e, 1u);
        }
    } else {
        for (uint32_t e = tid; e < p.E; e += kSortThreads) {
            by_warp[e] = p.totals[e];
            by_warp[p.E + e] = p.counts[(size_t)blockIdx.x * p.E + e];
        }
    }
    __syncthreads();
    uint32_t run = 0;
    for (uint32_t e0 = 0; e0 < p.E; e0 += kSortThreads) {
        const uint32_t e = e0 + tid, all = e < p.E ? by_warp[e] : 0u;
        const uint32_t first = run + sum_before(all, warps);
        if (e < p.E) {
            base[e] = first + by_warp[p.E + e];
            if (blockIdx.x == 0) {
                p.offsets[e] = first;
                if (e + 1u == p.E) p.offsets[p.E] = first + all;
            }
        }
        if (tid == kSortThreads - 1u) warps[31] = first + all;
        __syncthreads();
        run = warps[31];
        __syncthreads();
    }
    for (uint32_t q = tid; q < 2u * p.E; q += kSortThreads) by_warp[q] = 0;
    __syncthreads();
    for (uint32_t c0 = lo; c0 < hi; c0 += kSortThreads) {
        const uint32_t i = c0 + tid;
        const uint32_t e = i < hi ? pair_expert(p, i) : p.E;
        const uint32_t same = __match_any_sync(0xffffffffu, e), ahead = __popc(same & ((1u << lane) - 1u));
        const bool first = e < p.E && ahead == 0;
        if (first) by_warp[warp * p.E + e] = __popc(same);
        __syncthreads();
        uint32_t place = VLB_NO_ROW;
        if (e < p.E) {
            place = base[e] + ahead;
            for (uint32_t w = 0; w < warp; ++w) place += by_warp[w * p.E + e];
        }
        if (i < hi) put_pair(p, i, place);
        if (c0 + kSortThreads >= hi) break;
        __syncthreads();
        if (first) {
            atomicAdd(base + e, by_warp[warp * p.E + e]);
            by_warp[warp * p.E + e] = 0;
        }
        __syncthreads();
    }
}

// ---- rows by expert --------------------------------------------------------------------------------

// LANES lanes (a warp, or 8 for short rows) move a segment of a token's row, kSegment pieces a lane: read once, written
// once a live slot. HBM-bound (16,384 x 8 of 2048 bf16, a fifth dropped: 83 us, 5.9 TB/s); a block an item, since the
// blocks that come after keep the stores going (persistent ones 125 us where these take 109).
constexpr uint32_t kSegment = 4;
template <uint32_t LANES>
__device__ __forceinline__ void copy_segment(const SortParams& p, uint32_t first, uint32_t units, const uint4 (&v)[kSegment],
                                             uint32_t row) {
    if (row == VLB_NO_ROW) return;
    uint4* to = reinterpret_cast<uint4*>(p.rows + row * p.rows_stride);
#pragma unroll
    for (uint32_t i = 0; i < kSegment; ++i)
        if (first + LANES * i < units) to[first + LANES * i] = v[i];
}
template <uint32_t LANES>
__global__ void __launch_bounds__(256) sort_rows_kernel(const SortParams p, uint32_t segments) {
    constexpr uint32_t kItems = 256u / LANES;
    const uint32_t units = (uint32_t)(p.row_bytes / 16u), lane = threadIdx.x % LANES;
    const uint64_t items = (uint64_t)p.T * segments;
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    for (uint64_t q0 = (uint64_t)blockIdx.x * kItems; q0 < items; q0 += (uint64_t)gridDim.x * kItems) {
        const uint64_t q = q0 + threadIdx.x / LANES;
        const size_t t = q / segments;
        const uint32_t first = (uint32_t)(q - t * segments) * LANES * kSegment + lane;
        const bool have = q < items;
        const uint4* x = reinterpret_cast<const uint4*>(p.x + t * p.x_stride);
        uint4 v[kSegment];
#pragma unroll
        for (uint32_t i = 0; i < kSegment; ++i)
            if (have && first + LANES * i < units) v[i] = x[first + LANES * i];
        for (uint32_t s0 = 0; s0 < p.k; s0 += LANES) {
            const uint32_t mine = have && s0 + lane < p.k ? p.elem_row[t * p.k + s0 + lane] : VLB_NO_ROW;
            for (uint32_t s = 0; s < min(LANES, p.k - s0); ++s)
                copy_segment<LANES>(p, first, units, v, __shfl_sync(0xffffffffu, mine, s, LANES));
        }
    }
}

// Rows at any offset: LANES lanes move a segment of a pair's row, in pieces of the row written. E: a type of the
// elements' size. 16,384 x 8 of 1001 bf16 82 us (element by element 102; 3.6 TB/s), of 333 int8 44.
template <typename E, uint32_t LANES>
__device__ __forceinline__ void copy_shifted(const SortParams& p, uint32_t pair, uint32_t segment, uint32_t row, uint32_t lane) {
    constexpr uint32_t V = 16u / sizeof(E);
    if (row == VLB_NO_ROW) return;
    const uint32_t H = (uint32_t)(p.row_bytes / sizeof(E)), t = pair / p.k;
    const E* x = reinterpret_cast<const E*>(p.x + (size_t)t * p.x_stride);
    E* to = reinterpret_cast<E*>(p.rows + row * p.rows_stride);
    const int32_t c0 = (int32_t)((segment * LANES * kSegment + lane) * V) - row_offset<V>(to);
    const uint32_t shift = Raw<V, true, E>::shift_of(x, c0);
    if (!inside_rows<V, true, E>(t, p.T, p.x_stride / sizeof(E), H)) {  // the first and the last row
        for (uint32_t i = 0; i < kSegment; ++i) {
            const int32_t c = c0 + (int32_t)(LANES * i * V);
            E v[V];
#pragma unroll
            for (uint32_t j = 0; j < V; ++j) v[j] = (uint32_t)(c + (int32_t)j) < H ? x[c + (int32_t)j] : E();
#pragma unroll
            for (uint32_t j = 0; j < V; ++j)
                if ((uint32_t)(c + (int32_t)j) < H) to[c + (int32_t)j] = v[j];
        }
        return;
    }
    Raw<V, true, E> a[kSegment];
#pragma unroll
    for (uint32_t i = 0; i < kSegment; ++i)
        if (c0 + (int32_t)(LANES * i * V) < (int32_t)H) a[i].load(x, c0 + (int32_t)(LANES * i * V), shift);
#pragma unroll
    for (uint32_t i = 0; i < kSegment; ++i) {
        const int32_t c = c0 + (int32_t)(LANES * i * V);
        if (c >= (int32_t)H) break;
        const Pack<E, V> v = a[i].get(shift);
        if (inside(c, V, H)) {
            *reinterpret_cast<Pack<E, V>*>(to + c) = v;
        } else {
#pragma unroll
            for (uint32_t j = 0; j < V; ++j)
                if ((uint32_t)(c + (int32_t)j) < H) to[c + (int32_t)j] = v.v[j];
        }
    }
}
template <typename E, uint32_t LANES>
__global__ void __launch_bounds__(256) sort_rows_shifted_kernel(const SortParams p, uint32_t segments) {
    constexpr uint32_t kItems = 256u / LANES;
    const uint64_t items = (uint64_t)p.T * p.k * segments;
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    uint64_t q = (uint64_t)blockIdx.x * kItems + threadIdx.x / LANES;
    uint32_t next = q < items ? p.elem_row[q / segments] : VLB_NO_ROW;
    for (; q < items;) {
        const uint32_t pair = (uint32_t)(q / segments), segment = (uint32_t)(q - (uint64_t)pair * segments), row = next;
        q += (uint64_t)gridDim.x * kItems;
        if (q < items) next = p.elem_row[q / segments];  // on its way beside this one's row
        copy_shifted<E, LANES>(p, pair, segment, row, threadIdx.x % LANES);
    }
}

// ---- few pairs: one launch -------------------------------------------------------------------------

// Every block holds all pairs' experts, a warp finds a pair's place by counting the pairs before it (of smaller
// experts, and of its own with a smaller number), and the block moves its tokens' rows; the last block takes the
// offsets. Latency: 64 x 8 over 256 experts with rows of 4096 bf16 3.5 us, the order alone 2.1. Shared: [n] experts. E: a type of the elements' size, where SHIFTED.
constexpr uint32_t kFewPairs = 4096, kFewWork = 1u << 19, kFewBytes = 64u * 1024u;
template <typename E, bool SHIFTED>
__global__ void __launch_bounds__(256) sort_few_kernel(const SortParams p, uint32_t segments) {
    extern __shared__ uint32_t sort_smem[];
    __shared__ uint32_t place_s[64], hist[kSortMaxExperts], warps[32];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, n = p.T * p.k;
    const uint32_t t = blockIdx.x;
    const bool last = t == p.T;
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    const uint32_t units = (uint32_t)(p.row_bytes / 16u);
    uint4 v[kSegment];
    const auto fetch = [&](uint32_t segment) {
        const uint4* x = reinterpret_cast<const uint4*>(p.x + (size_t)t * p.x_stride);
#pragma unroll
        for (uint32_t i = 0; i < kSegment; ++i)
            if (segment * 32u * kSegment + lane + 32u * i < units) v[i] = x[segment * 32u * kSegment + lane + 32u * i];
    };
    if (!SHIFTED && p.rows && !last && warp < segments) fetch(warp);  // on its way beside the order
    for (uint32_t i = tid; i < n; i += 256u) sort_smem[i] = pair_expert(p, i);
    if (last)
        for (uint32_t e = tid; e < p.E; e += 256u) hist[e] = 0;
    __syncthreads();
    if (last) {
        for (uint32_t i = tid; i < n; i += 256u)
            if (sort_smem[i] < p.E) atomicAdd(hist + sort_smem[i], 1u);
        __syncthreads();
        uint32_t run = 0;
        for (uint32_t e0 = 0; e0 < p.E; e0 += 256u) {
            const uint32_t e = e0 + tid, all = e < p.E ? hist[e] : 0u;
            const uint32_t first = run + sum_before(all, warps);
            if (e < p.E) p.offsets[e] = first;
            if (e + 1u == p.E) p.offsets[p.E] = first + all;
            if (tid == 255u) warps[31] = first + all;
            __syncthreads();
            run = warps[31];
            __syncthreads();
        }
        return;
    }
    for (uint32_t s = warp; s < p.k; s += 8u) {
        const uint32_t i = t * p.k + s, e = sort_smem[i];
        uint32_t before = 0;
        for (uint32_t j = lane; j < n; j += 32u) before += sort_smem[j] < e + (j < i ? 1u : 0u) ? 1u : 0u;
        before = __reduce_add_sync(0xffffffffu, before);
        if (lane == 0) {
            place_s[s] = e < p.E ? before : VLB_NO_ROW;
            put_pair(p, i, place_s[s]);
        }
    }
    if (!p.rows) return;
    __syncthreads();
    if constexpr (SHIFTED) {
        for (uint32_t q = warp; q < p.k * segments; q += 8u)
            copy_shifted<E, 32>(p, t * p.k + q % p.k, q / p.k, place_s[q % p.k], lane);
    } else {
        for (uint32_t segment = warp; segment < segments; segment += 8u) {
            if (segment != warp) fetch(segment);
            for (uint32_t s = 0; s < p.k; ++s)
                copy_segment<32>(p, segment * 32u * kSegment + lane, units, v, place_s[s]);
        }
    }
}

// ---- weighted sums ---------------------------------------------------------------------------------

// LANES lanes (a warp, or 8 for short rows) take a segment of a token, KEEP pieces of V columns a lane (16 bytes of the
// rows), summed in registers over the slots in order, SLOTS slots' loads in flight. Pieces lie on the boundaries of out.
// HBM-bound: 16,384 x 8 of 2048 bf16 onto f32 115 us (6.1 TB/s; with branches between the loads 463), of 1001 bf16 83.
template <typename T, typename O, uint32_t LANES, uint32_t KEEP, uint32_t SLOTS, bool SHIFTED>
__global__ void __launch_bounds__(256, SLOTS > 2u ? 2 : SHIFTED ? 3 : 4) combine_kernel(const CombineParams p, uint32_t segments) {
    constexpr uint32_t V = 16u / sizeof(T), kItems = 256u / LANES;
    constexpr int32_t kStep = LANES * V;
    const uint32_t lane = threadIdx.x % LANES;
    const uint64_t items = (uint64_t)p.T * segments;
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    // the first LANES slots of the next item are on their way beside this one's rows
    uint32_t row_next = VLB_NO_ROW;
    float weight_next = 1.f;
    const auto ask = [&](uint64_t q) {
        if (q >= items || lane >= p.k) return;
        row_next = p.elem_row[q / segments * p.k + lane];
        if (p.weights) weight_next = p.weights[q / segments * p.k + lane];
    };
    ask((uint64_t)blockIdx.x * kItems + threadIdx.x / LANES);
    for (uint64_t q0 = (uint64_t)blockIdx.x * kItems; q0 < items; q0 += (uint64_t)gridDim.x * kItems) {
        const uint64_t q = q0 + threadIdx.x / LANES;
        const size_t t = q / segments;
        O* out = static_cast<O*>(p.out) + t * p.out_stride;
        const int32_t c0 = (int32_t)(((uint32_t)(q - t * segments) * LANES * KEEP + lane) * V) - (SHIFTED ? row_offset<V>(out) : 0);
        // this lane's columns: from c0 to before end
        const int32_t end = q < items ? (int32_t)p.H : c0;
        const O* res = static_cast<const O*>(p.residual) + t * p.residual_stride;
        const bool res_whole = inside_rows<V, SHIFTED, O>((uint32_t)t, p.T, p.residual_stride, p.H);
        const uint32_t res_shift = Piece<V, SHIFTED, O>::shift_of(res, c0);
        Piece<V, SHIFTED, O> r[KEEP];
        if (p.residual && res_whole) {
#pragma unroll
            for (uint32_t i = 0; i < KEEP; ++i)
                if (c0 + (int32_t)i * kStep < end) r[i].load(res, c0 + (int32_t)i * kStep, res_shift);
        }
        float acc[KEEP][V] = {};
        for (uint32_t s0 = 0; s0 < p.k; s0 += LANES) {
            uint32_t row_of = VLB_NO_ROW;
            float weight_of = 1.f;
            if (q < items && s0 + lane < p.k) {
                row_of = s0 ? p.elem_row[t * p.k + s0 + lane] : row_next;
                if (p.weights) weight_of = s0 ? p.weights[t * p.k + s0 + lane] : weight_next;
            }
            if (s0 == 0) ask(q + (uint64_t)gridDim.x * kItems);
            const uint32_t slots = min(LANES, p.k - s0);
            for (uint32_t s1 = 0; s1 < slots; s1 += SLOTS) {
                Piece<V, SHIFTED, T> a[SLOTS][KEEP];
                uint32_t row[SLOTS], shift[SLOTS];
                float w[SLOTS];
                bool whole = true;
#pragma unroll
                for (uint32_t s = 0; s < SLOTS; ++s) {
                    row[s] = __shfl_sync(0xffffffffu, row_of, (s1 + s) % LANES, LANES);
                    w[s] = __shfl_sync(0xffffffffu, weight_of, (s1 + s) % LANES, LANES);
                    if (s1 + s >= slots || row[s] >= p.n_rows) row[s] = VLB_NO_ROW;
                    whole = whole && (row[s] == VLB_NO_ROW || inside_rows<V, SHIFTED, T>(row[s], p.n_rows, p.rows_stride, p.H));
                }
                const T* rows = static_cast<const T*>(p.rows);
                if (!__all_sync(0xffffffffu, whole)) {
#pragma unroll
                    for (uint32_t s = 0; s < SLOTS; ++s) {
                        if (row[s] == VLB_NO_ROW) continue;
#pragma unroll
                        for (uint32_t i = 0; i < KEEP; ++i)
                            add_each<V>(w[s], rows + row[s] * p.rows_stride, c0 + (int32_t)i * kStep, p.H, acc[i]);
                    }
                    continue;
                }
#pragma unroll
                for (uint32_t s = 0; s < SLOTS; ++s) {
                    const T* from = rows + row[s] * p.rows_stride;
                    shift[s] = a[s][0].shift_of(from, c0);
#pragma unroll
                    for (uint32_t i = 0; i < KEEP; ++i)
                        if (row[s] != VLB_NO_ROW && c0 + (int32_t)i * kStep < end)
                            a[s][i].load(from, c0 + (int32_t)i * kStep, shift[s]);
                }
#pragma unroll
                for (uint32_t s = 0; s < SLOTS; ++s) {
                    if (row[s] == VLB_NO_ROW) continue;
#pragma unroll
                    for (uint32_t i = 0; i < KEEP; ++i) {
                        float f[V];
                        a[s][i].get(shift[s], f);
#pragma unroll
                        for (uint32_t j = 0; j < V; ++j) acc[i][j] = fmaf(w[s], f[j], acc[i][j]);
                    }
                }
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i) {
            const int32_t c = c0 + (int32_t)i * kStep;
            if (c >= end) break;
            if (p.residual && res_whole) {
                float f[V];
                r[i].get(res_shift, f);
#pragma unroll
                for (uint32_t j = 0; j < V; ++j) acc[i][j] += f[j];
            } else if (p.residual) {
                add_each<V>(1.f, res, c, p.H, acc[i]);
            }
            if constexpr (V * sizeof(O) == 32u && !SHIFTED) {
                if (inside(c, V, p.H)) {
                    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out + c), "f"(acc[i][0]),
                                 "f"(acc[i][1]), "f"(acc[i][2]), "f"(acc[i][3]), "f"(acc[i][4]), "f"(acc[i][5]), "f"(acc[i][6]),
                                 "f"(acc[i][7])
                                 : "memory");
                    continue;
                }
            }
            store_piece<V>(out + c, acc[i], c, p.H);
        }
    }
}

// ROW lanes (a warp; 8 for short rows; the CTA where pairs are few) take a pair: its row in pieces of its own
// boundaries (of drows where they are written), dout beside it, which the pairs of a token share in L1. HBM-bound: 8192 x 8
// of 2048 bf16 89 us (5.3 TB/s). Two pieces in flight in 32 warps an SM: 32,768 x 8 of 128 bf16 38 us, four pieces in 24
// warps 48; 16,384 x 8 of 2048 195 and 202, 256 x 8 7.6 and 6.9. Shifted, 16 warps: 16,384 x 8 of 1001 168, 24 warps 178.
template <typename T, typename O, uint32_t ROW, bool SHIFTED>
__global__ void __launch_bounds__(256, SHIFTED ? 2 : 4) combine_grad_kernel(const CombineGradParams p) {
    constexpr uint32_t V = 16u / sizeof(T), kRows = 256u / ROW, kAtOnce = !SHIFTED || sizeof(O) > sizeof(T) ? 2u : 4u;
    __shared__ float scratch[2][8];
    const uint32_t tid = threadIdx.x % ROW;
    const uint64_t pairs = (uint64_t)p.T * p.k;
    tc::grid_dependency_wait();
    tc::grid_launch_dependents();
    uint32_t turn = 0, row_next = VLB_NO_ROW;
    float w_next = 1.f;
    const auto ask = [&](uint64_t q) {  // the next pair's place and weight, on their way beside this one's row
        if (q >= pairs) return;
        row_next = p.elem_row[q];
        if (p.weights) w_next = p.weights[q];
    };
    ask((uint64_t)blockIdx.x * kRows + threadIdx.x / ROW);
    for (uint64_t q0 = (uint64_t)blockIdx.x * kRows; q0 < pairs; q0 += (uint64_t)gridDim.x * kRows) {
        const uint64_t q = q0 + threadIdx.x / ROW;
        const uint32_t row = q < pairs ? row_next : VLB_NO_ROW;
        const float w = w_next;
        ask(q + (uint64_t)gridDim.x * kRows);
        float acc = 0.f;
        if (row < p.n_rows) {
            const O* dout = static_cast<const O*>(p.dout) + (q / p.k) * p.dout_stride;
            const T* from = static_cast<const T*>(p.rows) + row * p.rows_stride;
            T* to = static_cast<T*>(p.drows) + row * p.drows_stride;
            const int32_t off = !SHIFTED ? 0 : p.drows ? row_offset<V>(to) : row_offset<V>(from);
            const bool whole = inside_rows<V, SHIFTED, O>((uint32_t)(q / p.k), p.T, p.dout_stride, p.H) &&
                               (!p.dweights || inside_rows<V, SHIFTED, T>(row, p.n_rows, p.rows_stride, p.H));
            const uint32_t shift_a = Piece<V, SHIFTED, T>::shift_of(from, (int32_t)(tid * V) - off);
            const uint32_t shift_d = Piece<V, SHIFTED, O>::shift_of(dout, (int32_t)(tid * V) - off);
            for (int32_t c0 = (int32_t)(tid * V) - off; whole && c0 < (int32_t)p.H; c0 += (int32_t)(kAtOnce * ROW * V)) {
                Piece<V, SHIFTED, T> a[kAtOnce];
                Piece<V, SHIFTED, O> d[kAtOnce];
#pragma unroll
                for (uint32_t i = 0; i < kAtOnce; ++i) {
                    const int32_t c = c0 + (int32_t)(i * ROW * V);
                    if (c >= (int32_t)p.H) continue;
                    if (p.dweights) a[i].load(from, c, shift_a);
                    d[i].load(dout, c, shift_d);
                }
#pragma unroll
                for (uint32_t i = 0; i < kAtOnce; ++i) {
                    const int32_t c = c0 + (int32_t)(i * ROW * V);
                    if (c >= (int32_t)p.H) continue;
                    float f[V], g[V];
                    d[i].get(shift_d, g);
                    if (p.dweights) {
                        a[i].get(shift_a, f);
                        clip(f, c, p.H);
                        clip(g, c, p.H);
#pragma unroll
                        for (uint32_t j = 0; j < V; ++j) acc = fmaf(g[j], f[j], acc);
                    }
                    if (p.drows) {
#pragma unroll
                        for (uint32_t j = 0; j < V; ++j) g[j] *= w;
                        store_piece<V>(to + c, g, c, p.H);
                    }
                }
            }
#pragma unroll 4
            for (uint32_t c = tid; c < (whole ? 0u : p.H); c += ROW) {  // the first and the last row
                const float g = to_float(dout[c]);
                if (p.dweights) acc = fmaf(g, to_float(from[c]), acc);
                if (p.drows) to[c] = from_float<T>(w * g);
            }
        }
        if (!p.dweights) continue;
        // in a fixed order: lanes, then warps; 0 of a dropped pair
        __syncwarp();
#pragma unroll
        for (uint32_t m = ROW < 32u ? ROW / 2u : 16u; m; m >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, m);
        if constexpr (ROW == 256u) {
            if ((tid & 31u) == 0) scratch[turn][tid >> 5] = acc;
            __syncthreads();
            acc = 0.f;
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) acc += scratch[turn][i];
            turn ^= 1u;
        }
        if (tid == 0 && q < pairs) p.dweights[q] = acc;
    }
}

// ---- hosts -----------------------------------------------------------------------------------------

template <typename F>
cudaError_t by_type(int type, F&& f) {
    switch (type) {
        case VLB_DTYPE_F32: return f(float{});
        case VLB_DTYPE_F16: return f(__half{});
        case VLB_DTYPE_BF16: return f(__nv_bfloat16{});
        default: return cudaErrorInvalidValue;
    }
}

// Pairs of a block in the order's kernels: a round of kSortThreads, or as many rounds as leave kSortBlocks blocks.
uint32_t sort_each(uint64_t pairs) {
    const uint64_t rounds = (pairs + kSortThreads * kSortBlocks - 1u) / (kSortThreads * kSortBlocks);
    return (uint32_t)((rounds ? rounds : 1u) * kSortThreads);
}

// Blocks for so many items of 256 / lanes a block: at most `per_sm` an SM, whose warps then ask for an item's places while they
// move the one before.
uint32_t item_blocks(uint64_t items, uint32_t lanes, uint32_t per_sm = 16u) {
    const uint64_t blocks = (items + 256u / lanes - 1u) / (256u / lanes), most = per_sm * sm_count();
    return (uint32_t)(blocks < most ? blocks : most);
}

// Whether rows of `bytes` at p lie on whole units of n.
bool on(const void* p, size_t stride_bytes, size_t n) {
    return !p || (reinterpret_cast<uintptr_t>(p) % n == 0 && stride_bytes % n == 0);
}

template <typename E, bool SHIFTED, uint32_t LANES>
cudaError_t sort_moved(const SortParams& p, bool few, cudaStream_t s) {
    // 16-byte pieces of a row, one more at an offset
    const uint32_t pieces = p.rows ? (uint32_t)((p.row_bytes + 15u) / 16u) + (SHIFTED ? 1u : 0u) : 0u;
    const uint32_t lanes = few ? 32u : LANES, segments = (pieces + lanes * kSegment - 1u) / (lanes * kSegment);
    if (few) return launch_chained(sort_few_kernel<E, SHIFTED>, dim3(p.T + 1u), 256, (size_t)p.T * p.k * 4u, 0, s, p, segments);
    if constexpr (SHIFTED)
        return launch_chained(sort_rows_shifted_kernel<E, LANES>, dim3(item_blocks((uint64_t)p.T * p.k * segments, LANES)), 256,
                              0, 0, s, p, segments);
    else
        return launch_chained(sort_rows_kernel<LANES>, dim3(item_blocks((uint64_t)p.T * segments, LANES, 1u << 12)), 256, 0, 0, s, p,
                              segments);
}
// By what moves the rows: whole 16-byte units, or elements at any offset. Rows of up to 512 bytes take 8 lanes.
cudaError_t sort_rows(const SortParams& p, bool few, cudaStream_t s) {
    const bool whole = p.row_bytes % 16u == 0 && on(p.x, p.x_stride, 16) && on(p.rows, p.rows_stride, 16);
    const auto move = [&](auto e) {
        using E = decltype(e);
        return p.row_bytes <= 512u ? sort_moved<E, true, 8>(p, few, s) : sort_moved<E, true, 32>(p, few, s);
    };
    if (!p.rows || whole)
        return p.row_bytes <= 512u ? sort_moved<uint32_t, false, 8>(p, few, s) : sort_moved<uint32_t, false, 32>(p, few, s);
    return p.elem == 1 ? move(uint8_t{}) : p.elem == 2 ? move(uint16_t{}) : move(uint32_t{});
}

// Pieces of 16 bytes of the rows; of the others, 32, 16 or 8.
template <typename T, typename O>
bool on_pieces(const void* rows, size_t rows_stride, const void* other, size_t other_stride) {
    constexpr uint32_t V = 16u / sizeof(T), kOther = V * sizeof(O);
    return on(rows, rows_stride * sizeof(T), 16) && on(other, other_stride * sizeof(O), kOther);
}

template <typename T, typename O>
cudaError_t combine_typed(const CombineParams& p, cudaStream_t s) {
    constexpr uint32_t V = 16u / sizeof(T);
    const bool whole = on_pieces<T, O>(p.rows, p.rows_stride, p.out, p.out_stride) &&
                       on_pieces<T, O>(nullptr, 0, p.residual, p.residual_stride);
    const uint32_t pieces = (p.H + V - 1u) / V + (whole ? 0u : 1u);
    const auto run = [&](auto* kernel, uint32_t lanes, uint32_t keep) {
        const uint32_t segments = (pieces + lanes * keep - 1u) / (lanes * keep);
        return launch_chained(kernel, dim3(item_blocks((uint64_t)p.T * segments, lanes)), 256, 0, 0, s, p, segments);
    };
    if (pieces <= 16u) return whole ? run(combine_kernel<T, O, 8, 2, 2, false>, 8, 2) : run(combine_kernel<T, O, 8, 2, 2, true>, 8, 2);
    // few tokens: a piece a lane, all slots at once (8 slots of 2048 bf16 onto f32, this way / below: 64 tokens 3.4 / 4.5 us,
    // 256 5.1 / 6.7, 512 9.2 / 7.8; of two slots, which need no more in flight, 64 3.0 / 2.6, 512 7.8 / 4.6)
    if ((uint64_t)p.T * pieces <= (1u << 17))
        return whole ? run(combine_kernel<T, O, 32, 1, 8, false>, 32, 1) : run(combine_kernel<T, O, 32, 1, 4, true>, 32, 1);
    // Two pieces of two slots a lane in flight and 32 warps an SM (shifted 24) rather than more of both and 16 warps: 16,384
    // tokens of 2048 bf16 onto f32 with 8 slots 129 us (four of four 137), with two 66 (86); shifted,
    // of 1001 bf16, 83 us, in 16 warps 92, one piece of two or four slots 89 and 100. The 64 (80) registers of so many warps
    // spill: 16-bit rows onto f32 48 bytes a thread, shifted 124, onto 16 bits 84; f32 12 and 48.
    return whole ? run(combine_kernel<T, O, 32, 2, 2, false>, 32, 2) : run(combine_kernel<T, O, 32, 2, 2, true>, 32, 2);
}

template <typename T, typename O>
cudaError_t combine_grad_typed(const CombineGradParams& p, cudaStream_t s) {
    constexpr uint32_t V = 16u / sizeof(T);
    const bool whole = on_pieces<T, O>(p.dweights ? p.rows : nullptr, p.rows_stride, p.dout, p.dout_stride) &&
                       on(p.drows, p.drows_stride * sizeof(T), 16);
    const uint64_t pairs = (uint64_t)p.T * p.k;
    const auto run = [&](auto shifted) {
        constexpr bool kShifted = decltype(shifted)::value;
        // A CTA a pair while warps would leave SMs idle, longer for long rows (bf16, CTA / warp: 512 pairs of 1024 3.4 / 2.5
        // us, of 4096 4.0 / 5.3; 2048 pairs of 2048 11.3 / 6.3).
        if (pairs < (p.H >= 256u * V ? 1024u : 256u) && p.H >= 64u * V)
            return launch_chained(combine_grad_kernel<T, O, 256, kShifted>, dim3((uint32_t)pairs), 256, 0, 0, s, p);
        if (p.H <= 32u * V)
            return launch_chained(combine_grad_kernel<T, O, 8, kShifted>, dim3(item_blocks(pairs, 8)), 256, 0, 0, s, p);
        return launch_chained(combine_grad_kernel<T, O, 32, kShifted>, dim3(item_blocks(pairs, 32)), 256, 0, 0, s, p);
    };
    return whole ? run(std::false_type{}) : run(std::true_type{});
}

}  // namespace

uint32_t sort_blocks(uint64_t pairs) {
    const uint64_t each = sort_each(pairs);
    return (uint32_t)((pairs + each - 1u) / each);
}

// Blocks fall where a round is added to each: the bound does not.
uint32_t sort_blocks_bound(uint64_t pairs) {
    const uint64_t rounds = (pairs + kSortThreads - 1u) / kSortThreads;
    return (uint32_t)(rounds < kSortBlocks ? rounds : kSortBlocks);
}

cudaError_t launch_sort_tokens(const SortParams& p, cudaStream_t s) {
    const uint32_t n = p.T * p.k;
    // Every token's block goes through all pairs: 256 tokens of 8 5.9 us, 512 13.1, 4000 of one 24 (else 13 to 14). Long
    // rows are moved by a launch of their own: a token's block would take its pairs' one after another.
    if (n <= kFewPairs && (uint64_t)p.T * n <= kFewWork) {
        if (!p.rows || p.k * p.row_bytes <= kFewBytes) return sort_rows(p, true, s);
        SortParams order = p;
        order.rows = nullptr;
        const cudaError_t e = sort_rows(order, true, s);
        return e != cudaSuccess ? e : sort_rows(p, false, s);
    }
    const uint32_t each = sort_each(n), blocks = sort_blocks(n);
    const bool self = n <= kSelfPairs;
    cudaError_t e = cudaSuccess;
    if (!self) {
        if ((e = launch_chained(sort_count_kernel, dim3(blocks), kSortThreads, 0, 0, s, p, each)) != cudaSuccess) return e;
        e = launch_chained(sort_prefix_kernel, dim3((p.E + 31u) / 32u), 1024, 0, 0, s, p, blocks);
        if (e != cudaSuccess) return e;
    }
    const auto kernel = self ? sort_place_kernel<true> : sort_place_kernel<false>;
    if ((e = smem_once(kernel, (kSortWarps + 1u) * kSortMaxExperts * 4u)) != cudaSuccess) return e;
    e = launch_chained(kernel, dim3(blocks), kSortThreads, (size_t)(kSortWarps + 1u) * p.E * 4u, 0, s, p, each);
    return e != cudaSuccess || !p.rows ? e : sort_rows(p, false, s);
}

cudaError_t launch_combine(const CombineParams& p, int type, int out_type, cudaStream_t s) {
    return by_type(type, [&](auto t) {
        return by_type(out_type, [&](auto o) { return combine_typed<decltype(t), decltype(o)>(p, s); });
    });
}

cudaError_t launch_combine_grad(const CombineGradParams& p, int type, int out_type, cudaStream_t s) {
    return by_type(type, [&](auto t) {
        return by_type(out_type, [&](auto o) { return combine_grad_typed<decltype(t), decltype(o)>(p, s); });
    });
}

}  // namespace vlb
