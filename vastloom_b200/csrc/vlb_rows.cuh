// Rows of elements, as the row operators read and write them.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

namespace vlb {

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

// V neighbouring elements, moved with one access of up to 16 bytes (two for 8 floats).
template <typename T, uint32_t V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack {
    T v[V];
};
// The columns c .. c + V - 1 of a row, p at column c: those inside [0, cols), zeros for the others. A piece that
// is inside lies on its own alignment.
__device__ __forceinline__ bool inside(int32_t c, uint32_t n, uint32_t cols) { return c >= 0 && (uint32_t)c + n <= cols; }
template <uint32_t V, typename T>
__device__ __forceinline__ Pack<T, V> load_piece(const T* p, int32_t c, uint32_t cols) {
    Pack<T, V> a;
    if (inside(c, V, cols)) {
        a = *reinterpret_cast<const Pack<T, V>*>(p);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) a.v[i] = (uint32_t)(c + (int32_t)i) < cols ? p[i] : from_float<T>(0.f);
    }
    return a;
}
// Zeros outside [0, cols).
template <uint32_t V>
__device__ __forceinline__ void clip(float (&f)[V], int32_t c, uint32_t cols) {
    if (inside(c, V, cols)) return;
#pragma unroll
    for (uint32_t i = 0; i < V; ++i)
        if ((uint32_t)(c + (int32_t)i) >= cols) f[i] = 0.f;
}

// Two elements an instruction, or a shift and a mask, where they come in pairs. a lies in registers: of one in memory
// a copy is made first, or it is read element by element.
template <uint32_t V, typename T>
__device__ __forceinline__ void unpack(const Pack<T, V>& a, float (&f)[V]) {
    if constexpr (sizeof(T) == 2 && V % 2 == 0) {
#pragma unroll
        for (uint32_t i = 0; i < V; i += 2) {
            const uint32_t w = reinterpret_cast<const uint32_t*>(&a)[i / 2];
            if constexpr (std::is_same<T, __half>::value) {
                const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w));
                f[i] = v.x, f[i + 1] = v.y;
            } else {
                f[i] = __uint_as_float(w << 16), f[i + 1] = __uint_as_float(w & 0xffff0000u);
            }
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) f[i] = to_float(a.v[i]);
    }
}
template <typename T, uint32_t V>
__device__ __forceinline__ Pack<T, V> pack(const float (&f)[V]) {
    Pack<T, V> a;
    if constexpr (sizeof(T) == 2 && V % 2 == 0) {
#pragma unroll
        for (uint32_t i = 0; i < V; i += 2) {
            if constexpr (std::is_same<T, __half>::value)
                *reinterpret_cast<__half2*>(&a.v[i]) = __floats2half2_rn(f[i], f[i + 1]);
            else
                *reinterpret_cast<__nv_bfloat162*>(&a.v[i]) = __floats2bfloat162_rn(f[i], f[i + 1]);
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) a.v[i] = from_float<T>(f[i]);
    }
    return a;
}
// V values rounded to the columns c .. c + V - 1, p at column c, where they are inside [0, cols).
template <uint32_t V, typename T>
__device__ __forceinline__ void store_piece(T* p, const float (&f)[V], int32_t c, uint32_t cols) {
    const Pack<T, V> a = pack<T>(f);
    if (inside(c, V, cols)) {
        *reinterpret_cast<Pack<T, V>*>(p) = a;
    } else {
#pragma unroll
        for (uint32_t i = 0; i < V; ++i)
            if ((uint32_t)(c + (int32_t)i) < cols) p[i] = a.v[i];
    }
}

// Sum and largest over the ROW threads of a row (a warp, or neighbouring warps), the same in each of them and
// in a fixed order. at: two sets of ROW / 32 words of the row's own that take turns, so that one barrier is
// enough; barrier: its number, where a CTA of THREADS holds several rows.
template <uint32_t ROW, uint32_t THREADS = ROW>
struct RowReduce {
    float (*at)[ROW / 32u];
    uint32_t turn = 0;
    __device__ __forceinline__ void sync() const {
        if constexpr (ROW == THREADS) __syncthreads();
        else asm volatile("bar.sync %0, %1;" ::"r"(1u + threadIdx.x / ROW), "n"(ROW) : "memory");
    }
    __device__ __forceinline__ static uint32_t warp() { return threadIdx.x % ROW >> 5; }
    __device__ __forceinline__ float sum(float v) {
#pragma unroll
        for (uint32_t d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
        if constexpr (ROW > 32u) {
            if ((threadIdx.x & 31u) == 0) at[turn][warp()] = v;
            sync();
            v = 0.f;
#pragma unroll
            for (uint32_t i = 0; i < ROW / 32u; ++i) v += at[turn][i];
            turn ^= 1u;
        }
        return v;
    }
    __device__ __forceinline__ uint32_t most(uint32_t v) {
        v = __reduce_max_sync(0xffffffffu, v);
        if constexpr (ROW > 32u) {
            if ((threadIdx.x & 31u) == 0) at[turn][warp()] = __uint_as_float(v);
            sync();
#pragma unroll
            for (uint32_t i = 0; i < ROW / 32u; ++i) v = max(v, __float_as_uint(at[turn][i]));
            turn ^= 1u;
        }
        return v;
    }
};
// Two sums behind one barrier.
template <uint32_t ROW, uint32_t THREADS>
__device__ __forceinline__ void reduce_two(RowReduce<ROW, THREADS>& first, RowReduce<ROW, THREADS>& second, float& a, float& b) {
#pragma unroll
    for (uint32_t d = 16; d; d >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, d);
        b += __shfl_xor_sync(0xffffffffu, b, d);
    }
    if constexpr (ROW > 32u) {
        float *x = first.at[first.turn], *y = second.at[second.turn];
        if ((threadIdx.x & 31u) == 0) x[first.warp()] = a, y[first.warp()] = b;
        first.sync();
        a = b = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < ROW / 32u; ++i) a += x[i], b += y[i];
        first.turn ^= 1u;
        second.turn ^= 1u;
    }
}

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

// A vector's bytes at q; `n` of them (N but at a row's end).
template <uint32_t N>
__device__ __forceinline__ void store_bytes(int8_t* q, const float (&x)[N], const RowStep& st, uint32_t n) {
    uint32_t w[N / 4];
#pragma unroll
    for (uint32_t i = 0; i < N; i += 4u) {
        uint32_t b[4];
#pragma unroll
        for (uint32_t j = 0; j < 4u; ++j) b[j] = __float_as_uint(__fadd_rn(__fmul_rn(x[i + j], st.inv), 12582912.f));
        w[i / 4u] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
    if (n < N) {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i)
            if (i < n) q[i] = (int8_t)(w[i / 4u] >> (8u * (i % 4u)));
    } else if constexpr (N == 8) *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(q) = w[0];
}

}  // namespace vlb
