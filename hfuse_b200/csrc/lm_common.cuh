// Shared pieces of the language-model operators (layer norm, embedding, gated recurrence):
// element types, packed loads and stores, and the host-side choice of a template by type.
// All arithmetic is 32-bit floating point; 16-bit types exist in memory only and a value is
// rounded to them once, when it is stored.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace hfuse {

template <class T>
__device__ __forceinline__ float to_f32(T v) { return static_cast<float>(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// N neighbouring elements as one memory access (2 to 32 bytes, aligned to its size, 16 at most), kept as the words that
// were loaded: two 16-bit elements to a register
template <class T, int N>
struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Pack {
    static constexpr int BYTES = N * (int)sizeof(T);
    using Word = std::conditional_t<BYTES >= 4, unsigned, unsigned short>;
    Word w[BYTES / sizeof(Word)];
};
// inputs that are read once bypass L1
template <class T, int N>
__device__ __forceinline__ Pack<T, N> load_stream(const T* p) {
    Pack<T, N> r;
    if constexpr (r.BYTES == 16)
        asm("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]) : "l"(p));
    else if constexpr (r.BYTES == 8)
        asm("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r.w[0]), "=r"(r.w[1]) : "l"(p));
    else if constexpr (r.BYTES == 4)
        asm("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(r.w[0]) : "l"(p));
    else
        asm("ld.global.nc.L1::no_allocate.u16 %0, [%1];" : "=h"(r.w[0]) : "l"(p));
    return r;
}
// inputs that several blocks or rows read (weights, tables), in accesses of 16 bytes at most
template <class T, int N>
__device__ __forceinline__ Pack<T, N> load_cached(const T* p) {
    Pack<T, N> r;
    if constexpr (r.BYTES >= 16) {
#pragma unroll
        for (int k = 0; k < r.BYTES / 16; ++k) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + k);
            r.w[4 * k] = u.x;
            r.w[4 * k + 1] = u.y;
            r.w[4 * k + 2] = u.z;
            r.w[4 * k + 3] = u.w;
        }
    } else if constexpr (r.BYTES == 8) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
        r.w[0] = u.x;
        r.w[1] = u.y;
    } else {
        r.w[0] = __ldg(reinterpret_cast<const typename Pack<T, N>::Word*>(p));
    }
    return r;
}
// the same from shared memory (32-bit address)
template <class T, int N>
__device__ __forceinline__ Pack<T, N> load_shared(uint32_t p) {
    Pack<T, N> r;
    if constexpr (r.BYTES == 16)
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]) : "r"(p) : "memory");
    else if constexpr (r.BYTES == 8)
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r.w[0]), "=r"(r.w[1]) : "r"(p) : "memory");
    else if constexpr (r.BYTES == 4)
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r.w[0]) : "r"(p) : "memory");
    else
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(r.w[0]) : "r"(p) : "memory");
    return r;
}
// outputs that this kernel does not read again
template <class T, int N>
__device__ __forceinline__ void store_stream(T* p, const Pack<T, N>& r) {
    if constexpr (r.BYTES == 16)
        asm volatile("st.global.cs.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(r.w[0]), "r"(r.w[1]), "r"(r.w[2]), "r"(r.w[3]) : "memory");
    else if constexpr (r.BYTES == 8)
        asm volatile("st.global.cs.v2.u32 [%0], {%1,%2};" ::"l"(p), "r"(r.w[0]), "r"(r.w[1]) : "memory");
    else if constexpr (r.BYTES == 4)
        asm volatile("st.global.cs.u32 [%0], %1;" ::"l"(p), "r"(r.w[0]) : "memory");
    else
        asm volatile("st.global.cs.u16 [%0], %1;" ::"l"(p), "h"(r.w[0]) : "memory");
}

// the k-th pair of N elements; an odd element is a pair with a second value of zero
template <class T, int N>
__device__ __forceinline__ float2 pair_of(const Pack<T, N>& p, int k) {
    if constexpr (N == 1) {
        T v;
        memcpy(&v, p.w, sizeof(T));
        return make_float2(to_f32(v), 0.f);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        return make_float2(__uint_as_float(p.w[k] << 16), __uint_as_float(p.w[k] & 0xffff0000u));
    } else if constexpr (std::is_same_v<T, __half>) {
        __half2 h;
        memcpy(&h, &p.w[k], 4);
        return __half22float2(h);
    } else {
        return make_float2(__uint_as_float(p.w[2 * k]), __uint_as_float(p.w[2 * k + 1]));
    }
}
// pairs of floats rounded to N elements of type T (N = 1: the pair's first value)
template <class T, int N>
__device__ __forceinline__ Pack<T, N> pack_pairs(const float2 (&v)[(N + 1) / 2]) {
    Pack<T, N> r;
    if constexpr (N == 1) {
        const T t = from_f32<T>(v[0].x);
        memcpy(r.w, &t, sizeof(T));
    } else {
#pragma unroll
        for (int k = 0; k < N / 2; ++k) {
            if constexpr (std::is_same_v<T, __half>) {
                const __half2 h = __floats2half2_rn(v[k].x, v[k].y);
                memcpy(&r.w[k], &h, 4);
            } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[k].x, v[k].y);
                memcpy(&r.w[k], &h, 4);
            } else {
                r.w[2 * k] = __float_as_uint(v[k].x);
                r.w[2 * k + 1] = __float_as_uint(v[k].y);
            }
        }
    }
    return r;
}

// two floats in one instruction: these kernels are short of issue slots sooner than of arithmetic
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long r, x, y, z;
    memcpy(&x, &a, 8);
    memcpy(&y, &b, 8);
    memcpy(&z, &c, 8);
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    memcpy(&a, &r, 8);
    return a;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long r, x, y;
    memcpy(&x, &a, 8);
    memcpy(&y, &b, 8);
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    memcpy(&a, &r, 8);
    return a;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    unsigned long long r, x, y;
    memcpy(&x, &a, 8);
    memcpy(&y, &b, 8);
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    memcpy(&a, &r, 8);
    return a;
}

// the warp's index in its block, known to the compiler to be the same in all lanes
__device__ __forceinline__ int warp_index() { return __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// sum over the block, the same bits in every thread; `sh` holds one float per warp.  The closing barrier lets the
// caller use `sh` again at once.
__device__ __forceinline__ float block_sum(float v, float* sh) {
    const int warps = (blockDim.x + 31) >> 5;
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.f;
    for (int w = 0; w < warps; ++w) s += sh[w];
    __syncthreads();
    return s;
}

constexpr int kMaxWidth = 1 << 30;       // elements of a row: the kernels step beyond the last one in 32 bits

// ---- host: element types -------------------------------------------------------------------
inline bool lm_type_ok(int t) { return t == HFUSE_F32 || t == HFUSE_BF16 || t == HFUSE_F16; }
inline int lm_type_size(int t) { return t == HFUSE_F32 ? 4 : 2; }
inline bool aligned_to(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

template <class T>
struct TypeTag {
    using type = T;
};
// f(TypeTag<float>{}) or its 16-bit counterparts
template <class F>
int by_type(int t, F&& f) {
    if (t == HFUSE_BF16) return f(TypeTag<__nv_bfloat16>{});
    if (t == HFUSE_F16) return f(TypeTag<__half>{});
    return f(TypeTag<float>{});
}
// weights have the activations' type or float
template <class F>
int by_types(int t, int wt, F&& f) {
    return by_type(t, [&](auto a) {
        using T = typename decltype(a)::type;
        if (wt == HFUSE_F32) return f(a, TypeTag<float>{});
        return f(a, TypeTag<T>{});
    });
}

}  // namespace hfuse
