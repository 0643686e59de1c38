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

// N neighbouring elements as one memory access (2 to 16 bytes, aligned to its size)
template <class T, int N>
struct alignas(N * sizeof(T)) Pack {
    T v[N];
};
// inputs that are read once bypass L1
template <class T, int N>
__device__ __forceinline__ Pack<T, N> load_stream(const T* p) {
    Pack<T, N> r;
    if constexpr (sizeof(r) == 16) {
        uint4 u;
        asm("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p));
        memcpy(&r, &u, 16);
    } else if constexpr (sizeof(r) == 8) {
        uint2 u;
        asm("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(u.x), "=r"(u.y) : "l"(p));
        memcpy(&r, &u, 8);
    } else if constexpr (sizeof(r) == 4) {
        unsigned u;
        asm("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(u) : "l"(p));
        memcpy(&r, &u, 4);
    } else {
        unsigned short u;
        asm("ld.global.nc.L1::no_allocate.u16 %0, [%1];" : "=h"(u) : "l"(p));
        memcpy(&r, &u, 2);
    }
    return r;
}
// inputs that several blocks or rows read (weights, ids, states)
template <class T, int N>
__device__ __forceinline__ Pack<T, N> load_cached(const T* p) {
    Pack<T, N> r;
    if constexpr (sizeof(r) == 16) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
        memcpy(&r, &u, 16);
    } else if constexpr (sizeof(r) == 8) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
        memcpy(&r, &u, 8);
    } else if constexpr (sizeof(r) == 4) {
        const unsigned u = __ldg(reinterpret_cast<const unsigned*>(p));
        memcpy(&r, &u, 4);
    } else {
        const unsigned short u = __ldg(reinterpret_cast<const unsigned short*>(p));
        memcpy(&r, &u, 2);
    }
    return r;
}
// weights: N elements, in accesses of 16 bytes at most
template <class T, int N>
__device__ __forceinline__ void load_weights(const T* p, Pack<T, N>& r) {
    constexpr int M = N * sizeof(T) > 16 ? 16 / sizeof(T) : N;
#pragma unroll
    for (int k = 0; k < N; k += M) {
        const Pack<T, M> q = load_cached<T, M>(p + k);
        memcpy(r.v + k, q.v, sizeof(q));
    }
}
// outputs that this kernel does not read again
template <class T, int N>
__device__ __forceinline__ void store_stream(T* p, const Pack<T, N>& r) {
    if constexpr (sizeof(r) == 16) {
        uint4 u;
        memcpy(&u, &r, 16);
        asm volatile("st.global.cs.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(u.x), "r"(u.y), "r"(u.z), "r"(u.w) : "memory");
    } else if constexpr (sizeof(r) == 8) {
        uint2 u;
        memcpy(&u, &r, 8);
        asm volatile("st.global.cs.v2.u32 [%0], {%1,%2};" ::"l"(p), "r"(u.x), "r"(u.y) : "memory");
    } else if constexpr (sizeof(r) == 4) {
        unsigned u;
        memcpy(&u, &r, 4);
        asm volatile("st.global.cs.u32 [%0], %1;" ::"l"(p), "r"(u) : "memory");
    } else {
        unsigned short u;
        memcpy(&u, &r, 2);
        asm volatile("st.global.cs.u16 [%0], %1;" ::"l"(p), "h"(u) : "memory");
    }
}

// two neighbouring elements, one 32-bit word where they are 16-bit
template <class T>
__device__ __forceinline__ float2 unpack2(const Pack<T, 2>& p) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        unsigned u;
        memcpy(&u, &p, 4);
        return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    } else if constexpr (std::is_same_v<T, __half>) {
        __half2 h;
        memcpy(&h, &p, 4);
        return __half22float2(h);
    } else {
        return make_float2(p.v[0], p.v[1]);
    }
}
// the k-th pair of N elements
template <class T, int N>
__device__ __forceinline__ float2 pair_of(const Pack<T, N>& p, int k) {
    Pack<T, 2> q;
    q.v[0] = p.v[2 * k];
    q.v[1] = p.v[2 * k + 1];
    return unpack2(q);
}
// N floats rounded to T
template <class T, int N>
__device__ __forceinline__ Pack<T, N> pack_f32(const float (&v)[N]) {
    Pack<T, N> r;
    if constexpr (sizeof(T) == 2 && N % 2 == 0) {
#pragma unroll
        for (int k = 0; k < N; k += 2) {
            if constexpr (std::is_same_v<T, __half>) {
                const __half2 h = __floats2half2_rn(v[k], v[k + 1]);
                r.v[k] = h.x;
                r.v[k + 1] = h.y;
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[k], v[k + 1]);
                r.v[k] = h.x;
                r.v[k + 1] = h.y;
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) r.v[k] = from_f32<T>(v[k]);
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
