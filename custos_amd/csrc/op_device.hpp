// Device-side helpers of the operators that are compiled with the library (group_norm.hip,
// policy_loss.hip): vectors of storage elements, conversions to the f32 they are computed in, sums
// over a workgroup.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace custos_hip {

typedef unsigned long long u64;

// 16 bytes of T, at any address that is a multiple of sizeof(T): rows of odd length start anywhere, and
// the global loads and stores of gfx950 take any alignment.
template <class T>
struct VecOf {
    static constexpr int elems = 16 / sizeof(T);
};

template <class T, int V>
struct Pack {
    T v[V];
};

template <int BYTES, int ALIGN>
struct Raw;
#define CUSTOS_RAW(BYTES, ALIGN, ...)                             \
    template <>                                                   \
    struct Raw<BYTES, ALIGN> {                                    \
        typedef __VA_ARGS__ base;                                 \
        typedef base type __attribute__((aligned(ALIGN)));        \
    };
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
CUSTOS_RAW(16, 4, u32x4)
CUSTOS_RAW(16, 2, u32x4)
CUSTOS_RAW(8, 1, u32x2)
CUSTOS_RAW(4, 4, unsigned int)
CUSTOS_RAW(4, 1, unsigned int)
CUSTOS_RAW(2, 2, unsigned short)
CUSTOS_RAW(1, 1, unsigned char)
#undef CUSTOS_RAW

// V elements at p; `STREAM`: past the caches (what is not read again soon).
template <bool STREAM, class T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
    using R = Raw<V * sizeof(T), sizeof(T)>;
    const typename R::type* q = reinterpret_cast<const typename R::type*>(p);
    typename R::base bits;
    if (STREAM) bits = __builtin_nontemporal_load(q);
    else bits = *q;
    using Out = Pack<T, V>;
    return __builtin_bit_cast(Out, bits);
}
template <bool STREAM, class T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& pack) {
    using R = Raw<V * sizeof(T), sizeof(T)>;
    typename R::type* q = reinterpret_cast<typename R::type*>(p);
    const typename R::base bits = __builtin_bit_cast(typename R::base, pack);
    if (STREAM) __builtin_nontemporal_store(bits, q);
    else *q = bits;
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(_Float16 x) { return static_cast<float>(x); }
__device__ __forceinline__ float to_f32(__bf16 x) { return static_cast<float>(x); }
// one rounding, to nearest even
template <class T>
__device__ __forceinline__ T from_f32(float x) {
    return static_cast<T>(x);
}

// Makes the compiler forget what it knows of a held value, so that it converts the stored bits again where
// they are used next instead of keeping the converted values, which take twice the registers or more.
__device__ __forceinline__ void forget(u32x4& v) {
    unsigned int a = v[0], b = v[1], c = v[2], d = v[3];
    __asm__("" : "+v"(a), "+v"(b), "+v"(c), "+v"(d));
    v = u32x4{a, b, c, d};
}
__device__ __forceinline__ void forget(u32x2& v) {
    unsigned int a = v[0], b = v[1];
    __asm__("" : "+v"(a), "+v"(b));
    v = u32x2{a, b};
}
__device__ __forceinline__ void forget(unsigned int& v) { __asm__("" : "+v"(v)); }
__device__ __forceinline__ void forget(unsigned short&) {}
__device__ __forceinline__ void forget(unsigned char&) {}

// A vector as it is stored.
template <class T, int V>
struct Bits {
    using Storage = typename Raw<V * sizeof(T), sizeof(T)>::base;
    Storage bits;
    // STREAM: past the caches (what is not read again soon)
    template <bool STREAM = false>
    __device__ __forceinline__ void load(const T* p) {
        using Any = typename Raw<V * sizeof(T), sizeof(T)>::type;
        if (STREAM) bits = __builtin_nontemporal_load(reinterpret_cast<const Any*>(p));
        else bits = *reinterpret_cast<const Any*>(p);
    }
    __device__ __forceinline__ void zero() { bits = Storage(0); }
    __device__ __forceinline__ void forget_values() { forget(bits); }
    __device__ __forceinline__ Pack<T, V> pack() const {
        using Out = Pack<T, V>;
        return __builtin_bit_cast(Out, bits);
    }
};

// Sum over a wavefront, in every lane (a fixed tree: results do not depend on timing).
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int step = 32; step > 0; step /= 2) v += __shfl_xor(v, step, 64);
    return v;
}
__device__ __forceinline__ double lanes_sum_f64(double v) {
#pragma unroll
    for (int step = 32; step > 0; step /= 2) v += __shfl_xor(v, step, 64);
    return v;
}

}  // namespace custos_hip
