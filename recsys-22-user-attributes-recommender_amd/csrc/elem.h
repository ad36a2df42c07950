// Element types of the operators that take fp32 or bf16 storage (fp32 arithmetic either way): 16-byte vectors of either
// type as floats, and the dtype codes of the C ABI.
#pragma once
#include "common.h"

namespace asme {

enum { kF32 = 0, kBF16 = 1 };  // the `dtype` argument

template <class T>
struct Elem;
template <>
struct Elem<float> {
    static constexpr int V = 4;  // elements of a 16-byte vector
    static __device__ __forceinline__ float get(const float* p) { return *p; }
    static __device__ __forceinline__ void put(float* p, float x) { *p = x; }
    static __device__ __forceinline__ void load(const float* p, float (&x)[V]) {
        const floatx4 v = *reinterpret_cast<const floatx4*>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = v[i];
    }
    static __device__ __forceinline__ void store(float* p, const float (&x)[V]) {
        *reinterpret_cast<floatx4*>(p) = floatx4{x[0], x[1], x[2], x[3]};
    }
    static __device__ __forceinline__ void store_nt(float* p, const float (&x)[V]) {
        __builtin_nontemporal_store(floatx4{x[0], x[1], x[2], x[3]}, reinterpret_cast<floatx4*>(p));
    }
};
template <>
struct Elem<__bf16> {
    static constexpr int V = 8;
    static __device__ __forceinline__ float get(const __bf16* p) { return (float)*p; }
    static __device__ __forceinline__ void put(__bf16* p, float x) { *p = (__bf16)x; }
    static __device__ __forceinline__ void load(const __bf16* p, float (&x)[V]) {
        const bf16x8 v = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = (float)v[i];
    }
    static __device__ __forceinline__ bf16x8 pack(const float (&x)[V]) {  // round to nearest even
        bf16x8 v;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (__bf16)x[i];
        return v;
    }
    static __device__ __forceinline__ void store(__bf16* p, const float (&x)[V]) {
        *reinterpret_cast<bf16x8*>(p) = pack(x);
    }
    static __device__ __forceinline__ void store_nt(__bf16* p, const float (&x)[V]) {
        __builtin_nontemporal_store(__builtin_bit_cast(floatx4, pack(x)), reinterpret_cast<floatx4*>(p));
    }
};

inline bool dtype_ok(int dtype) { return dtype == kF32 || dtype == kBF16; }
inline int64_t dtype_size(int dtype) { return dtype == kF32 ? 4 : 2; }

// f(T{}) for the storage type of a checked dtype code
template <class F>
inline void with_dtype(int dtype, F&& f) {
    if (dtype == kF32) f(float{});
    else f(__bf16{});
}

}  // namespace asme
