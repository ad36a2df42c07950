// Element types of the operators that take fp32 or bf16 storage (fp32 arithmetic either way): 16-byte vectors of either
// type as floats, sums over lanes, and the dtype codes of the C ABI.
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

template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
    return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, true));
}
// sum over aligned groups of N lanes, in every lane (quad permutes, then mirrors of 8 and 16 lanes whose quads agree)
template <int N>
__device__ __forceinline__ float group_sum(float x) {
    if constexpr (N >= 2) x = dpp_add<0xB1>(x);   // quad_perm 1 0 3 2
    if constexpr (N >= 4) x = dpp_add<0x4E>(x);   // quad_perm 2 3 0 1
    if constexpr (N >= 8) x = dpp_add<0x141>(x);  // row_half_mirror
    if constexpr (N >= 16) x = dpp_add<0x140>(x); // row_mirror
    if constexpr (N >= 32) x += __shfl_xor(x, 16, 64);
    if constexpr (N >= 64) x += __shfl_xor(x, 32, 64);
    return x;
}

inline bool dtype_ok(int dtype) { return dtype == kF32 || dtype == kBF16; }
inline int64_t dtype_size(int dtype) { return dtype == kF32 ? 4 : 2; }

// on 16-byte boundaries (null is)
inline bool aligned(std::initializer_list<const void*> ps) {
    for (const void* p : ps)
        if ((uintptr_t)p & 15) return false;
    return true;
}

// f(T{}) for the storage type of a checked dtype code
template <class F>
inline void with_dtype(int dtype, F&& f) {
    if (dtype == kF32) f(float{});
    else f(__bf16{});
}

}  // namespace asme
