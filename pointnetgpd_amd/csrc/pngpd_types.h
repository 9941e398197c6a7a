// 16-bit storage types of the training operators: values are widened to float32 on load and rounded once
// (to nearest, ties to even) on store.
#pragma once
#include "pngpd_common.h"

typedef unsigned short u16;

// one value, type known at run time (dt: PNGPD_BF16 or PNGPD_F16)
__device__ __forceinline__ float half_to_f(int dt, u16 b) {
    return dt == PNGPD_BF16 ? __uint_as_float((unsigned)b << 16) : (float)__builtin_bit_cast(_Float16, b);
}
__device__ __forceinline__ u16 f_to_half(int dt, float x) {
    return dt == PNGPD_BF16 ? __builtin_bit_cast(u16, (__bf16)x) : __builtin_bit_cast(u16, (_Float16)x);
}

// one value, type known at compile time (DT: PNGPD_F32, PNGPD_BF16, PNGPD_F16)
template <int DT> struct elem { typedef u16 t; };
template <> struct elem<PNGPD_F32> { typedef float t; };
template <int DT> __device__ __forceinline__ float ld_elem(const typename elem<DT>::t *p) {
    if constexpr (DT == PNGPD_F32) return *p;
    else return half_to_f(DT, *p);
}
template <int DT> __device__ __forceinline__ void st_elem(typename elem<DT>::t *p, float x) {
    if constexpr (DT == PNGPD_F32) *p = x;
    else *p = f_to_half(DT, x);
}

// two values to a dword (the first in the low half): one instruction for the pair where single conversions take one each and
// the merging
typedef __bf16 pk_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 pk_f16x2 __attribute__((ext_vector_type(2)));
template <int DT> __device__ __forceinline__ unsigned pk_half(float a, float b) {
    const f32x2 v = {a, b};
    if constexpr (DT == PNGPD_BF16) return __builtin_bit_cast(unsigned, __builtin_convertvector(v, pk_bf16x2));
    else return __builtin_bit_cast(unsigned, __builtin_convertvector(v, pk_f16x2));
}
