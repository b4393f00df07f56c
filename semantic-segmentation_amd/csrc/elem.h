// Element types of the operators that take bf16 (0), fp32 (1) and fp16 (2) tensors.
#pragma once
#include "common.h"

// Vectors of 16 bytes whose address is only aligned to the element: a tensor may start at any element, and a row of an odd
// number of classes moves the next row off every other boundary.  gfx950 does unaligned global accesses in hardware (the
// amdhsa target enables them); the compiler emits one wide access.
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef u16 u16x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef u16 u16x8u __attribute__((ext_vector_type(8), aligned(2)));

template <int DT> struct Elem;
template <> struct Elem<0> {
    typedef u16 T; typedef u16x8u V; typedef u16x4u V4;
    static constexpr int N = 8;
    static __device__ __forceinline__ float up(u16 x) { return __uint_as_float((uint32_t)x << 16); }
    static __device__ __forceinline__ u16 down(float x) { return (u16)f2bf_bits(x); }
};
template <> struct Elem<1> {
    typedef float T; typedef f32x4u V; typedef f32x4u V4;
    static constexpr int N = 4;
    static __device__ __forceinline__ float up(float x) { return x; }
    static __device__ __forceinline__ float down(float x) { return x; }
};
template <> struct Elem<2> {
    typedef u16 T; typedef u16x8u V; typedef u16x4u V4;
    static constexpr int N = 8;
    static __device__ __forceinline__ float up(u16 x) { return (float)__builtin_bit_cast(_Float16, x); }
    static __device__ __forceinline__ u16 down(float x) { return __builtin_bit_cast(u16, (_Float16)x); }
};
