// Element types of the operators that take more than f32 (nrf_dtype): loads of VW neighbouring elements as f32, stores with one
// rounding (to nearest, ties to even).  A vector access needs its address aligned to an element only.
#pragma once
#include "nrf_common.h"

namespace nrf {

struct bf16_t { uint16_t bits; };
struct f16_t { uint16_t bits; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return __uint_as_float((uint32_t)v.bits << 16); }
__device__ __forceinline__ float to_f32(f16_t v) { return (float)__builtin_bit_cast(_Float16, v.bits); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16_t from_f32<bf16_t>(float v) { return bf16_t{__builtin_bit_cast(uint16_t, (__bf16)v)}; }
template <> __device__ __forceinline__ f16_t from_f32<f16_t>(float v) { return f16_t{__builtin_bit_cast(uint16_t, (_Float16)v)}; }

template <typename T, int VW> struct __attribute__((packed, aligned(sizeof(T)))) Pack { T e[VW]; };

inline int dtype_size(int32_t t) { return t == NRF_F32 ? 4 : (t == NRF_BF16 || t == NRF_F16) ? 2 : 0; }

}  // namespace nrf
