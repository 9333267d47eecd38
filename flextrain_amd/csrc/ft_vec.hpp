// ft_vec.hpp -- vector types and 16-bit <-> 32-bit conversions shared by the kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ft_adam.h"

namespace ftk {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// ---- 16-bit <-> 32-bit helpers ------------------------------------------------------------
template <int DT>
__device__ __forceinline__ float half_to_float(uint32_t bits16);
template <>
__device__ __forceinline__ float half_to_float<FT_BF16>(uint32_t b)
{
    return __builtin_bit_cast(float, b << 16);
}
template <>
__device__ __forceinline__ float half_to_float<FT_F16>(uint32_t b)
{
    return (float)__builtin_bit_cast(_Float16, (uint16_t)b);
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<FT_BF16>(float lo, float hi)
{
    f32x2 x = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
}
template <>
__device__ __forceinline__ uint32_t pack2<FT_F16>(float lo, float hi)
{
    f32x2 x = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, f16x2));
}

}  // namespace ftk
