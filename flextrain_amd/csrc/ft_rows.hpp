// ft_rows.hpp -- eight consecutive elements of a row in registers: what a lane of the row operators
// (embedding lookup, its gradient, dropout) moves at a time.
#pragma once

#include "ft_vec.hpp"

namespace ftk {

// The vector types promise the alignment of one element only: the hardware takes 16-byte accesses
// at any address, so rows of an odd width need no code of their own.
typedef float row_f32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t row_u16x8 __attribute__((ext_vector_type(8), aligned(2)));

constexpr int kRowUnit = 8;  // elements a lane moves at a time

template <int DT>
__device__ __forceinline__ float row_load1(const void* base, uint64_t i)
{
    if constexpr (DT == FT_F32)
        return static_cast<const float*>(base)[i];
    else
        return half_to_float<DT>(static_cast<const uint16_t*>(base)[i]);
}

template <int DT>
__device__ __forceinline__ void row_store1(void* base, uint64_t i, float x)
{
    if constexpr (DT == FT_F32)
        static_cast<float*>(base)[i] = x;
    else
        static_cast<uint16_t*>(base)[i] = static_cast<uint16_t>(pack2<DT>(x, x));
}

// Raw bits of eight elements as they come from memory, so that several loads can be in flight
// before the first conversion waits for one.
template <int DT>
struct RowBits {
    row_u16x8 w;
};
template <>
struct RowBits<FT_F32> {
    row_f32x4 a, b;
};

template <int DT, bool NT>
__device__ __forceinline__ RowBits<DT> row_load8(const void* base, uint64_t i)
{
    RowBits<DT> r;
    if constexpr (DT == FT_F32) {
        const row_f32x4* p = reinterpret_cast<const row_f32x4*>(static_cast<const float*>(base) + i);
        if constexpr (NT) {
            r.a = __builtin_nontemporal_load(p);
            r.b = __builtin_nontemporal_load(p + 1);
        } else {
            r.a = p[0];
            r.b = p[1];
        }
    } else {
        const row_u16x8* p = reinterpret_cast<const row_u16x8*>(static_cast<const uint16_t*>(base) + i);
        if constexpr (NT)
            r.w = __builtin_nontemporal_load(p);
        else
            r.w = *p;
    }
    return r;
}

// The first `count` (1 ... 7) of eight elements; the others read as zero.
template <int DT>
__device__ __forceinline__ RowBits<DT> row_load_some(const void* base, uint64_t i, uint32_t count)
{
    RowBits<DT> r;
    if constexpr (DT == FT_F32) {
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            r.a[k] = k < count ? static_cast<const float*>(base)[i + k] : 0.0f;
            r.b[k] = k + 4 < count ? static_cast<const float*>(base)[i + 4 + k] : 0.0f;
        }
    } else {
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) r.w[k] = k < count ? static_cast<const uint16_t*>(base)[i + k] : static_cast<uint16_t>(0);
    }
    return r;
}

template <int DT>
__device__ __forceinline__ void row_floats(float (&x)[kRowUnit], const RowBits<DT>& r)
{
#pragma unroll
    for (int k = 0; k < kRowUnit; ++k) {
        if constexpr (DT == FT_F32)
            x[k] = k < 4 ? r.a[k & 3] : r.b[k & 3];
        else
            x[k] = half_to_float<DT>(r.w[k]);
    }
}

template <int DT, bool NT>
__device__ __forceinline__ void row_store8(void* base, uint64_t i, const float (&x)[kRowUnit])
{
    if constexpr (DT == FT_F32) {
        row_f32x4* p = reinterpret_cast<row_f32x4*>(static_cast<float*>(base) + i);
        const row_f32x4 a = {x[0], x[1], x[2], x[3]}, b = {x[4], x[5], x[6], x[7]};
        if constexpr (NT) {
            __builtin_nontemporal_store(a, p);
            __builtin_nontemporal_store(b, p + 1);
        } else {
            p[0] = a;
            p[1] = b;
        }
    } else {
        const u32x4 w = {pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]), pack2<DT>(x[4], x[5]), pack2<DT>(x[6], x[7])};
        row_u16x8* p = reinterpret_cast<row_u16x8*>(static_cast<uint16_t*>(base) + i);
        if constexpr (NT)
            __builtin_nontemporal_store(__builtin_bit_cast(row_u16x8, w), p);
        else
            *p = __builtin_bit_cast(row_u16x8, w);
    }
}

template <int DT>
__device__ __forceinline__ void row_store_some(void* base, uint64_t i, const float (&x)[kRowUnit], uint32_t count)
{
#pragma unroll
    for (uint32_t k = 0; k < kRowUnit; ++k)
        if (k < count) row_store1<DT>(base, i + k, x[k]);
}

}  // namespace ftk
