// ft_rows.hpp -- a few consecutive elements of a row in registers: what a lane of the row operators
// (embedding lookup, its gradient, dropout) moves at a time.
#pragma once

#include <type_traits>

#include "ft_vec.hpp"

namespace ftk {

// Elements a lane moves at a time: 16 bytes of the widest type it touches, so that a wavefront's
// access is one contiguous KiB of that array. (Eight elements of an fp32 array per lane, two 16-byte
// accesses 32 bytes apart from lane to lane, took 460 us for the lookup of 32,768 rows of 8192 fp16
// elements into fp32.)
template <int A, int B>
constexpr int row_unit() { return A == FT_F32 || B == FT_F32 ? 4 : 8; }

// The vector types promise the alignment of one element only: the hardware takes 16-byte accesses
// at any address, so rows of an odd width need no code of their own.
template <int DT, int U>
struct RowVec {
    typedef uint16_t type __attribute__((ext_vector_type(U), aligned(2)));
};
template <int U>
struct RowVec<FT_F32, U> {
    typedef float type __attribute__((ext_vector_type(U), aligned(4)));
};

// Raw bits of U elements as they come from memory, so that several loads can be in flight before the
// first conversion waits for one.
template <int DT, int U>
using RowBits = typename RowVec<DT, U>::type;

template <int DT>
using RowElement = typename std::conditional<DT == FT_F32, float, uint16_t>::type;

template <int DT, int U, bool NT>
__device__ __forceinline__ RowBits<DT, U> row_load(const void* base, uint64_t i)
{
    const RowBits<DT, U>* p = reinterpret_cast<const RowBits<DT, U>*>(static_cast<const RowElement<DT>*>(base) + i);
    if constexpr (NT)
        return __builtin_nontemporal_load(p);
    else
        return *p;
}

// The first `count` (below U) of U elements; the others read as zero.
template <int DT, int U>
__device__ __forceinline__ RowBits<DT, U> row_load_some(const void* base, uint64_t i, uint32_t count)
{
    RowBits<DT, U> r;
#pragma unroll
    for (uint32_t k = 0; k < U; ++k) r[k] = k < count ? static_cast<const RowElement<DT>*>(base)[i + k] : static_cast<RowElement<DT>>(0);
    return r;
}

template <int DT, int U>
__device__ __forceinline__ void row_floats(float (&x)[U], const RowBits<DT, U>& r)
{
#pragma unroll
    for (int k = 0; k < U; ++k) {
        if constexpr (DT == FT_F32)
            x[k] = r[k];
        else
            x[k] = half_to_float<DT>(r[k]);
    }
}

template <int DT, int U>
__device__ __forceinline__ RowBits<DT, U> row_round(const float (&x)[U])
{
    RowBits<DT, U> r;
    if constexpr (DT == FT_F32) {
#pragma unroll
        for (int k = 0; k < U; ++k) r[k] = x[k];
    } else {
        typedef uint32_t words __attribute__((ext_vector_type(U / 2)));
        words w;
#pragma unroll
        for (int k = 0; k < U / 2; ++k) w[k] = pack2<DT>(x[2 * k], x[2 * k + 1]);
        r = __builtin_bit_cast(decltype(r), w);
    }
    return r;
}

template <int DT, int U, bool NT>
__device__ __forceinline__ void row_store(void* base, uint64_t i, const float (&x)[U])
{
    RowBits<DT, U>* p = reinterpret_cast<RowBits<DT, U>*>(static_cast<RowElement<DT>*>(base) + i);
    const RowBits<DT, U> r = row_round<DT, U>(x);
    if constexpr (NT)
        __builtin_nontemporal_store(r, p);
    else
        *p = r;
}

template <int DT, int U>
__device__ __forceinline__ void row_store_some(void* base, uint64_t i, const float (&x)[U], uint32_t count)
{
    const RowBits<DT, U> r = row_round<DT, U>(x);
#pragma unroll
    for (uint32_t k = 0; k < U; ++k)
        if (k < count) static_cast<RowElement<DT>*>(base)[i + k] = r[k];
}

}  // namespace ftk
