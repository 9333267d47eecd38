// ft_row_args.hpp -- argument checks and type dispatch shared by the row operators' C entries.
#pragma once

#include <cmath>
#include <numeric>
#include <type_traits>

#include "ft_counter.hpp"
#include "ft_internal.hpp"

namespace ftr {

constexpr uint64_t kMaxElements = 1ull << 46;  // of one array: far beyond the memory, far below an overflow of its bytes

inline bool valid_dtype(int dt) { return dt == FT_F32 || dt == FT_F16 || dt == FT_BF16; }

inline bool aligned_to(const void* p, int dt) { return reinterpret_cast<uintptr_t>(p) % (dt == FT_F32 ? 4 : 2) == 0; }

// Rows of a call's array.
struct Rows {
    const void* base;
    int dtype;
    uint64_t rows, stride, cols;

    uint64_t bytes(uint64_t elements) const { return elements * (dtype == FT_F32 ? 4 : 2); }
};

// Whether the arrays share a byte. Rows that lie apart may lie between each other (two slices of one tensor): all begins of
// rows differ by multiples of the distances' common divisor, so that the rows are compared modulo that. Exact where the
// distances are equal; arrays interleaved at different distances count as apart only if that shows it.
inline bool overlap(const Rows& a, const Rows& b)
{
    if (a.rows == 0 || b.rows == 0 || a.cols == 0 || b.cols == 0) return false;
    const uintptr_t a0 = reinterpret_cast<uintptr_t>(a.base), b0 = reinterpret_cast<uintptr_t>(b.base);
    const uint64_t a_step = a.rows > 1 ? a.bytes(a.stride) : 0, b_step = b.rows > 1 ? b.bytes(b.stride) : 0;
    const uint64_t a_row = a.bytes(a.cols), b_row = b.bytes(b.cols);
    if (a0 + (a.rows - 1) * a_step + a_row <= b0 || b0 + (b.rows - 1) * b_step + b_row <= a0) return false;
    const uint64_t step = std::gcd(a_step, b_step);
    if (step == 0) return true;  // one row each (a row that is repeated is one)
    const uint64_t apart = b0 >= a0 ? (b0 - a0) % step : (step - (a0 - b0) % step) % step;
    return apart < a_row || apart + b_row > step;
}

// The same elements at the same places: may be read and written by one call.
inline bool same_rows(const Rows& a, const Rows& b)
{
    return a.base == b.base && a.dtype == b.dtype && a.rows == b.rows && a.cols == b.cols && (a.rows <= 1 || a.stride == b.stride);
}

// fn(std::integral_constant<int, dtype code>) for a valid dtype code.
template <typename F>
inline int with_dtype(int dt, F fn)
{
    switch (dt) {
        case FT_F32: return fn(std::integral_constant<int, FT_F32>{});
        case FT_F16: return fn(std::integral_constant<int, FT_F16>{});
        default: return fn(std::integral_constant<int, FT_BF16>{});
    }
}

// What the kernels take: factor = scale / (1 - p), rounded once.
inline int dropout_args(const ft_dropout_t* d, double scale, ftc::DropoutArgs* out)
{
    if (!(d->p >= 0.0 && d->p <= 1.0)) return fth::fail(FT_EINVAL, "the drop probability must lie in [0, 1], not %g", d->p);
    if (reinterpret_cast<uintptr_t>(d->seed_dev) % 8) return fth::fail(FT_EALIGN, "seed_dev is not aligned to 8 bytes");
    const uint64_t limit = static_cast<uint64_t>(std::nearbyint(d->p * 281474976710656.0));  // 2^48
    out->seed_dev = static_cast<const uint64_t*>(d->seed_dev);
    out->key = ftc::stream_key(d->seed, d->substream);
    out->first = d->first_index;
    out->substream = d->substream;
    out->hi = static_cast<uint32_t>(limit >> 32);
    out->lo = static_cast<uint32_t>(limit);
    out->factor = d->p < 1.0 ? static_cast<float>(scale / (1.0 - d->p)) : 0.0f;
    return FT_OK;
}

}  // namespace ftr
