// ft_row_args.hpp -- argument checks and type dispatch shared by the row operators' C entries.
#pragma once

#include <cmath>
#include <type_traits>

#include "ft_counter.hpp"
#include "ft_internal.hpp"

namespace ftr {

constexpr uint64_t kMaxElements = 1ull << 46;  // of one array: far beyond the memory, far below an overflow of its bytes

inline bool valid_dtype(int dt) { return dt == FT_F32 || dt == FT_F16 || dt == FT_BF16; }

inline bool aligned_to(const void* p, int dt) { return reinterpret_cast<uintptr_t>(p) % (dt == FT_F32 ? 4 : 2) == 0; }

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
