// ft_counter.hpp -- the counter-based generator: random bits as a pure function of
// (seed, substream, index), the same on the GPU and on the host.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#define FT_HD __host__ __device__ __forceinline__

namespace ftc {

constexpr uint64_t kGolden = 0x9e3779b97f4a7c15ull;
constexpr uint64_t kIndexStep = 0xd1342543de82ef95ull;

FT_HD uint64_t mix64(uint64_t z)  // the splitmix64 finaliser
{
    z ^= z >> 30;
    z *= 0xbf58476d1ce4e5b9ull;
    z ^= z >> 27;
    z *= 0x94d049bb133111ebull;
    z ^= z >> 31;
    return z;
}

FT_HD uint64_t stream_key(uint64_t seed, uint32_t substream)
{
    return mix64(seed ^ (kGolden * (static_cast<uint64_t>(substream) + 1u)));
}

// 64 random bits of element `index` of `substream` under `seed`.
FT_HD uint64_t element_bits(uint64_t seed, uint32_t substream, uint64_t index)
{
    return mix64(stream_key(seed, substream) + kIndexStep * index);
}

// ---- dropout masks --------------------------------------------------------------------------
// Four neighbouring elements share one 64-bit hash (17 vector instructions), 16 bits each: a hash
// per element would cost more than the element's memory traffic. Sixteen bits alone would round the
// drop probability to multiples of 2^-16; the 48-bit number of an element is therefore its 16 bits
// followed by 32 bits of a second hash, and the second hash is only computed where the first 16 bits
// equal those of the limit (one element in 65,536).
//   h    = mix64(key + kIndexStep * (i >> 2))
//   u(i) = ((h >> 16 (i & 3)) & 0xffff) << 32 | mix64(h + kGolden * ((i & 3) + 1)) >> 32
//   dropped where u(i) < limit, limit = round(p * 2^48)
struct DropoutArgs {
    const uint64_t* seed_dev;  // the seed in device memory (it replaces key), or nullptr
    uint64_t key;              // stream_key of a seed that travels by value
    uint64_t first;            // index of the first element
    uint32_t substream;
    uint32_t hi;               // limit >> 32 (65536 for p = 1)
    uint32_t lo;               // limit & 0xffffffff
    float factor;              // what the kept elements are multiplied with
};

#ifdef __HIPCC__
__device__ __forceinline__ uint64_t dropout_key(const DropoutArgs& a)
{
    return a.seed_dev ? stream_key(*a.seed_dev, a.substream) : a.key;  // wave-uniform
}

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// The hash's argument for the group of element base + offset, offset a multiple of four. Where base is
// wave-uniform, all but two multiplies of it are scalar instructions.
__device__ __forceinline__ uint64_t group_argument(uint64_t key, uint64_t base, uint32_t offset)
{
    return key + kIndexStep * (base >> 2) + kIndexStep * static_cast<uint64_t>(offset >> 2);
}

// Which of U (4 or 8) consecutive elements stay. z: group_argument of the first one, which is element
// r of its group.
template <int U>
__device__ __forceinline__ void keep_units(bool (&keep)[U], uint64_t z, uint32_t r, const DropoutArgs& a)
{
    constexpr int G = U / 4;  // groups of four
    uint64_t w[G + 1];
#pragma unroll
    for (int g = 0; g < G; ++g) w[g] = mix64(z + kIndexStep * g);
    if (r) {  // rows of a width that is no multiple of four: the elements touch one more group
        w[G] = mix64(z + kIndexStep * G);
#pragma unroll
        for (int g = 0; g < G; ++g) w[g] = (w[g] >> (16 * r)) | (w[g + 1] << (64 - 16 * r));
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
        const uint32_t half = static_cast<uint32_t>(j & 2 ? w[j >> 2] >> 32 : w[j >> 2]);
        keep[j] = ((j & 1) ? half >> 16 : half & 0xffffu) >= a.hi;
    }
    if (a.lo == 0) return;  // wave-uniform: p is a multiple of 2^-16
    // any 16 bits equal to the limit's? (all words at once: one xor and one packed minimum each)
    const uint32_t both = (a.hi & 0xffffu) * 0x10001u;
    u16x2 least = __builtin_bit_cast(u16x2, 0xffffffffu);
#pragma unroll
    for (int g = 0; g < G; ++g) {
        least = __builtin_elementwise_min(least, __builtin_bit_cast(u16x2, static_cast<uint32_t>(w[g]) ^ both));
        least = __builtin_elementwise_min(least, __builtin_bit_cast(u16x2, static_cast<uint32_t>(w[g] >> 32) ^ both));
    }
    if (least.x != 0 && least.y != 0) return;
    uint32_t drop = 0;
#pragma clang loop unroll(disable)
    for (uint32_t j = 0; j < U; ++j) {
        const uint64_t h = mix64(z + kIndexStep * static_cast<uint64_t>((r + j) >> 2));
        const uint32_t k = (r + j) & 3u;
        const bool tie = (static_cast<uint32_t>(h >> (16 * k)) & 0xffffu) == a.hi;
        if (tie && static_cast<uint32_t>(mix64(h + kGolden * (k + 1u)) >> 32) < a.lo) drop |= 1u << j;
    }
#pragma unroll
    for (int j = 0; j < U; ++j) keep[j] = keep[j] && !(drop >> j & 1u);
}
#endif

}  // namespace ftc
