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
// Four neighbouring elements share one 64-bit hash, 16 bits each: a hash is six 32-bit multiplies,
// which run at a quarter of the rate of simple operations, so one per element would cost more than
// the element's memory traffic. Sixteen bits alone would round the drop probability to multiples of
// 2^-16; the 48-bit number of an element is therefore its 16 bits followed by 32 bits of a second
// hash, and the second hash is only computed where the first 16 bits equal those of the limit (one
// element in 65,536).
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

// Which of the eight elements i ... i + 7 stay.
__device__ __forceinline__ void keep8(bool (&keep)[8], uint64_t key, uint64_t i, uint32_t hi, uint32_t lo)
{
    const uint64_t z = key + kIndexStep * (i >> 2);
    uint64_t w0 = mix64(z), w1 = mix64(z + kIndexStep);
    const uint32_t r = static_cast<uint32_t>(i) & 3u;
    if (r) {  // rows of a width that is no multiple of four: the eight elements touch a third group
        const uint64_t w2 = mix64(z + 2 * kIndexStep);
        w0 = (w0 >> (16 * r)) | (w1 << (64 - 16 * r));
        w1 = (w1 >> (16 * r)) | (w2 << (64 - 16 * r));
    }
    const uint32_t w[4] = {static_cast<uint32_t>(w0), static_cast<uint32_t>(w0 >> 32), static_cast<uint32_t>(w1),
                           static_cast<uint32_t>(w1 >> 32)};
    uint32_t tie = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t u = (j & 1) ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu;
        keep[j] = u >= hi;
        if (u == hi) tie |= 1u << j;
    }
    if (lo != 0 && tie != 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (!(tie >> j & 1u)) continue;
            const uint64_t e = i + static_cast<uint64_t>(j);
            const uint64_t h = mix64(key + kIndexStep * (e >> 2));
            keep[j] = static_cast<uint32_t>(mix64(h + kGolden * ((e & 3u) + 1u)) >> 32) >= lo;
        }
    }
}
#endif

}  // namespace ftc
