// ft_embedding.hip -- rows of an embedding table: the lookup, and its gradient added into an accumulator.
//
//   lookup    out[i] = f * table[token[i] - first_row], zero where the token lies outside the table
//   gradient  acc[v] (+)= f * sum of g[i] over the tokens i with row v
// with f = scale / (1 - p) and, where p > 0, the dropout mask of ft_counter.hpp on the rows of out / g.
//
// Both are HBM-bound. The gradient must not depend on the order in which workgroups run, so nothing
// is added with atomics: the tokens are sorted by row (stably: equal rows keep the order of their
// positions), every wavefront sums a run of consecutive sorted tokens in registers, and runs that
// cross the edge of a wavefront or a workgroup are joined in a fixed order.
#include <atomic>
#include <type_traits>

#include "ft_counter.hpp"
#include "ft_internal.hpp"
#include "ft_row_args.hpp"
#include "ft_rows.hpp"

namespace {

using namespace ftk;

constexpr int kLanes = 64;
constexpr uint32_t kNoRow = 0xffffffffu;
constexpr uint64_t kMaxCount = 0x7fffffffull;  // tokens of a call, rows of a table
constexpr uint64_t kMaxCols = 1ull << 24;      // elements of a row
constexpr uint64_t kMaxReach = 1ull << 38;     // ids from the first to the last token of either dimension: more than the memory holds

// Token i of a call: id at outer index i / inner, inner index i % inner.
struct Tokens {
    const void* ids;
    uint64_t outer_stride, inner_stride;
    uint64_t first_row;
    int64_t padding;
    uint32_t n, inner;
    uint32_t rows;
    int32_t wide;  // 64-bit ids

    // The row of the table, kNoRow for a token outside it.
    __device__ __forceinline__ uint32_t row(uint32_t i) const
    {
        uint64_t at;
        if (inner == n) {
            at = i * inner_stride;
        } else {
            const uint32_t o = i / inner;
            at = o * outer_stride + (i - o * inner) * inner_stride;
        }
        return row_of(wide ? static_cast<const int64_t*>(ids)[at] : static_cast<int64_t>(static_cast<const int32_t*>(ids)[at]));
    }

    __device__ __forceinline__ uint32_t row_of(int64_t id) const
    {
        const uint64_t r = static_cast<uint64_t>(id) - first_row;
        return r < rows && id != padding ? static_cast<uint32_t>(r) : kNoRow;
    }
};

// The rows of the tokens base + 64 r (base: a lane's first token), kNoRow behind the last. All ids are
// fetched before the first is looked at: one wait for all of them.
template <int ITEMS>
__device__ __forceinline__ void load_rows(uint32_t (&key)[ITEMS], const Tokens& t, uint32_t base)
{
    auto fetch = [&](auto element) {
        using T = decltype(element);
        T id[ITEMS];
        const T* ids = static_cast<const T*>(t.ids);
#pragma unroll
        for (int r = 0; r < ITEMS; ++r) {
            const uint32_t i = base + r * kLanes;
            id[r] = ids[i < t.n ? i : t.n - 1];
        }
#pragma unroll
        for (int r = 0; r < ITEMS; ++r) key[r] = base + r * kLanes < t.n ? t.row_of(id[r]) : kNoRow;
    };
    if (t.inner == t.n && t.inner_stride == 1) {
        if (t.wide)
            fetch(int64_t{});
        else
            fetch(int32_t{});
    } else {
#pragma unroll
        for (int r = 0; r < ITEMS; ++r) key[r] = base + r * kLanes < t.n ? t.row(base + r * kLanes) : kNoRow;
    }
}

// ---- lookup -----------------------------------------------------------------------------------
struct LookupPass {
    Tokens tokens;
    const void* table;
    void* out;
    uint64_t table_stride, out_stride;
    uint32_t cols;
    uint32_t chunks;  // wavefronts per token (LPR == 64)
    float factor;
    ftc::DropoutArgs drop;
};

// LPR lanes per row. 64: a wavefront takes K units per lane of one token's row; fewer: one unit per
// lane, several tokens per wavefront, for rows too short to feed 64 lanes (32,768 rows of 256 bf16 elements: 5.0 us
// instead of 6.9). HBM-bound: 6.2 TB/s for 16,376 rows of 4096 bf16 elements, 6.6 TB/s into fp32. The result is
// stored past the caches (46 us instead of 29 without that), the table is read through them: frequent
// rows are met again (44 us past them).
template <int TT, int OT, bool DROP, int LPR, int K>
__global__ __launch_bounds__(256) void embedding_lookup_kernel(LookupPass a)
{
    constexpr int U = row_unit<TT, OT>();
    const uint32_t wave = blockIdx.x * 4u + (threadIdx.x >> 6), lane = threadIdx.x & 63u;
    uint32_t token, col;
    if constexpr (LPR == kLanes) {
        const uint32_t w = __builtin_amdgcn_readfirstlane(wave);
        token = w / a.chunks;
        col = ((w - token * a.chunks) * K * kLanes + lane) * U;
    } else {
        token = wave * (kLanes / LPR) + lane / LPR;
        col = (lane % LPR) * U;
    }
    if (token >= a.tokens.n) return;
    const uint32_t row = a.tokens.row(token);
    const uint64_t from = static_cast<uint64_t>(row) * a.table_stride, to = token * a.out_stride;
    RowBits<TT, U> bits[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const uint32_t c = col + k * kLanes * U;
        if (row == kNoRow || c >= a.cols) continue;
        bits[k] = a.cols - c >= U ? row_load<TT, U, false>(a.table, from + c) : row_load_some<TT, U>(a.table, from + c, a.cols - c);
    }
    uint64_t key = 0;
    if constexpr (DROP) key = ftc::dropout_key(a.drop);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const uint32_t c = col + k * kLanes * U;
        if (c >= a.cols) continue;
        float x[U] = {};
        if (row != kNoRow) {
            row_floats<TT, U>(x, bits[k]);
            bool keep[U];
            if constexpr (DROP) {
                const uint64_t b = a.drop.first + static_cast<uint64_t>(token) * a.cols;
                ftc::keep_units<U>(keep, ftc::group_argument(key, b, c), static_cast<uint32_t>(b) & 3u, a.drop);
            }
#pragma unroll
            for (int j = 0; j < U; ++j) {
                x[j] *= a.factor;
                if constexpr (DROP) x[j] = keep[j] ? x[j] : 0.0f;
            }
        }
        if (a.cols - c >= U)
            row_store<OT, U, true>(a.out, to + c, x);
        else
            row_store_some<OT, U>(a.out, to + c, x, a.cols - c);
    }
}

template <int TT, int OT, bool DROP>
int launch_lookup(LookupPass a, hipStream_t stream)
{
    constexpr int U = row_unit<TT, OT>();
    const uint32_t units = (a.cols + U - 1) / U;
    auto go = [&](auto lpr, auto k) -> int {
        constexpr int LPR = decltype(lpr)::value, K = decltype(k)::value;
        a.chunks = (units + kLanes * K - 1) / (kLanes * K);
        const uint64_t waves = LPR == kLanes ? static_cast<uint64_t>(a.tokens.n) * a.chunks
                                             : (static_cast<uint64_t>(a.tokens.n) * LPR + kLanes - 1) / kLanes;
        const uint64_t groups = (waves + 3) / 4;
        if (groups > 0xffffffull) return fth::fail(FT_EINVAL, "%u tokens of %u elements are too many for one call", a.tokens.n, a.cols);
        hipLaunchKernelGGL((embedding_lookup_kernel<TT, OT, DROP, LPR, K>), dim3(static_cast<unsigned>(groups)), dim3(256), 0, stream, a);
        FT_HIP(hipGetLastError());
        return FT_OK;
    };
    using std::integral_constant;
    if (units <= 16) return go(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    if (units <= 32) return go(integral_constant<int, 32>{}, integral_constant<int, 1>{});
    // 16,376 rows of 4096 bf16 elements, one / two / four units per lane: 29 / 32 / 32 us; with dropout 45 / 33 / 33 us;
    // 32,768 rows of 8192 fp16 elements into fp32: 268 / 202 / 226 us. Few rows need every wavefront they can get.
    const bool few = static_cast<uint64_t>(a.tokens.n) * ((units + kLanes - 1) / kLanes) < 16384;
    if (few || (U == 8 && !DROP)) return go(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    return go(integral_constant<int, 64>{}, integral_constant<int, 2>{});
}

// ---- gradient ---------------------------------------------------------------------------------
struct GradPass {
    Tokens tokens;
    const void* g;
    void* acc;
    uint64_t g_stride, acc_stride;
    uint32_t cols;
    int32_t accumulate;
    float factor;
    ftc::DropoutArgs drop;
    // sorted tokens (long calls)
    const uint32_t* row_s;   // tokens outside the table last, as row tokens.rows
    const uint32_t* pos_s;
    float* head;             // [groups][padded cols]: the end of a run that began in an earlier workgroup
    float* tail;             // the beginning of a run that goes on in the next one
    uint32_t rotate;         // the rows' order is that of their numbers rotated right by this many bits
    uint32_t per_wave;       // sorted tokens per wavefront
    uint32_t groups;         // workgroups per block of columns
    uint32_t padded;         // columns rounded up to whole blocks
};

// RAGGED: rows whose width is no multiple of U, the last unit of a row has `count` elements. Kernels without it
// have no second way to load a unit, and the loads of several tokens are issued one behind the other; with it the
// compiler waits for each (128 equal tokens of 4096 elements: 38 us instead of 21).
template <int DT, int U, bool NT, bool RAGGED>
__device__ __forceinline__ RowBits<DT, U> load_unit(const void* base, uint64_t at, uint32_t count)
{
    if constexpr (RAGGED) {
        if (count != U) return row_load_some<DT, U>(base, at, count);
    }
    return row_load<DT, U, NT>(base, at);
}

// Adds the gradient's unit of token `pos` at column `col`, masked.
template <int GT, int U, bool DROP>
__device__ __forceinline__ void add_unit(float (&sum)[U], const RowBits<GT, U>& bits, const GradPass& a, uint64_t key, uint32_t pos, uint32_t col)
{
    float x[U];
    row_floats<GT, U>(x, bits);
    if constexpr (DROP) {
        bool keep[U];
        const uint64_t b = a.drop.first + static_cast<uint64_t>(pos) * a.cols;
        ftc::keep_units<U>(keep, ftc::group_argument(key, b, col), static_cast<uint32_t>(b) & 3u, a.drop);
#pragma unroll
        for (int j = 0; j < U; ++j) sum[j] += keep[j] ? x[j] : 0.0f;
    } else {
#pragma unroll
        for (int j = 0; j < U; ++j) sum[j] += x[j];
    }
}

// acc[row] = [old +] factor * sum: the one rounding to the accumulator's type. The product is rounded to fp32 before the
// addition, as a gradient that is written and then added is: a fused multiply-add would keep the rounding of the factor, and
// sums on the border between two 16-bit numbers would all go to the same side.
template <int AT, int U, bool RAGGED>
__device__ __forceinline__ void finish_unit(const GradPass& a, uint32_t row, uint32_t col, uint32_t count, const float (&sum)[U],
                                            const RowBits<AT, U>& old)
{
    const uint64_t at = static_cast<uint64_t>(row) * a.acc_stride + col;
    float x[U];
#pragma unroll
    for (int j = 0; j < U; ++j) x[j] = sum[j] * a.factor;
    if (a.accumulate) {
        float before[U];
        row_floats<AT, U>(before, old);
#pragma unroll
        for (int j = 0; j < U; ++j) x[j] = before[j] + x[j];
    }
    if constexpr (RAGGED) {
        if (count != U) {
            row_store_some<AT, U>(a.acc, at, x, count);
            return;
        }
    }
    row_store<AT, U, true>(a.acc, at, x);
}

template <int AT, int U, bool RAGGED>
__device__ __forceinline__ RowBits<AT, U> load_old(const GradPass& a, uint32_t row, uint32_t col, uint32_t count)
{
    RowBits<AT, U> old{};
    if (a.accumulate) old = load_unit<AT, U, false, RAGGED>(a.acc, static_cast<uint64_t>(row) * a.acc_stride + col, count);
    return old;
}

// ---- sorting the tokens by row ------------------------------------------------------------------
// Stable: tokens of one row keep their order, so that sums do not depend on how workgroups run. Which
// order the rows have among each other does not matter, as long as clear_unmet knows it.
//
// Up to 16,384 tokens: one launch, no workgroup waits for another. Workgroup b looks through ALL
// tokens (sixteen per thread at most), keeps those whose row ends in the byte b, counts those that go
// in front of them, and sorts its own by the row's other bits in LDS. That is 256 times the reading, all of it
// from the L2, and still faster than sorting in one workgroup (23 us for 8,192 tokens as text has them) and than the radix
// sort below (50 us for 16,384). Uniform tokens take 5.6 us for 8,192 and 8.1 us for 16,384, tokens as text has them 7.7 and
// 10.9: looking through costs 2.5 us per 8,192 tokens (60 instructions per token and wavefront), the bucket of the most
// frequent token, which ends the launch, 2 to 3 us, and the launch and the latency of its steps the other 3 us.
// More: radix sort by digits of at most nine bits, two launches a pass (count 4 us, place 8 us: 131,072 tokens),
// which are little more than the latency of their steps.
//
// Ranking inside a workgroup: wavefront w holds 64 * R consecutive items, 64 at a time, and counts them
// per digit in LDS counters of its own; lanes with the same digit find each other with one ballot per bit
// of the digit, so ranks follow the items' order and no LDS atomic is needed.
constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kLanes;
constexpr uint32_t kMaxDigitBits = 9;
constexpr uint32_t kBucketBits = 8;
constexpr uint32_t kBuckets = 1u << kBucketBits;
constexpr uint32_t kBucketPosBits = 14;
constexpr uint32_t kBucketTokens = 1u << kBucketPosBits;       // tokens of a one-launch sort
constexpr uint64_t kBucketRows = 1ull << (32 - kBucketPosBits + kBucketBits);  // its rows: the other bits share 32 with the position
constexpr uint32_t kFewTokens = 128;                           // up to here a bucket is sorted by comparing all pairs
constexpr uint32_t kPairTokens = 512;                          // up to here what is left of it without its most frequent row is
// Radix sort: tiles of two tokens per thread keep more compute units busy (131,073 tokens 46 us a call against 69 with
// eight, 1,048,576 tokens 146 against 151), tiles of eight have fewer counts to add up (4,194,304: 451 against 463).
constexpr uint32_t kSmallTileTokens = 1u << 21;
constexpr uint32_t kDirectTiles = 128;  // up to here every tile adds up the others' counts itself (at the limit as fast as a scan between)

struct SortPass {
    Tokens tokens;
    const uint32_t* row_in;  // nullptr: the first pass, rows come from the tokens
    const uint32_t* pos_in;
    uint32_t* row_out;
    uint32_t* pos_out;
    uint32_t* count;         // [tiles + 1][1 << digit_bits]; the last row: all tiles together (scanned counts only)
    uint32_t shift, digit_bits, passes, tiles;
    int32_t scanned;         // count[t] holds the sum over the tiles before t
};

// The radix sort's items base + 64 r: rows (of tokens outside the table: `rows`) and positions.
template <int ITEMS>
__device__ __forceinline__ void load_items(uint32_t (&key)[ITEMS], const SortPass& a, uint32_t base)
{
    if (a.row_in) {
#pragma unroll
        for (int r = 0; r < ITEMS; ++r) key[r] = a.row_in[base + r * kLanes < a.tokens.n ? base + r * kLanes : a.tokens.n - 1];
    } else {
        load_rows<ITEMS>(key, a.tokens, base);
#pragma unroll
        for (int r = 0; r < ITEMS; ++r) key[r] = key[r] == kNoRow ? a.tokens.rows : key[r];
    }
}

// Lanes of the wavefront whose digit is this lane's; `active` lanes only.
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, bool active)
{
    const uint64_t among = __builtin_amdgcn_ballot_w64(active);
    uint32_t lo = static_cast<uint32_t>(among), hi = static_cast<uint32_t>(among >> 32);
#pragma unroll
    for (uint32_t b = 0; b < kMaxDigitBits; ++b) {
        const uint32_t bit = static_cast<uint32_t>(static_cast<int32_t>(digit << (31 - b)) >> 31);  // all ones or none
        const uint64_t v = __builtin_amdgcn_ballot_w64(bit != 0);
        lo &= ~(static_cast<uint32_t>(v) ^ bit);
        hi &= ~(static_cast<uint32_t>(v >> 32) ^ bit);
    }
    return static_cast<uint64_t>(hi) << 32 | lo;
}

// Sum over the lanes up to and with this one.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x)
{
    // lane permutes inside the vector unit: rows of 16 lanes shifted by 1, 2, 4, 8, then the rows' last lanes handed on
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
    return x;
}

// Sum over the threads before this one (1024 threads).
__device__ __forceinline__ uint32_t exclusive_scan(uint32_t x, uint32_t* wave_sums)
{
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t s = wave_scan(x);
    if (lane == 63) wave_sums[wave] = s;
    __syncthreads();
    uint32_t before = 0;
#pragma unroll
    for (uint32_t w = 0; w < kSortWaves; ++w) before += w < wave ? wave_sums[w] : 0;
    return before + s - x;
}

// Ranks items by digit: a wavefront's are its lanes' keys [0], then their keys [1] ..., `have` of them.
// counters[w][digit] ends as the number of wavefront w's items with that digit; rank[] as the number of them in
// front of each item.
template <int ITEMS>
__device__ __forceinline__ void rank_items(uint32_t (&rank)[ITEMS], const uint32_t (&key)[ITEMS], uint32_t have, uint32_t shift, uint32_t bits,
                                           uint32_t* counters)
{
    const uint32_t lane = threadIdx.x & 63u, bins = 1u << bits;
    uint32_t* share = counters + (threadIdx.x >> 6) * bins;
    for (uint32_t b = lane * 4; b < bins; b += kLanes * 4) *reinterpret_cast<u32x4*>(share + b) = u32x4{0, 0, 0, 0};
    volatile uint32_t* mine = share;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        if (r * kLanes < have) {  // wave-uniform
            const bool active = r * kLanes + lane < have;
            const uint32_t digit = key[r] >> shift & (bins - 1);
            const uint64_t same = same_digit(digit, active);
            const uint32_t in_front = __builtin_popcountll(same & ((1ull << lane) - 1));
            const uint32_t before = active ? mine[digit] : 0;
            rank[r] = before + in_front;
            __builtin_amdgcn_wave_barrier();
            if (active && in_front == 0) mine[digit] = before + __builtin_popcountll(same);
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// Turns the counters of rank_items into where each wavefront's items with a digit begin.
__device__ __forceinline__ void scan_counters(uint32_t* counters, uint32_t bins, uint32_t* wave_sums)
{
    const uint32_t each = bins * kSortWaves / kSortThreads;  // counters per thread, 1 ... 8, in the order (digit, wavefront)
    uint32_t local[8], sum = 0;
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k) {
        const uint32_t e = threadIdx.x * each + k;
        local[k] = k < each ? counters[(e % kSortWaves) * bins + e / kSortWaves] : 0;
        sum += local[k];
    }
    uint32_t at = exclusive_scan(sum, wave_sums);
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k) {
        const uint32_t e = threadIdx.x * each + k;
        if (k < each) counters[(e % kSortWaves) * bins + e / kSortWaves] = at;
        at += local[k];
    }
}

// ITEMS: tokens per thread, at least n / 1024.
template <int ITEMS>
__global__ __launch_bounds__(kSortThreads) void sort_buckets_kernel(SortPass a)
{
    extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
    __shared__ uint32_t kept[kSortWaves], in_front[kSortWaves], often_of[kSortWaves], below_of[kSortWaves], wave_sums[kSortWaves];
    __shared__ __attribute__((aligned(16))) uint32_t pairs[kPairTokens + 4];
    const uint32_t n = a.tokens.n, rows = a.tokens.rows, me = blockIdx.x;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr uint32_t per_wave = ITEMS * kLanes;
    uint32_t* list = lds;  // the bucket's tokens (the row's other bits, then the position), each wavefront's from its own begin
    uint32_t* counters = lds + ITEMS * kSortThreads;

    uint32_t key[ITEMS];
    load_rows<ITEMS>(key, a.tokens, wave * per_wave + lane);
    // Rotated, a row's bucket is its upper byte and what the bucket is sorted by the rest; kNoRow stays behind all rows.
    const uint32_t first_of_bucket = me << (32 - kBucketBits);
    uint32_t own = 0, before = 0;
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const uint32_t rotated = key[r] >> kBucketBits | key[r] << (32 - kBucketBits), rest = rotated - first_of_bucket;
        const bool is_mine = rest < (1u << (32 - kBucketPosBits));
        const uint64_t mine = __builtin_amdgcn_ballot_w64(is_mine);
        before += __builtin_popcountll(__builtin_amdgcn_ballot_w64(rotated < first_of_bucket));
        if (is_mine)
            list[wave * per_wave + own + __builtin_popcountll(mine & ((1ull << lane) - 1))] = rest << kBucketPosBits | (wave * per_wave + r * kLanes + lane);
        own += __builtin_popcountll(mine);
    }
    if (lane == 0) {
        kept[wave] = own;
        in_front[wave] = before;
    }
    __syncthreads();
    uint32_t size = 0, begin = 0;  // of the bucket
    uint32_t shares[kSortWaves];   // wavefronts' tokens
#pragma unroll
    for (uint32_t w = 0; w < kSortWaves; ++w) {
        shares[w] = __builtin_amdgcn_readfirstlane(kept[w]);
        size += shares[w];
        begin += __builtin_amdgcn_readfirstlane(in_front[w]);
    }
    if (me == kBuckets - 1)  // tokens outside the table, behind all others
        for (uint32_t i = begin + size + threadIdx.x; i < n; i += kSortThreads) {
            a.row_out[i] = rows;
            a.pos_out[i] = 0;
        }
    if (size == 0) return;
    auto in_order = [&](uint32_t i) {  // the bucket's token i, below size
        uint32_t skipped = 0, at = i;
#pragma unroll
        for (uint32_t w = 0; w < kSortWaves; ++w) {
            at = i >= skipped ? w * per_wave + i - skipped : at;
            skipped += shares[w];
        }
        return list[at];
    };
    auto write = [&](uint32_t to, uint32_t packed) {
        a.row_out[begin + to] = packed >> kBucketPosBits << kBucketBits | me;
        a.pos_out[begin + to] = packed & (kBucketTokens - 1);
    };
    // The rank of packed value x among `m` in pairs[]: they are all different, it is the number of smaller ones.
    auto rank_among = [&](uint32_t x, uint32_t m) {
        uint32_t rank = 0;
#pragma unroll 4
        for (uint32_t j = 0; j < m; j += 4) {
            const u32x4 y = *reinterpret_cast<const u32x4*>(pairs + j);
            rank += (y.x < x) + (y.y < x) + (y.z < x) + (y.w < x);
        }
        return rank;
    };
    if (size <= kFewTokens) {
        if (threadIdx.x < size + 4) pairs[threadIdx.x] = threadIdx.x < size ? in_order(threadIdx.x) : 0xffffffffu;
        __syncthreads();
        if (threadIdx.x >= size) return;
        const uint32_t x = pairs[threadIdx.x];
        write(rank_among(x, size), x);
        return;
    }
    uint32_t have = __builtin_amdgcn_readfirstlane(kept[wave]), from = wave * per_wave;  // this wavefront's items and their place in the list
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) key[r] = r * kLanes + lane < have ? list[from + r * kLanes + lane] : 0;

    // A large bucket mostly holds one frequent token and few others. The frequent one's tokens are in order
    // already; the others, if few enough, are ranked in pairs. Which row is taken for the frequent one only
    // decides about speed: the most common one of eight samples among 64.
    {
        const uint32_t sample = in_order(static_cast<uint32_t>(static_cast<uint64_t>(lane) * size / kLanes)) >> kBucketPosBits;
        uint32_t often = 0, most = 0;
#pragma unroll
        for (uint32_t l = 0; l < kLanes; l += 8) {
            const uint32_t row = __builtin_amdgcn_readlane(sample, l);
            const uint32_t alike = __builtin_popcountll(__builtin_amdgcn_ballot_w64(sample == row));
            often = alike > most ? row : often;
            most = alike > most ? alike : most;
        }
        uint32_t own_often = 0, own_below = 0;
#pragma unroll
        for (int r = 0; r < ITEMS; ++r) {
            if (r * kLanes < have) {
                const bool valid = r * kLanes + lane < have;
                const uint32_t row = key[r] >> kBucketPosBits;
                own_often += __builtin_popcountll(__builtin_amdgcn_ballot_w64(valid && row == often));
                own_below += __builtin_popcountll(__builtin_amdgcn_ballot_w64(valid && row < often));
            }
        }
        if (lane == 0) {
            often_of[wave] = own_often;
            below_of[wave] = own_below;
        }
        __syncthreads();
        uint32_t often_all = 0, often_before = 0, before_all = 0, below = 0;
#pragma unroll
        for (uint32_t w = 0; w < kSortWaves; ++w) {
            often_before += w < wave ? often_of[w] : 0;
            before_all += w < wave ? shares[w] : 0;
            often_all += often_of[w];
            below += below_of[w];
        }
        const uint32_t others = __builtin_amdgcn_readfirstlane(size - often_all);
        if (others <= kPairTokens) {
            uint32_t others_before = before_all - often_before;
#pragma unroll
            for (int r = 0; r < ITEMS; ++r) {
                if (r * kLanes < have) {
                    const bool valid = r * kLanes + lane < have, is_often = valid && key[r] >> kBucketPosBits == often, is_other = valid && !is_often;
                    const uint64_t m_often = __builtin_amdgcn_ballot_w64(is_often), m_other = __builtin_amdgcn_ballot_w64(is_other);
                    const uint64_t front = (1ull << lane) - 1;
                    if (is_often) write(below + often_before + __builtin_popcountll(m_often & front), key[r]);
                    if (is_other) pairs[others_before + __builtin_popcountll(m_other & front)] = key[r];
                    often_before += __builtin_popcountll(m_often);
                    others_before += __builtin_popcountll(m_other);
                }
            }
            if (threadIdx.x < 4) pairs[others + threadIdx.x] = 0xffffffffu;
            __syncthreads();
            if (threadIdx.x >= others) return;
            const uint32_t x = pairs[threadIdx.x];
            write(rank_among(x, others) + (x >> kBucketPosBits > often ? often_all : 0), x);
            return;
        }
    }
    const uint32_t per_wave_later = (size + kSortThreads - 1) / kSortThreads * kLanes, bins = 1u << a.digit_bits;
    uint32_t rank[ITEMS];
    for (uint32_t pass = 0; pass < a.passes; ++pass) {
        const uint32_t shift = kBucketPosBits + pass * a.digit_bits;
        rank_items<ITEMS>(rank, key, have, shift, a.digit_bits, counters);
        __syncthreads();
        scan_counters(counters, bins, wave_sums);
        __syncthreads();
        const bool last = pass + 1 == a.passes;
#pragma unroll
        for (int r = 0; r < ITEMS; ++r) {
            if (r * kLanes + lane < have) {
                const uint32_t to = counters[wave * bins + (key[r] >> shift & (bins - 1))] + rank[r];
                if (last)
                    write(to, key[r]);
                else
                    list[to] = key[r];
            }
        }
        if (last) return;
        __syncthreads();
        from = wave * per_wave_later;
        have = from >= size ? 0 : size - from < per_wave_later ? size - from : per_wave_later;
#pragma unroll
        for (int r = 0; r < ITEMS; ++r) key[r] = r * kLanes + lane < have ? list[from + r * kLanes + lane] : 0;
        __syncthreads();
    }
}

// Radix sort, first launch of a pass: how often each digit occurs in each tile.
template <int ITEMS>
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(SortPass a)
{
    __shared__ uint32_t counters[1u << kMaxDigitBits];
    const uint32_t bins = 1u << a.digit_bits;
    const uint32_t base = (blockIdx.x * kSortWaves + (threadIdx.x >> 6)) * kLanes * ITEMS + (threadIdx.x & 63u);
    uint32_t key[ITEMS];
    load_items<ITEMS>(key, a, base);
    if (threadIdx.x < bins) counters[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r)
        if (base + r * kLanes < a.tokens.n) __hip_atomic_fetch_add(&counters[key[r] >> a.shift & (bins - 1)], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    __syncthreads();
    if (threadIdx.x < bins) a.count[static_cast<uint64_t>(blockIdx.x) * bins + threadIdx.x] = counters[threadIdx.x];
}

// Many tiles: turns their counts into sums over the tiles before. A workgroup has 64 digits, a
// wavefront of it one sixteenth of the tiles.
__global__ __launch_bounds__(kSortThreads) void sort_scan_kernel(SortPass a)
{
    __shared__ uint32_t part[kSortWaves][kLanes];
    const uint32_t bins = 1u << a.digit_bits, lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t* count = a.count + blockIdx.x * kLanes + lane;
    const uint32_t lo = static_cast<uint64_t>(a.tiles) * wave / kSortWaves, hi = static_cast<uint64_t>(a.tiles) * (wave + 1) / kSortWaves;
    uint32_t sum = 0;
#pragma unroll 8
    for (uint32_t t = lo; t < hi; ++t) sum += count[static_cast<uint64_t>(t) * bins];
    part[wave][lane] = sum;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (uint32_t w = 0; w < kSortWaves; ++w) {
        before += w < wave ? part[w][lane] : 0;
        all += part[w][lane];
    }
#pragma unroll 8
    for (uint32_t t = lo; t < hi; ++t) {
        const uint32_t c = count[static_cast<uint64_t>(t) * bins];
        count[static_cast<uint64_t>(t) * bins] = before;
        before += c;
    }
    if (wave == 0) count[static_cast<uint64_t>(a.tiles) * bins] = all;
}

// Last launch of a pass: every tile moves its tokens to where their digits begin.
template <int ITEMS>
__global__ __launch_bounds__(kSortThreads) void sort_place_kernel(SortPass a)
{
    extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
    __shared__ uint32_t wave_sums[kSortWaves];
    const uint32_t bins = 1u << a.digit_bits, n = a.tokens.n;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t base = (blockIdx.x * kSortWaves + wave) * kLanes * ITEMS;
    uint32_t key[ITEMS], pos[ITEMS], rank[ITEMS];
    load_items<ITEMS>(key, a, base + lane);
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const uint32_t i = base + r * kLanes + lane;
        pos[r] = a.row_in && i < n ? a.pos_in[i] : i;
    }
    // this digit in the tiles before this one, and in all tiles: two threads per digit add half of the tiles each
    __shared__ uint32_t halves[2][1u << kMaxDigitBits];
    uint32_t before = 0, all = 0;
    if (a.scanned) {
        if (threadIdx.x < bins) {
            before = a.count[static_cast<uint64_t>(blockIdx.x) * bins + threadIdx.x];
            all = a.count[static_cast<uint64_t>(a.tiles) * bins + threadIdx.x];
        }
    } else if (threadIdx.x < 2 * bins) {
        const uint32_t half = threadIdx.x >= bins, digit = threadIdx.x - half * bins;
#pragma unroll 16
        for (uint32_t t = half; t < a.tiles; t += 2) {
            const uint32_t c = a.count[t * bins + digit];
            before += t < blockIdx.x ? c : 0;
            all += c;
        }
        if (half) {
            halves[0][digit] = before;
            halves[1][digit] = all;
        }
    }
    const uint32_t have = base >= n ? 0 : n - base < ITEMS * kLanes ? n - base : ITEMS * kLanes;
    rank_items<ITEMS>(rank, key, have, a.shift, a.digit_bits, lds);
    __syncthreads();
    if (threadIdx.x < bins && !a.scanned) {
        before += halves[0][threadIdx.x];
        all += halves[1][threadIdx.x];
    }
    uint32_t at = exclusive_scan(threadIdx.x < bins ? all : 0, wave_sums) + before;
    if (threadIdx.x < bins) {
        uint32_t c[kSortWaves];
#pragma unroll
        for (uint32_t w = 0; w < kSortWaves; ++w) c[w] = lds[w * bins + threadIdx.x];
#pragma unroll
        for (uint32_t w = 0; w < kSortWaves; ++w) {
            lds[w * bins + threadIdx.x] = at;
            at += c[w];
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        if (base + r * kLanes + lane >= n) continue;
        const uint32_t to = lds[wave * bins + (key[r] >> a.shift & (bins - 1))] + rank[r];
        a.row_out[to] = key[r];
        a.pos_out[to] = pos[r];
    }
}

// ---- rows without a token ----------------------------------------------------------------------
// A gradient that is written, not added: the other rows become zero. A workgroup takes kClearRows rows at a time.
// 64 rows at a time left the last workgroups alone for longer: 82 us against 77, sums included, for 32,000 rows of 4096
// bf16 elements.
constexpr uint32_t kClearRows = 16;
constexpr uint32_t kMostClearing = 1u << 20;  // workgroups of a launch that clear

// Clears the rows first + b of the bits b in `clear`, which are inside the table.
template <int AT>
__device__ __forceinline__ void clear_rows(const GradPass& a, uint64_t first, uint64_t clear)
{
    constexpr int U = AT == FT_F32 ? 4 : 8;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const float zero[U] = {};
    for (uint32_t k = 0; clear; ++k, clear &= clear - 1) {
        if (k % waves != wave) continue;
        const uint64_t at = (first + __builtin_ctzll(clear)) * a.acc_stride;
        for (uint32_t col = lane * U; col < a.cols; col += kLanes * U) {
            if (a.cols - col >= U)
                row_store<AT, U, true>(a.acc, at + col, zero);
            else
                row_store_some<AT, U>(a.acc, at + col, zero, a.cols - col);
        }
    }
}

// The workgroup `me` of `of`; a lane looks a row up in the sorted tokens.
template <int AT>
__device__ __forceinline__ void clear_unmet(const GradPass& a, uint32_t me, uint32_t of)
{
    const uint32_t lane = threadIdx.x & 63u, n = a.tokens.n;
    for (uint64_t first = static_cast<uint64_t>(me) * kClearRows; first < a.tokens.rows; first += static_cast<uint64_t>(of) * kClearRows) {
        const uint64_t row = first + lane;
        const bool mine = lane < kClearRows && row < a.tokens.rows;
        auto order = [&](uint32_t r) { return r >= a.tokens.rows ? kNoRow : (r >> a.rotate) | (a.rotate ? r << (32 - a.rotate) : 0); };
        const uint32_t want = order(mine ? static_cast<uint32_t>(row) : kNoRow);
        uint32_t lo = 0, hi = mine ? n : 0;  // the first sorted token of a row not in front of this one
        while (lo < hi) {
            const uint32_t mid = (lo + hi) >> 1;
            if (order(a.row_s[mid]) < want)
                lo = mid + 1;
            else
                hi = mid;
        }
        const bool met = mine && lo < n && a.row_s[lo] == row;
        clear_rows<AT>(a, first, __builtin_amdgcn_ballot_w64(mine && !met));
    }
}

// ---- calls without sorting ----------------------------------------------------------------------
// Few tokens: one launch. A workgroup has a token and eight blocks of columns (a unit per lane each); its threads look
// through all tokens and list those of the workgroup's row in order. The workgroups of one row's tokens all have the
// same list then, and share the row's blocks of columns without a word to each other: of a row with one token every
// wavefront has a block, of a row with more than eight every workgroup has, with the list dealt to its wavefronts eight
// tokens at a time and their sums joined in LDS in the wavefronts' order.
//
// What bounds it is the latency of its steps: 512 different tokens x 4096 bf16 into fp32 5.2 us and a call every 6.9
// (the host's side of it), where the three launches of the sorted way take 8.9 and 13.7; 512 as text has them 5.8
// (10.5), one row that has all 512 12.3 (11.4), for which two wavefronts' loads in flight are not enough (sixteen
// tokens at a time took longer for text: 6.9). With two tokens per thread 1,024 tokens x 4096 take 10.3 us (sorted
// 11.3; text 9.8 against 12.0, one row 18 against 15), x 512 4.6 (8.3), but x 8192, two workgroups per token, 22.4
// (20.6).
constexpr int kUnsortedThreads = 512;
constexpr int kUnsortedWaves = kUnsortedThreads / kLanes;
constexpr uint32_t kUnsortedBlocks = kUnsortedWaves;
constexpr uint32_t kUnsortedAhead = 8;  // gradient rows in flight

// Tokens per thread of a call that is not sorted; 0: sorted.
uint32_t unsorted_items(uint64_t n, uint64_t cols, uint32_t unit)
{
    if (n <= kUnsortedThreads) return 1;
    return n <= 2 * kUnsortedThreads && cols <= kUnsortedBlocks * kLanes * unit ? 2 : 0;
}

template <int GT, int AT, bool DROP, bool RAGGED, int ITEMS>
__global__ __launch_bounds__(kUnsortedThreads) void embedding_grad_unsorted_kernel(GradPass a, uint32_t sums)
{
    constexpr int U = row_unit<GT, AT>();
    __shared__ uint32_t list[ITEMS * kUnsortedThreads];
    __shared__ uint32_t found[kUnsortedWaves];
    __shared__ float parts[kUnsortedWaves][U][kLanes];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t n = a.tokens.n, at = wave * ITEMS * kLanes + lane;
    uint32_t row[ITEMS];
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) row[r] = at + r * kLanes < n ? a.tokens.row(at + r * kLanes) : kNoRow;
    if (blockIdx.x >= sums) {  // a gradient that is written, not added
        const uint64_t step = static_cast<uint64_t>(gridDim.x - sums) * kClearRows;
        for (uint64_t first = static_cast<uint64_t>(blockIdx.x - sums) * kClearRows; first < a.tokens.rows; first += step) {
            uint32_t met = 0;
#pragma unroll
            for (int r = 0; r < ITEMS; ++r)
                if (row[r] != kNoRow && row[r] - first < kClearRows) met |= 1u << (row[r] - first);
#pragma unroll
            for (int d = 1; d < kLanes; d <<= 1) met |= __shfl_xor(met, d);
            if (lane == 0) found[wave] = met;
            __syncthreads();
            met = 0;
#pragma unroll
            for (int w = 0; w < kUnsortedWaves; ++w) met |= found[w];
            __syncthreads();
            const uint64_t left = a.tokens.rows - first;
            const uint32_t there = left < kClearRows ? (1u << left) - 1 : (1u << kClearRows) - 1;
            clear_rows<AT>(a, first, __builtin_amdgcn_readfirstlane(there & ~met));
        }
        return;
    }
    const uint32_t part = blockIdx.x / n, me = blockIdx.x - part * n;
    const uint32_t mine = a.tokens.row(me);
    if (mine == kNoRow) return;
    uint32_t own = 0;
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) own += __builtin_popcountll(__builtin_amdgcn_ballot_w64(row[r] == mine));
    if (lane == 0) found[wave] = own;
    __syncthreads();
    uint32_t to = 0, total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kUnsortedWaves; ++w) {
        const uint32_t f = __builtin_amdgcn_readfirstlane(found[w]);
        to += w < wave ? f : 0;
        total += f;
    }
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const uint64_t match = __builtin_amdgcn_ballot_w64(row[r] == mine);
        if (row[r] == mine) list[to + __builtin_popcountll(match & ((1ull << lane) - 1))] = at + r * kLanes;
        to += __builtin_popcountll(match);
    }
    __syncthreads();
    const uint32_t blocks = (a.cols + kLanes * U - 1) / (kLanes * U) - part * kUnsortedBlocks;
    const uint32_t shared = blocks < kUnsortedBlocks ? blocks : kUnsortedBlocks, sharers = total < shared ? total : shared;
    const uint64_t chosen = __builtin_amdgcn_ballot_w64(lane < sharers && list[lane] == me);
    if (!chosen) return;
    const uint32_t rank = __builtin_ctzll(chosen);  // of this token among its row's
    // Eight tokens or fewer: a wavefront has a block. More: the workgroup has one (as many sharers as blocks), the
    // wavefronts have their tokens of it.
    const bool many = total > kUnsortedAhead;
    const uint32_t block = many ? rank : rank + wave * sharers;
    const uint32_t col = ((part * kUnsortedBlocks + block) * kLanes + lane) * U;
    const uint32_t count = block >= shared || col >= a.cols ? 0 : a.cols - col < U ? a.cols - col : U;
    float sum[U] = {};
    RowBits<AT, U> old{};
    if (count) {
        if (!many || wave == 0) old = load_old<AT, U, RAGGED>(a, mine, col, count);
        uint64_t key = 0;
        if constexpr (DROP) key = ftc::dropout_key(a.drop);
        auto add = [&](auto ahead, uint32_t from) {
            constexpr uint32_t AHEAD = decltype(ahead)::value;
            uint32_t pos[AHEAD];
            RowBits<GT, U> bits[AHEAD];
#pragma unroll
            for (uint32_t j = 0; j < AHEAD; ++j) {  // behind the last token: the last one again
                pos[j] = __builtin_amdgcn_readfirstlane(list[from + j < total ? from + j : total - 1]);
                if (!RAGGED || from + j < total) bits[j] = load_unit<GT, U, true, RAGGED>(a.g, static_cast<uint64_t>(pos[j]) * a.g_stride + col, count);
            }
#pragma unroll
            for (uint32_t j = 0; j < AHEAD; ++j)
                if (from + j < total) add_unit<GT, U, DROP>(sum, bits[j], a, key, pos[j], col);
        };
        if (total == 1)
            add(std::integral_constant<uint32_t, 1>{}, 0);
        else
            for (uint32_t from = many ? wave * kUnsortedAhead : 0; from < total; from += kUnsortedWaves * kUnsortedAhead)
                add(std::integral_constant<uint32_t, kUnsortedAhead>{}, from);
    }
    if (many) {
        if (wave) {
#pragma unroll
            for (int j = 0; j < U; ++j) parts[wave][j][lane] = sum[j];
        }
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int w = 1; w < kUnsortedWaves; ++w) {
#pragma unroll
            for (int j = 0; j < U; ++j) sum[j] += parts[w][j][lane];
        }
    }
    if (count) finish_unit<AT, U, RAGGED>(a, mine, col, count, sum, old);
}

// ---- summing runs of equal rows -------------------------------------------------------------------
// Workgroup (block of 64 units of columns, group): eight wavefronts with per_wave consecutive sorted
// tokens each, one unit of columns per lane. A run inside a wavefront goes straight to the accumulator; one
// that crosses into the next wavefront is joined in LDS by the wavefront it begins in; one that crosses
// workgroups leaves its parts in memory (tail: where it begins, head: in the others) for
// embedding_grad_join_kernel. (Having the workgroup that delivers a run's last part add them up took longer than the
// second launch: 38 us against 30 + 4 for 8,192 tokens x 4096.)
//
// HBM-bound: 8,192 tokens x 4096 bf16 into fp32 (159 MB) 30 us, 131,072 x 2048 into bf16 with 60 % one token (676 MB)
// 127 us = 5.3 TB/s; one row that has all tokens runs at 6.2 TB/s, rows that are read and written back one by one at 5.2.
// At most sixteen tokens per wavefront: a run that stays in registers costs a third of as many single rows, and
// with 64 tokens each the wavefronts of the single rows were left alone at the end (151 us). Eight wavefronts per
// workgroup halve the parts of cut runs against four (join 10 instead of 20 us) at the same speed; sixteen wait for
// each other (139 us).
constexpr int kSumWaves = 8;

// Gradient rows in flight per wavefront; the accumulator rows of the runs that end among them are
// fetched with them, so that a wavefront waits once for all of them and not once per run. (Two, four, eight: 131,
// 126, 126 us, 30.5, 30.2, 31.6 us for the smaller call.)
constexpr int kAhead = 4;

template <int GT, int AT, bool DROP, bool RAGGED>
__global__ __launch_bounds__(kSumWaves * kLanes) void embedding_grad_sum_kernel(GradPass a)
{
    constexpr int U = row_unit<GT, AT>();
    __shared__ float parts[kSumWaves][2][U][kLanes];               // 0: head, 1: tail
    __shared__ uint32_t head_row[kSumWaves], tail_row[kSumWaves];  // kNoRow: none
    __shared__ uint32_t through[kSumWaves];                        // the head goes on behind the wavefront's end
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t n = a.tokens.n, rows = a.tokens.rows;
    const uint32_t blocks = a.padded / (kLanes * U);
    // A gradient that is written, not added: workgroups behind those of the sums clear rows. (In front of them the
    // launch took 101 us instead of 82, spread among them 89, as a launch of their own 100: 16,384 tokens, 32,000 rows
    // of 4096 bf16 elements.)
    if (blockIdx.x >= a.groups * blocks) {
        clear_unmet<AT>(a, blockIdx.x - a.groups * blocks, gridDim.x - a.groups * blocks);
        return;
    }
    const uint32_t group = blockIdx.x / blocks, block = blockIdx.x - group * blocks;
    const uint32_t col = (block * kLanes + lane) * U;
    const uint32_t count = col >= a.cols ? 0 : (a.cols - col < U ? a.cols - col : U);
    const uint32_t from = count ? col : 0;  // lanes behind the row's end read its beginning and store nothing
    const uint64_t base = (static_cast<uint64_t>(group) * kSumWaves + wave) * a.per_wave;
    uint64_t key = 0;
    if constexpr (DROP) key = ftc::dropout_key(a.drop);

    const uint64_t i = base + lane;
    const bool inside = lane < a.per_wave && i < n;
    const uint32_t my_row = inside ? a.row_s[i] : rows;
    const uint32_t my_pos = inside ? a.pos_s[i] : 0;
    const uint32_t prev = base > 0 && base - 1 < n ? a.row_s[base - 1] : kNoRow;
    const uint32_t next = base + a.per_wave < n ? a.row_s[base + a.per_wave] : kNoRow;
    const uint32_t valid = __builtin_popcountll(__builtin_amdgcn_ballot_w64(my_row < rows));  // tokens outside the table are last

    uint32_t h_row = kNoRow, t_row = kNoRow, thru = 0;
    if (valid) {
        const uint32_t first_row = __builtin_amdgcn_readlane(my_row, 0);
        const bool came_in = first_row == prev;  // the first run began before this wavefront
        float sum[U] = {};
        auto keep_part = [&](int slot) {
#pragma unroll
            for (int j = 0; j < U; ++j) parts[wave][slot][j][lane] = sum[j];
        };
        for (uint32_t j0 = 0; j0 < valid; j0 += kAhead) {
            RowBits<GT, U> bits[kAhead];
            RowBits<AT, U> old[kAhead];
            uint32_t pos[kAhead], r[kAhead + 1];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const uint32_t at = j0 + j < valid ? j0 + j : valid - 1;
                pos[j] = __builtin_amdgcn_readlane(my_pos, at);
                r[j] = __builtin_amdgcn_readlane(my_row, at);
                bits[j] = load_unit<GT, U, true, RAGGED>(a.g, static_cast<uint64_t>(pos[j]) * a.g_stride + from, count);
            }
            r[kAhead] = j0 + kAhead < valid ? __builtin_amdgcn_readlane(my_row, j0 + kAhead) : next;
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const uint32_t behind = j0 + j + 1 < valid ? r[j + 1] : next;
                if (j0 + j < valid && behind != r[j] && !(came_in && r[j] == first_row)) old[j] = load_old<AT, U, RAGGED>(a, r[j], from, count);
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (j0 + j >= valid) break;
                add_unit<GT, U, DROP>(sum, bits[j], a, key, pos[j], from);
                const uint32_t behind = j0 + j + 1 < valid ? r[j + 1] : next;
                if (behind == r[j]) continue;
                if (came_in && r[j] == first_row) {
                    keep_part(0);
                    h_row = first_row;
                } else if (count) {
                    finish_unit<AT, U, RAGGED>(a, r[j], col, count, sum, old[j]);
                }
#pragma unroll
                for (int e = 0; e < U; ++e) sum[e] = 0.0f;
            }
        }
        const uint32_t last = __builtin_amdgcn_readlane(my_row, valid - 1);
        if (last == next) {  // goes on behind this wavefront
            if (came_in && last == first_row) {
                keep_part(0);
                h_row = last;
                thru = 1;
            } else {
                keep_part(1);
                t_row = last;
            }
        }
    }
    if (lane == 0) {
        head_row[wave] = h_row;
        tail_row[wave] = t_row;
        through[wave] = thru;
    }
    __syncthreads();
    // The wavefront a run begins in joins it; the one that came in from the workgroup before, wavefront 0.
    auto join = [&](uint32_t r, uint32_t w, int slot, bool goes_on, bool from_before) {
        float sum[U];
#pragma unroll
        for (int j = 0; j < U; ++j) sum[j] = parts[w][slot][j][lane];
        while (goes_on && ++w < kSumWaves) {
#pragma unroll
            for (int j = 0; j < U; ++j) sum[j] += parts[w][0][j][lane];
            goes_on = through[w];
        }
        if (from_before || goes_on)
            row_store<FT_F32, U, false>(from_before ? a.head : a.tail, static_cast<uint64_t>(group) * a.padded + col, sum);
        else if (count)
            finish_unit<AT, U, RAGGED>(a, r, col, count, sum, load_old<AT, U, RAGGED>(a, r, col, count));
    };
    if (wave == 0 && head_row[0] != kNoRow) join(head_row[0], 0, 0, through[0], true);
    if (tail_row[wave] != kNoRow) join(tail_row[wave], wave, 1, true, false);
}

// Runs that cross workgroups of the sums. Up to kLightParts parts: the wavefront of the workgroup that the
// run begins in adds them up. More (a token that fills the batch, padding): such a run covers a group whose
// number is a multiple of kLightParts; the first of these has a workgroup per 128 columns, sixteen wavefronts
// with their share of the parts each. 1,200 parts of one run took 45 us with four wavefronts.
constexpr uint32_t kLightParts = 32;
constexpr int kJoinWaves = 16;
constexpr int kHeavyUnit = 2;
constexpr uint32_t kHeavyCols = kLanes * kHeavyUnit;

template <int U, int AHEAD>
__device__ __forceinline__ void add_parts(float (&sum)[U], const GradPass& a, uint32_t from, uint32_t lo, uint32_t hi, uint32_t col)
{
    for (uint32_t k0 = lo; k0 < hi; k0 += AHEAD) {
        RowBits<FT_F32, U> bits[AHEAD];
#pragma unroll
        for (uint32_t k = 0; k < AHEAD; ++k)
            if (k0 + k < hi) bits[k] = row_load<FT_F32, U, false>(k0 + k == 0 ? a.tail : a.head, static_cast<uint64_t>(from + k0 + k) * a.padded + col);
#pragma unroll
        for (uint32_t k = 0; k < AHEAD; ++k)
            if (k0 + k < hi) {
#pragma unroll
                for (int j = 0; j < U; ++j) sum[j] += bits[k][j];
            }
    }
}

template <int AT, int U>
__device__ __forceinline__ void join_light(const GradPass& a, uint32_t group, uint32_t block)
{
    const uint32_t lane = threadIdx.x & 63u, rows = a.tokens.rows;
    const uint64_t n = a.tokens.n, per_group = static_cast<uint64_t>(a.per_wave) * kSumWaves, begin = group * per_group, end = begin + per_group;
    if (end >= n) return;
    const uint32_t row = a.row_s[end];
    if (row >= rows || a.row_s[end - 1] != row) return;
    if (a.row_s[begin] == row && begin > 0 && a.row_s[begin - 1] == row) return;  // began earlier
    const uint64_t at = end + lane * per_group;  // the group in which part 1 + lane lies
    const uint64_t in = __builtin_amdgcn_ballot_w64(at < n && a.row_s[at < n ? at : 0] == row);
    const uint32_t all = 1 + (~in ? __builtin_ctzll(~in) : kLanes);
    const uint32_t col = (block * kLanes + lane) * U;
    if (all > kLightParts || col >= a.cols) return;
    const uint32_t count = a.cols - col < U ? a.cols - col : U;
    const RowBits<AT, U> old = load_old<AT, U, true>(a, row, col, count);
    float sum[U] = {};
    add_parts<U, 4>(sum, a, group, 0, all, col);
    finish_unit<AT, U, true>(a, row, col, count, sum, old);
}

// How many of lo + 1 ... hi satisfy `in`, which holds up to some index and for none behind it; 64 at a time.
template <typename F>
__device__ __forceinline__ uint32_t count_while(uint32_t lo, uint32_t hi, F in)
{
    const uint32_t lane = threadIdx.x & 63u, from = lo;
    while (lo < hi) {
        const uint32_t step = (hi - lo + kLanes - 1) / kLanes;
        const uint64_t at = lo + static_cast<uint64_t>(lane + 1) * step;
        lo += __builtin_popcountll(__builtin_amdgcn_ballot_w64(at <= hi && in(static_cast<uint32_t>(at)))) * step;
        hi = lo + step - 1 < hi ? lo + step - 1 : hi;
    }
    return lo - from;
}

template <int AT>
__device__ __forceinline__ void join_heavy(const GradPass& a, uint32_t group, uint32_t block)
{
    constexpr int U = kHeavyUnit;
    __shared__ float parts[kJoinWaves][U][kLanes];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t per_group = static_cast<uint64_t>(a.per_wave) * kSumWaves, at = group * per_group;
    const uint32_t row = a.row_s[at];
    if (row >= a.tokens.rows || a.row_s[at - 1] != row) return;
    // groups in front of which the run is there already, this one's predecessors first
    const uint32_t earlier = count_while(0, kLightParts, [&](uint32_t k) { return group > k && a.row_s[(group - k) * per_group - 1] == row; });
    if (earlier >= kLightParts) return;  // another multiple of kLightParts has it
    const uint32_t from = group - 1 - earlier;
    const uint32_t all = 2 + earlier + count_while(0, a.groups - 1 - group, [&](uint32_t k) { return a.row_s[(group + k) * per_group] == row; });
    if (all <= kLightParts) return;
    const uint32_t col = (block * kLanes + lane) * U;  // below padded, which is a multiple of kHeavyCols
    const uint32_t lo = static_cast<uint64_t>(all) * wave / kJoinWaves, hi = static_cast<uint64_t>(all) * (wave + 1) / kJoinWaves;
    float sum[U] = {};
    add_parts<U, 16>(sum, a, from, lo, hi, col);
#pragma unroll
    for (int j = 0; j < U; ++j) parts[wave][j][lane] = sum[j];
    __syncthreads();
    if (wave != 0 || col >= a.cols) return;
    const uint32_t count = a.cols - col < U ? a.cols - col : U;
    const RowBits<AT, U> old = load_old<AT, U, true>(a, row, col, count);
#pragma unroll
    for (int w = 1; w < kJoinWaves; ++w)
#pragma unroll
        for (int j = 0; j < U; ++j) sum[j] += parts[w][j][lane];
    finish_unit<AT, U, true>(a, row, col, count, sum, old);
}

template <int AT, int U>
__global__ __launch_bounds__(kJoinWaves * kLanes) void embedding_grad_join_kernel(GradPass a, uint32_t light)
{
    if (blockIdx.x < light) {
        const uint32_t blocks = a.padded / (kLanes * U), item = blockIdx.x * kJoinWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        if (item < a.groups * blocks) join_light<AT, U>(a, item / blocks, item % blocks);
    } else {
        const uint32_t blocks = a.padded / kHeavyCols, item = blockIdx.x - light;
        join_heavy<AT>(a, (item / blocks + 1) * kLightParts, item % blocks);
    }
}

// ---- host ---------------------------------------------------------------------------------------
struct GradPlan {
    uint32_t unsorted;                                  // tokens per thread without sorting, 0: sorted
    uint32_t digit_bits, passes, tiles, items, rotate;  // tiles 0: sorted in one launch
    uint32_t per_wave, groups, padded;
    size_t off_pos_a, off_row_b, off_pos_b, off_count, off_head, off_tail, bytes;  // row_a at 0
};

// unit: elements per lane for the call's types (row_unit).
GradPlan plan_grad(uint64_t n, uint64_t rows, uint64_t cols, uint32_t unit)
{
    GradPlan p{};
    p.unsorted = unsorted_items(n, cols, unit);
    if (p.unsorted) return p;
    uint32_t bits = 1;
    while (bits < 32 && (rows >> bits) != 0) ++bits;  // values up to `rows`
    if (n <= kBucketTokens && rows <= kBucketRows) {
        p.rotate = kBucketBits;
        bits = bits > kBucketBits ? bits - kBucketBits : 0;
    } else {
        p.items = n <= kSmallTileTokens ? 2 : 8;
        p.tiles = static_cast<uint32_t>((n + p.items * kSortThreads - 1) / (p.items * kSortThreads));
    }
    p.passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
    p.digit_bits = p.passes ? (bits + p.passes - 1) / p.passes : 0;
    if (p.digit_bits < 6) p.digit_bits = 6;  // at least one counter for each thread that scans them
    const uint64_t block_cols = kLanes * unit;
    p.padded = static_cast<uint32_t>((cols + block_cols - 1) / block_cols * block_cols);
    // enough wavefronts to fill the chip, at most sixteen tokens each (see the sums)
    const uint64_t blocks = p.padded / block_cols;
    uint64_t per_wave = n * blocks / 8192;
    per_wave = per_wave < 4 ? 4 : per_wave > 16 ? 16 : per_wave;
    p.per_wave = static_cast<uint32_t>(per_wave);
    p.groups = static_cast<uint32_t>((n + per_wave * kSumWaves - 1) / (per_wave * kSumWaves));
    auto up = [](size_t x) { return (x + 255) & ~static_cast<size_t>(255); };
    const size_t list = up(n * 4), part = static_cast<size_t>(p.groups) * p.padded * 4;
    p.off_pos_a = list;
    p.off_row_b = 2 * list;
    p.off_pos_b = p.off_row_b + (p.tiles ? list : 0);
    p.off_count = p.off_pos_b + (p.tiles ? list : 0);
    p.off_head = p.off_count + (p.tiles ? up((static_cast<size_t>(p.tiles + 1) << p.digit_bits) * 4) : 0);
    p.off_tail = p.off_head + part;
    p.bytes = p.off_tail + part;
    return p;
}

// Lets a workgroup of KERNEL have `bytes` of dynamic LDS; the attribute is set once per device.
template <auto KERNEL>
int allow_lds(size_t bytes)
{
    static std::atomic<uint64_t> done{0};  // a bit per device
    int device = 0;
    FT_HIP(hipGetDevice(&device));
    const uint64_t bit = device < 64 ? 1ull << device : 0;
    if (done.load(std::memory_order_relaxed) & bit) return FT_OK;
    FT_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
    done.fetch_or(bit, std::memory_order_relaxed);
    return FT_OK;
}

// Sorts the call's tokens into the workspace; the results' places in a.row_s / a.pos_s.
int sort_tokens(GradPass& a, const GradPlan& p, char* ws, hipStream_t stream)
{
    uint32_t* row_a = reinterpret_cast<uint32_t*>(ws);
    uint32_t* pos_a = reinterpret_cast<uint32_t*>(ws + p.off_pos_a);
    uint32_t* row_b = reinterpret_cast<uint32_t*>(ws + p.off_row_b);
    uint32_t* pos_b = reinterpret_cast<uint32_t*>(ws + p.off_pos_b);
    SortPass s{};
    s.tokens = a.tokens;
    s.digit_bits = p.digit_bits;
    s.passes = p.passes;
    s.tiles = p.tiles;
    const size_t counters = (static_cast<size_t>(kSortWaves) << p.digit_bits) * 4;
    if (p.tiles == 0) {
        s.row_out = row_a;
        s.pos_out = pos_a;
        auto go = [&](auto items) -> int {
            constexpr int ITEMS = decltype(items)::value;
            constexpr size_t kList = ITEMS * kSortThreads * 4, kMostCounters = (static_cast<size_t>(kSortWaves) << kMaxDigitBits) * 4;
            const size_t lds = kList + counters;
            if constexpr (kList + kMostCounters + sizeof(uint32_t) * (kPairTokens + 64) > 65536) {
                const int rc = allow_lds<sort_buckets_kernel<ITEMS>>(kList + kMostCounters);
                if (rc != FT_OK) return rc;
            }
            hipLaunchKernelGGL(sort_buckets_kernel<ITEMS>, dim3(kBuckets), dim3(kSortThreads), lds, stream, s);
            FT_HIP(hipGetLastError());
            return FT_OK;
        };
        using std::integral_constant;
        const uint32_t n = a.tokens.n;
        const int rc = n <= kSortThreads       ? go(integral_constant<int, 1>{})
                       : n <= 2 * kSortThreads ? go(integral_constant<int, 2>{})
                       : n <= 4 * kSortThreads ? go(integral_constant<int, 4>{})
                       : n <= 8 * kSortThreads ? go(integral_constant<int, 8>{})
                                               : go(integral_constant<int, 16>{});
        if (rc != FT_OK) return rc;
    } else {
        s.count = reinterpret_cast<uint32_t*>(ws + p.off_count);
        s.scanned = p.tiles > kDirectTiles;
        for (uint32_t pass = 0; pass < p.passes; ++pass) {
            s.shift = pass * p.digit_bits;
            s.row_out = pass & 1 ? row_b : row_a;
            s.pos_out = pass & 1 ? pos_b : pos_a;
            if (p.items == 2)
                hipLaunchKernelGGL(sort_count_kernel<2>, dim3(p.tiles), dim3(kSortThreads), 0, stream, s);
            else
                hipLaunchKernelGGL(sort_count_kernel<8>, dim3(p.tiles), dim3(kSortThreads), 0, stream, s);
            FT_HIP(hipGetLastError());
            if (s.scanned) {
                hipLaunchKernelGGL(sort_scan_kernel, dim3((1u << p.digit_bits) / kLanes), dim3(kSortThreads), 0, stream, s);
                FT_HIP(hipGetLastError());
            }
            if (p.items == 2)
                hipLaunchKernelGGL(sort_place_kernel<2>, dim3(p.tiles), dim3(kSortThreads), counters, stream, s);
            else
                hipLaunchKernelGGL(sort_place_kernel<8>, dim3(p.tiles), dim3(kSortThreads), counters, stream, s);
            FT_HIP(hipGetLastError());
            s.row_in = s.row_out;
            s.pos_in = s.pos_out;
        }
    }
    a.row_s = s.row_out;
    a.pos_s = s.pos_out;
    a.rotate = p.rotate;
    return FT_OK;
}

template <int GT, int AT, bool DROP, bool RAGGED>
int launch_grad(GradPass a, const GradPlan& p, char* ws, hipStream_t stream)
{
    constexpr int U = row_unit<GT, AT>();
    unsigned clearing = a.accumulate ? 0 : (a.tokens.rows + kClearRows - 1) / kClearRows;
    if (clearing > kMostClearing) clearing = kMostClearing;
    if (p.unsorted) {
        const uint32_t sums = a.tokens.n * ((a.cols + kUnsortedBlocks * kLanes * U - 1) / (kUnsortedBlocks * kLanes * U));
        auto go = [&](auto items) -> int {
            hipLaunchKernelGGL((embedding_grad_unsorted_kernel<GT, AT, DROP, RAGGED, decltype(items)::value>), dim3(sums + clearing),
                               dim3(kUnsortedThreads), 0, stream, a, sums);
            FT_HIP(hipGetLastError());
            return FT_OK;
        };
        return p.unsorted == 1 ? go(std::integral_constant<int, 1>{}) : go(std::integral_constant<int, 2>{});
    }
    a.head = reinterpret_cast<float*>(ws + p.off_head);
    a.tail = reinterpret_cast<float*>(ws + p.off_tail);
    a.per_wave = p.per_wave;
    a.groups = p.groups;
    a.padded = p.padded;
    const int rc = sort_tokens(a, p, ws, stream);
    if (rc != FT_OK) return rc;
    const unsigned workgroups = p.groups * (p.padded / (kLanes * U));
    hipLaunchKernelGGL((embedding_grad_sum_kernel<GT, AT, DROP, RAGGED>), dim3(workgroups + clearing), dim3(kSumWaves * kLanes), 0, stream, a);
    FT_HIP(hipGetLastError());
    const unsigned light = (workgroups + kJoinWaves - 1) / kJoinWaves;
    const unsigned heavy = (p.groups - 1) / kLightParts * (p.padded / kHeavyCols);  // groups kLightParts, 2 kLightParts, ... below p.groups
    hipLaunchKernelGGL((embedding_grad_join_kernel<AT, U>), dim3(light + heavy), dim3(kJoinWaves * kLanes), 0, stream, a, light);
    FT_HIP(hipGetLastError());
    return FT_OK;
}

int check_tokens(const ft_tokens_t* t, size_t rows, Tokens* out)
{
    if (!t) return fth::fail(FT_EINVAL, "tokens must not be NULL");
    if (t->id_bytes != 4 && t->id_bytes != 8) return fth::fail(FT_EINVAL, "token ids have 4 or 8 bytes, not %d", t->id_bytes);
    if (t->first_row < 0) return fth::fail(FT_EINVAL, "first_row must not be negative");
    if (rows > kMaxCount) return fth::fail(FT_EINVAL, "a table has at most 2^31 - 1 rows");
    if (t->outer > kMaxCount || t->inner > kMaxCount || t->outer * t->inner > kMaxCount)
        return fth::fail(FT_EINVAL, "a call takes at most 2^31 - 1 tokens");
    auto reaches_too_far = [](uint64_t count, uint64_t stride) { return stride > kMaxReach / (count ? count : 1); };
    if (reaches_too_far(t->outer, t->outer_stride) || reaches_too_far(t->inner, t->inner_stride)) return fth::fail(FT_EINVAL, "token strides are too large");
    const uint64_t n = t->outer * t->inner;
    if (n && !t->ids) return fth::fail(FT_EINVAL, "ids must not be NULL");
    if (reinterpret_cast<uintptr_t>(t->ids) % static_cast<uintptr_t>(t->id_bytes)) return fth::fail(FT_EALIGN, "ids are not aligned to their size");
    out->ids = t->ids;
    out->wide = t->id_bytes == 8;
    out->n = static_cast<uint32_t>(n);
    out->inner = static_cast<uint32_t>(t->outer == 1 ? n : t->inner);
    out->outer_stride = t->outer_stride;
    out->inner_stride = t->inner_stride;
    out->first_row = static_cast<uint64_t>(t->first_row);
    out->padding = t->padding;
    out->rows = static_cast<uint32_t>(rows);
    return FT_OK;
}

int check_matrix(const char* name, const void* base, int dtype, uint64_t rows, uint64_t stride, uint64_t cols)
{
    if (!ftr::valid_dtype(dtype)) return fth::fail(FT_EINVAL, "unknown dtype code %d of %s", dtype, name);
    if (cols > kMaxCols) return fth::fail(FT_EINVAL, "a row has at most 2^24 elements, not %zu", static_cast<size_t>(cols));
    if (rows && (stride > ftr::kMaxElements / rows)) return fth::fail(FT_EINVAL, "the stride of %s is too large", name);
    if (rows && cols && !base) return fth::fail(FT_EINVAL, "%s must not be NULL", name);
    if (!ftr::aligned_to(base, dtype)) return fth::fail(FT_EALIGN, "%s is not aligned to its element size", name);
    return FT_OK;
}

}  // namespace

extern "C" {

int ft_embedding_lookup(const ft_tokens_t* tokens, const void* table, int table_dtype, size_t rows, size_t table_stride, void* out, int out_dtype,
                        size_t out_stride, size_t cols, double scale, const ft_dropout_t* drop, void* stream)
{
    LookupPass a{};
    int rc = check_tokens(tokens, rows, &a.tokens);
    if (rc == FT_OK) rc = check_matrix("table", table, table_dtype, rows, table_stride, cols);
    if (rc == FT_OK) rc = check_matrix("out", out, out_dtype, a.tokens.n, out_stride, cols);
    if (rc != FT_OK) return rc;
    if (a.tokens.n > 1 && out_stride < cols) return fth::fail(FT_EINVAL, "rows of out overlap: stride %zu, %zu elements", out_stride, cols);
    a.factor = static_cast<float>(scale);
    if (drop) {
        rc = ftr::dropout_args(drop, scale, &a.drop);
        if (rc != FT_OK) return rc;
        a.factor = a.drop.factor;
    }
    if (a.tokens.n == 0 || cols == 0) return FT_OK;
    if (ftr::overlap({table, table_dtype, rows, table_stride, cols}, {out, out_dtype, a.tokens.n, out_stride, cols}))
        return fth::fail(FT_EINVAL, "out overlaps the table");
    a.tokens.padding = FT_NO_PADDING;  // padding has a row like any other token
    a.table = table;
    a.out = out;
    a.table_stride = table_stride;
    a.out_stride = out_stride;
    a.cols = static_cast<uint32_t>(cols);
    const bool masked = drop && drop->p > 0.0;
    return ftr::with_dtype(table_dtype, [&](auto tt) {
        return ftr::with_dtype(out_dtype, [&](auto ot) {
            constexpr int TT = decltype(tt)::value, OT = decltype(ot)::value;
            const hipStream_t s = static_cast<hipStream_t>(stream);
            return masked ? launch_lookup<TT, OT, true>(a, s) : launch_lookup<TT, OT, false>(a, s);
        });
    });
}

size_t ft_embedding_grad_workspace_bytes(size_t n_tokens, size_t rows, size_t cols)
{
    if (n_tokens > kMaxCount || rows > kMaxCount || cols > kMaxCols) return 0;  // the call refuses these
    const size_t a = plan_grad(n_tokens, rows, cols, 4).bytes, b = plan_grad(n_tokens, rows, cols, 8).bytes;
    return a > b ? a : b;
}

int ft_embedding_grad(const ft_tokens_t* tokens, const void* g, int g_dtype, size_t g_stride, void* acc, int acc_dtype, size_t rows,
                      size_t acc_stride, size_t cols, double scale, int accumulate, const ft_dropout_t* drop, void* workspace,
                      size_t workspace_bytes, void* stream)
{
    GradPass a{};
    int rc = check_tokens(tokens, rows, &a.tokens);
    if (rc == FT_OK) rc = check_matrix("g", g, g_dtype, a.tokens.n, g_stride, cols);
    if (rc == FT_OK) rc = check_matrix("acc", acc, acc_dtype, rows, acc_stride, cols);
    if (rc != FT_OK) return rc;
    if (rows > 1 && acc_stride < cols) return fth::fail(FT_EINVAL, "rows of acc overlap: stride %zu, %zu elements", acc_stride, cols);
    a.factor = static_cast<float>(scale);
    if (drop) {
        rc = ftr::dropout_args(drop, scale, &a.drop);
        if (rc != FT_OK) return rc;
        a.factor = a.drop.factor;
    }
    const uint32_t unit = g_dtype == FT_F32 || acc_dtype == FT_F32 ? 4 : 8;  // row_unit
    const GradPlan plan = plan_grad(a.tokens.n, rows, cols, unit);
    const size_t need = ft_embedding_grad_workspace_bytes(a.tokens.n, rows, cols);
    if (rows == 0 || cols == 0 || (a.tokens.n == 0 && accumulate)) return FT_OK;
    if (need && (!workspace || workspace_bytes < need))
        return fth::fail(FT_EINVAL, "the workspace holds %zu bytes, %zu are needed", workspace ? workspace_bytes : 0, need);
    if (need && reinterpret_cast<uintptr_t>(workspace) % 16) return fth::fail(FT_EALIGN, "the workspace is not aligned to 16 bytes");
    // the sums' launch holds at most 2^32 - 1 work-items
    if (static_cast<uint64_t>(plan.groups) * (plan.padded / (kLanes * unit)) + kMostClearing > 0xffffffffull / (kSumWaves * kLanes))
        return fth::fail(FT_EINVAL, "%u tokens of %zu elements are too many for one call", a.tokens.n, cols);
    if (ftr::overlap({g, g_dtype, a.tokens.n, g_stride, cols}, {acc, acc_dtype, rows, acc_stride, cols}))
        return fth::fail(FT_EINVAL, "acc overlaps the gradient rows");
    a.g = g;
    a.acc = acc;
    a.g_stride = g_stride;
    a.acc_stride = acc_stride;
    a.cols = static_cast<uint32_t>(cols);
    a.accumulate = accumulate != 0;
    const bool masked = drop && drop->p > 0.0;
    return ftr::with_dtype(g_dtype, [&](auto gt) {
        return ftr::with_dtype(acc_dtype, [&](auto at) {
            constexpr int GT = decltype(gt)::value, AT = decltype(at)::value;
            char* ws = static_cast<char*>(workspace);
            const hipStream_t s = static_cast<hipStream_t>(stream);
            if (cols % row_unit<GT, AT>() != 0) return masked ? launch_grad<GT, AT, true, true>(a, plan, ws, s) : launch_grad<GT, AT, false, true>(a, plan, ws, s);
            return masked ? launch_grad<GT, AT, true, false>(a, plan, ws, s) : launch_grad<GT, AT, false, false>(a, plan, ws, s);
        });
    });
}

}  // extern "C"
