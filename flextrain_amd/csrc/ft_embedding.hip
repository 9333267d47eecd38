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
        const int64_t id = wide ? static_cast<const int64_t*>(ids)[at] : static_cast<int64_t>(static_cast<const int32_t*>(ids)[at]);
        const uint64_t r = static_cast<uint64_t>(id) - first_row;
        return r < rows && id != padding ? static_cast<uint32_t>(r) : kNoRow;
    }
};

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
// lane, several tokens per wavefront, for rows too short to feed 64 lanes.
template <int TT, int OT, bool DROP, int LPR, int K>
__global__ __launch_bounds__(256) void embedding_lookup_kernel(LookupPass a)
{
    const uint32_t wave = blockIdx.x * 4u + (threadIdx.x >> 6), lane = threadIdx.x & 63u;
    uint32_t token, col;
    if constexpr (LPR == kLanes) {
        const uint32_t w = __builtin_amdgcn_readfirstlane(wave);
        token = w / a.chunks;
        col = ((w - token * a.chunks) * K * kLanes + lane) * kRowUnit;
    } else {
        token = wave * (kLanes / LPR) + lane / LPR;
        col = (lane % LPR) * kRowUnit;
    }
    if (token >= a.tokens.n) return;
    const uint32_t row = a.tokens.row(token);
    const uint64_t from = static_cast<uint64_t>(row) * a.table_stride, to = token * a.out_stride;
    RowBits<TT> bits[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const uint32_t c = col + k * kLanes * kRowUnit;
        if (row == kNoRow || c >= a.cols) continue;
        bits[k] = a.cols - c >= kRowUnit ? row_load8<TT, false>(a.table, from + c) : row_load_some<TT>(a.table, from + c, a.cols - c);
    }
    uint64_t key = 0;
    if constexpr (DROP) key = ftc::dropout_key(a.drop);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const uint32_t c = col + k * kLanes * kRowUnit;
        if (c >= a.cols) continue;
        float x[kRowUnit] = {};
        if (row != kNoRow) {
            row_floats<TT>(x, bits[k]);
            bool keep[kRowUnit];
            if constexpr (DROP) ftc::keep8(keep, key, a.drop.first + static_cast<uint64_t>(token) * a.cols + c, a.drop.hi, a.drop.lo);
#pragma unroll
            for (int j = 0; j < kRowUnit; ++j) {
                x[j] *= a.factor;
                if constexpr (DROP) x[j] = keep[j] ? x[j] : 0.0f;
            }
        }
        if (a.cols - c >= kRowUnit)
            row_store8<OT, true>(a.out, to + c, x);
        else
            row_store_some<OT>(a.out, to + c, x, a.cols - c);
    }
}

template <int TT, int OT, bool DROP>
int launch_lookup(LookupPass a, hipStream_t stream)
{
    const uint32_t units = (a.cols + kRowUnit - 1) / kRowUnit;
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
    if (static_cast<uint64_t>(a.tokens.n) * ((units + kLanes - 1) / kLanes) < 16384) return go(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    return go(integral_constant<int, 64>{}, integral_constant<int, 4>{});
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
    const uint32_t* row_s;
    const uint32_t* pos_s;
    float* head;             // [groups][padded cols]: the end of a run that began in an earlier workgroup
    float* tail;             // the beginning of a run that goes on in the next one
    uint32_t per_wave;       // sorted tokens per wavefront
    uint32_t groups;         // workgroups per block of columns
    uint32_t padded;         // columns rounded up to whole blocks
};

// The gradient's unit of eight elements of token `pos` at column `col`, masked.
template <int GT, bool DROP>
__device__ __forceinline__ void add_unit(float (&sum)[kRowUnit], const RowBits<GT>& bits, const GradPass& a, uint64_t key, uint32_t pos, uint32_t col)
{
    float x[kRowUnit];
    row_floats<GT>(x, bits);
    if constexpr (DROP) {
        bool keep[kRowUnit];
        ftc::keep8(keep, key, a.drop.first + static_cast<uint64_t>(pos) * a.cols + col, a.drop.hi, a.drop.lo);
#pragma unroll
        for (int j = 0; j < kRowUnit; ++j) sum[j] += keep[j] ? x[j] : 0.0f;
    } else {
#pragma unroll
        for (int j = 0; j < kRowUnit; ++j) sum[j] += x[j];
    }
}

template <int GT>
__device__ __forceinline__ RowBits<GT> load_unit(const GradPass& a, uint32_t pos, uint32_t col, uint32_t count)
{
    const uint64_t at = static_cast<uint64_t>(pos) * a.g_stride + col;
    if (count == kRowUnit) return row_load8<GT, true>(a.g, at);
    return row_load_some<GT>(a.g, at, count);
}

// acc[row] (+)= factor * sum: the one rounding to the accumulator's type.
template <int AT>
__device__ __forceinline__ void finish_unit(const GradPass& a, uint32_t row, uint32_t col, uint32_t count, float (&sum)[kRowUnit])
{
    const uint64_t at = static_cast<uint64_t>(row) * a.acc_stride + col;
    float x[kRowUnit] = {};
    if (a.accumulate) row_floats<AT>(x, count == kRowUnit ? row_load8<AT, false>(a.acc, at) : row_load_some<AT>(a.acc, at, count));
#pragma unroll
    for (int j = 0; j < kRowUnit; ++j) x[j] = a.accumulate ? __builtin_fmaf(sum[j], a.factor, x[j]) : sum[j] * a.factor;
    if (count == kRowUnit)
        row_store8<AT, false>(a.acc, at, x);
    else
        row_store_some<AT>(a.acc, at, x, count);
}

// Short calls: one launch without sorting. The wavefront of a token looks through all tokens (two
// per lane); the first token of a row sums the row's gradients, the others leave.
constexpr uint32_t kShortTokens = 2 * kLanes;

template <int GT, int AT, bool DROP>
__global__ __launch_bounds__(kLanes) void embedding_grad_short_kernel(GradPass a)
{
    const uint32_t lane = threadIdx.x, n = a.tokens.n, me = blockIdx.x;
    const uint32_t r0 = lane < n ? a.tokens.row(lane) : kNoRow;
    const uint32_t r1 = lane + kLanes < n ? a.tokens.row(lane + kLanes) : kNoRow;
    const uint32_t mine = __builtin_amdgcn_readlane(me < kLanes ? r0 : r1, me & 63u);
    if (mine == kNoRow) return;
    uint64_t m0 = __builtin_amdgcn_ballot_w64(r0 == mine), m1 = __builtin_amdgcn_ballot_w64(r1 == mine);
    const uint32_t first = m0 ? __builtin_ctzll(m0) : kLanes + __builtin_ctzll(m1);
    if (first != me) return;
    const uint32_t col = (blockIdx.y * kLanes + lane) * kRowUnit;
    if (col >= a.cols) return;
    const uint32_t count = a.cols - col < kRowUnit ? a.cols - col : kRowUnit;
    uint64_t key = 0;
    if constexpr (DROP) key = ftc::dropout_key(a.drop);
    float sum[kRowUnit] = {};
    while (m0 | m1) {
        uint32_t pos[4];
        RowBits<GT> bits[4];
        int have = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (!(m0 | m1)) break;
            pos[j] = m0 ? __builtin_ctzll(m0) : kLanes + __builtin_ctzll(m1);
            if (m0) m0 &= m0 - 1;
            else m1 &= m1 - 1;
            bits[j] = load_unit<GT>(a, pos[j], col, count);
            have = j + 1;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < have) add_unit<GT, DROP>(sum, bits[j], a, key, pos[j], col);
    }
    finish_unit<AT>(a, mine, col, count, sum);
}

// ---- sorting the tokens by row ------------------------------------------------------------------
// Stable radix sort of (row, position), least significant digits first, tokens outside the table
// behind all others (as row `rows`). A workgroup ranks a tile of 1024 * R tokens: wavefront w holds
// 64 * R consecutive ones, 64 at a time, and counts them per digit in LDS counters of its own; lanes
// with the same digit find each other with one ballot per bit of the digit, so ranks follow the order
// of the tokens and no LDS atomic is needed. Calls of at most one tile sort in one launch, all
// passes in LDS; longer ones take two launches a pass (count, place).
constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kLanes;
constexpr int kSortItems = 8;                             // R at most
constexpr uint32_t kSortTile = kSortThreads * kSortItems;
constexpr uint32_t kMaxDigitBits = 9;

struct SortPass {
    Tokens tokens;
    const uint32_t* row_in;  // nullptr: the first pass, rows come from the tokens
    const uint32_t* pos_in;
    uint32_t* row_out;
    uint32_t* pos_out;
    uint32_t* count;         // [tiles][1 << digit_bits]
    uint32_t shift, digit_bits, passes, tiles;
};

__device__ __forceinline__ uint32_t sort_key(const Tokens& t, uint32_t i)
{
    const uint32_t r = t.row(i);
    return r == kNoRow ? t.rows : r;
}

// Lanes of the wavefront whose digit is this lane's; `active` lanes only.
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, uint32_t bits, bool active)
{
    uint64_t m = __builtin_amdgcn_ballot_w64(active);
    for (uint32_t b = 0; b < bits; ++b) {
        const bool one = digit >> b & 1u;
        const uint64_t v = __builtin_amdgcn_ballot_w64(one);
        m &= one ? v : ~v;
    }
    return m;
}

// Sum over the threads before this one (1024 threads); total of all in *total.
__device__ __forceinline__ uint32_t exclusive_scan(uint32_t x, uint32_t* wave_sums, uint32_t* total)
{
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t s = x;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const uint32_t y = __shfl_up(s, d);
        if (lane >= d) s += y;
    }
    __syncthreads();
    if (lane == 63) wave_sums[wave] = s;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kSortWaves; ++w) {
        const uint32_t v = wave_sums[w];
        before += w < wave ? v : 0;
        all += v;
    }
    *total = all;
    return before + s - x;
}

// Ranks the tile's items by digit. counters[w][digit] ends as the number of the wavefront's items
// with that digit; rank[] as the number of them in front of each item.
__device__ __forceinline__ void rank_items(uint32_t (&rank)[kSortItems], const uint32_t (&key)[kSortItems], uint32_t r_count, uint32_t base, uint32_t n,
                                           uint32_t shift, uint32_t bits, uint32_t* counters)
{
    const uint32_t lane = threadIdx.x & 63u, bins = 1u << bits;
    volatile uint32_t* mine = counters + (threadIdx.x >> 6) * bins;
    for (uint32_t b = lane; b < bins; b += kLanes) mine[b] = 0;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
        if (static_cast<uint32_t>(r) >= r_count) break;
        const bool active = base + r * kLanes + lane < n;
        const uint32_t digit = key[r] >> shift & (bins - 1);
        const uint64_t same = same_digit(digit, bits, active);
        const uint32_t in_front = __builtin_popcountll(same & ((1ull << lane) - 1));
        const uint32_t before = active ? mine[digit] : 0;
        rank[r] = before + in_front;
        __builtin_amdgcn_wave_barrier();
        if (active && in_front == 0) mine[digit] = before + __builtin_popcountll(same);
        __builtin_amdgcn_wave_barrier();
    }
}

// One launch: at most kSortTile tokens.
__global__ __launch_bounds__(kSortThreads) void sort_tile_kernel(SortPass a)
{
    extern __shared__ uint32_t lds[];
    const uint32_t bins = 1u << a.digit_bits, n = a.tokens.n;
    uint32_t* counters = lds;                          // [kSortWaves][bins]
    uint32_t* wave_sums = counters + kSortWaves * bins;  // [kSortWaves]
    uint32_t* rows = wave_sums + kSortWaves;            // [r_count * 1024]
    const uint32_t r_count = (n + kSortThreads - 1) / kSortThreads;
    uint32_t* positions = rows + r_count * kSortThreads;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t base = wave * kLanes * r_count;
    uint32_t key[kSortItems], pos[kSortItems], rank[kSortItems];
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
        if (static_cast<uint32_t>(r) >= r_count) break;
        pos[r] = base + r * kLanes + lane;
        key[r] = pos[r] < n ? sort_key(a.tokens, pos[r]) : 0;
    }
    const uint32_t each = bins * kSortWaves / kSortThreads;  // counters a thread scans: 1 ... 8
    for (uint32_t pass = 0; pass < a.passes; ++pass) {
        const uint32_t shift = pass * a.digit_bits;
        rank_items(rank, key, r_count, base, n, shift, a.digit_bits, counters);
        __syncthreads();
        // offsets in the order (digit, wavefront)
        uint32_t local[8], sum = 0, total;
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) {
            if (k >= each) break;
            const uint32_t e = threadIdx.x * each + k;
            local[k] = counters[(e % kSortWaves) * bins + e / kSortWaves];
            sum += local[k];
        }
        uint32_t at = exclusive_scan(sum, wave_sums, &total);
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) {
            if (k >= each) break;
            const uint32_t e = threadIdx.x * each + k;
            counters[(e % kSortWaves) * bins + e / kSortWaves] = at;
            at += local[k];
        }
        __syncthreads();
        const bool last = pass + 1 == a.passes;
#pragma unroll
        for (int r = 0; r < kSortItems; ++r) {
            if (static_cast<uint32_t>(r) >= r_count) break;
            if (base + r * kLanes + lane >= n) continue;
            const uint32_t to = counters[wave * bins + (key[r] >> shift & (bins - 1))] + rank[r];
            if (last) {
                a.row_out[to] = key[r];
                a.pos_out[to] = pos[r];
            } else {
                rows[to] = key[r];
                positions[to] = pos[r];
            }
        }
        if (last) break;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kSortItems; ++r) {
            if (static_cast<uint32_t>(r) >= r_count) break;
            const uint32_t i = base + r * kLanes + lane;
            if (i < n) {
                key[r] = rows[i];
                pos[r] = positions[i];
            }
        }
        __syncthreads();
    }
}

// Long calls, first launch of a pass: how often each digit occurs in each tile.
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(SortPass a)
{
    extern __shared__ uint32_t lds[];
    const uint32_t bins = 1u << a.digit_bits, n = a.tokens.n;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t base = blockIdx.x * kSortTile + wave * kLanes * kSortItems;
    uint32_t key[kSortItems], rank[kSortItems];
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
        const uint32_t i = base + r * kLanes + lane;
        key[r] = i < n ? (a.row_in ? a.row_in[i] : sort_key(a.tokens, i)) : 0;
    }
    rank_items(rank, key, kSortItems, base, n, a.shift, a.digit_bits, lds);
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < bins; b += kSortThreads) {
        uint32_t sum = 0;
        for (uint32_t w = 0; w < kSortWaves; ++w) sum += lds[w * bins + b];
        a.count[blockIdx.x * bins + b] = sum;
    }
}

// Second launch of a pass: every tile adds up where its digits begin and moves its tokens there.
__global__ __launch_bounds__(kSortThreads) void sort_place_kernel(SortPass a)
{
    extern __shared__ uint32_t lds[];
    const uint32_t bins = 1u << a.digit_bits, n = a.tokens.n;
    uint32_t* counters = lds;                            // [kSortWaves][bins]
    uint32_t* wave_sums = counters + kSortWaves * bins;    // [kSortWaves]
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t base = blockIdx.x * kSortTile + wave * kLanes * kSortItems;
    uint32_t key[kSortItems], pos[kSortItems], rank[kSortItems];
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
        const uint32_t i = base + r * kLanes + lane;
        key[r] = i < n ? (a.row_in ? a.row_in[i] : sort_key(a.tokens, i)) : 0;
        pos[r] = i < n ? (a.row_in ? a.pos_in[i] : i) : 0;
    }
    rank_items(rank, key, kSortItems, base, n, a.shift, a.digit_bits, counters);
    __syncthreads();
    // this digit in the tiles before this one, and in all tiles
    uint32_t before = 0, all = 0, total;
    if (threadIdx.x < bins) {
        for (uint32_t t = 0; t < a.tiles; ++t) {
            const uint32_t c = a.count[t * bins + threadIdx.x];
            before += t < blockIdx.x ? c : 0;
            all += c;
        }
    }
    uint32_t at = exclusive_scan(all, wave_sums, &total) + before;
    if (threadIdx.x < bins) {
        for (uint32_t w = 0; w < kSortWaves; ++w) {
            const uint32_t c = counters[w * bins + threadIdx.x];
            counters[w * bins + threadIdx.x] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
        if (base + r * kLanes + lane >= n) continue;
        const uint32_t to = counters[wave * bins + (key[r] >> a.shift & (bins - 1))] + rank[r];
        a.row_out[to] = key[r];
        a.pos_out[to] = pos[r];
    }
}

// ---- summing runs of equal rows -------------------------------------------------------------------
// Workgroup (block of 512 columns, group): four wavefronts with per_wave consecutive sorted tokens
// each, eight columns per lane. A run inside a wavefront goes straight to the accumulator; one that
// crosses into the next wavefront is joined in LDS by the wavefront it begins in, one that crosses
// into the next workgroup leaves its parts in head / tail for embedding_grad_join_kernel.
constexpr int kSumWaves = 4;
constexpr int kBlockCols = kLanes * kRowUnit;
constexpr int kAhead = 8;  // gradient rows in flight per wavefront

template <int GT, int AT, bool DROP>
__global__ __launch_bounds__(kSumWaves * kLanes) void embedding_grad_sum_kernel(GradPass a)
{
    __shared__ float parts[kSumWaves][2][kRowUnit][kLanes];  // 0: head, 1: tail
    __shared__ uint32_t head_row[kSumWaves], tail_row[kSumWaves];  // kNoRow: none
    __shared__ uint32_t through[kSumWaves];                        // the head goes on behind the wavefront's end
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t n = a.tokens.n, rows = a.tokens.rows;
    const uint32_t blocks = a.padded / kBlockCols;
    const uint32_t group = blockIdx.x / blocks;
    const uint32_t col = ((blockIdx.x - group * blocks) * kLanes + lane) * kRowUnit;
    const uint32_t count = col >= a.cols ? 0 : (a.cols - col < kRowUnit ? a.cols - col : kRowUnit);
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
        float sum[kRowUnit] = {};
        uint32_t row = __builtin_amdgcn_readlane(my_row, 0);
        bool head = row == prev;  // the run that is being summed began before this wavefront
        auto flush = [&](uint32_t r, bool goes_on) {
            if (head || goes_on) {
                const int slot = head ? 0 : 1;
#pragma unroll
                for (int j = 0; j < kRowUnit; ++j) parts[wave][slot][j][lane] = sum[j];
                if (head) {
                    h_row = r;
                    thru = goes_on;
                } else {
                    t_row = r;
                }
            } else if (count) {
                finish_unit<AT>(a, r, col, count, sum);
            }
            head = false;
        };
        for (uint32_t j0 = 0; j0 < valid; j0 += kAhead) {
            RowBits<GT> bits[kAhead];
            uint32_t pos[kAhead], r[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const uint32_t at = j0 + j < valid ? j0 + j : valid - 1;
                pos[j] = __builtin_amdgcn_readlane(my_pos, at);
                r[j] = __builtin_amdgcn_readlane(my_row, at);
                if (j0 + j < valid && count) bits[j] = load_unit<GT>(a, pos[j], col, count);
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (j0 + j >= valid) break;
                if (r[j] != row) {
                    flush(row, false);
                    row = r[j];
#pragma unroll
                    for (int e = 0; e < kRowUnit; ++e) sum[e] = 0.0f;
                }
                if (count) add_unit<GT, DROP>(sum, bits[j], a, key, pos[j], col);
            }
        }
        flush(row, row == next);
    }
    if (lane == 0) {
        head_row[wave] = h_row;
        tail_row[wave] = t_row;
        through[wave] = thru;
    }
    __syncthreads();
    if (!count) return;
    const uint64_t slot = static_cast<uint64_t>(group) * a.padded + col;
    // The wavefront a run begins in joins it; the one that came in from the workgroup before, wavefront 0.
    auto join = [&](uint32_t r, uint32_t w, int first_slot, bool goes_on, bool from_before) {
        float sum[kRowUnit];
#pragma unroll
        for (int j = 0; j < kRowUnit; ++j) sum[j] = parts[w][first_slot][j][lane];
        while (goes_on && ++w < kSumWaves) {
#pragma unroll
            for (int j = 0; j < kRowUnit; ++j) sum[j] += parts[w][0][j][lane];
            goes_on = through[w];
        }
        if (from_before || goes_on) {
            float* to = (from_before ? a.head : a.tail) + slot;
#pragma unroll
            for (int j = 0; j < kRowUnit; ++j) to[j] = sum[j];
        } else {
            finish_unit<AT>(a, r, col, count, sum);
        }
    };
    if (wave == 0 && head_row[0] != kNoRow) join(head_row[0], 0, 0, through[0], true);
    if (tail_row[wave] != kNoRow) join(tail_row[wave], wave, 1, true, false);
}

// Runs that cross workgroups: the workgroup that a run begins in adds the parts up, each of its four
// wavefronts a quarter of them.
template <int AT>
__global__ __launch_bounds__(kSumWaves * kLanes) void embedding_grad_join_kernel(GradPass a)
{
    __shared__ float parts[kSumWaves][kRowUnit][kLanes];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t blocks = a.padded / kBlockCols;
    const uint32_t group = blockIdx.x / blocks;
    const uint64_t per_group = static_cast<uint64_t>(a.per_wave) * kSumWaves;
    const uint64_t begin = group * per_group, end = begin + per_group;
    const uint32_t n = a.tokens.n;
    if (end >= n) return;
    const uint32_t row = a.row_s[end];
    if (row >= a.tokens.rows || a.row_s[end - 1] != row) return;
    if (a.row_s[begin] == row && begin > 0 && a.row_s[begin - 1] == row) return;  // began earlier
    uint32_t heads = 0;  // groups behind this one that begin inside the run
    for (uint32_t first = group + 1;; first += kLanes) {
        const uint64_t at = static_cast<uint64_t>(first + lane) * per_group;
        const uint64_t in = __builtin_amdgcn_ballot_w64(at < n && a.row_s[at < n ? at : 0] == row);
        const uint32_t run = ~in ? __builtin_ctzll(~in) : kLanes;
        heads += run;
        if (run < kLanes) break;
    }
    const uint32_t col = ((blockIdx.x - group * blocks) * kLanes + lane) * kRowUnit;
    const uint32_t parts_all = heads + 1;  // the tail of this group, then the heads
    const uint32_t lo = static_cast<uint64_t>(parts_all) * wave / kSumWaves, hi = static_cast<uint64_t>(parts_all) * (wave + 1) / kSumWaves;
    float sum[kRowUnit] = {};
#pragma unroll 4
    for (uint32_t k = lo; k < hi; ++k) {
        const float* from = (k == 0 ? a.tail : a.head) + static_cast<uint64_t>(group + k) * a.padded + col;
#pragma unroll
        for (int j = 0; j < kRowUnit; ++j) sum[j] += from[j];
    }
#pragma unroll
    for (int j = 0; j < kRowUnit; ++j) parts[wave][j][lane] = sum[j];
    __syncthreads();
    if (wave != 0 || col >= a.cols) return;
#pragma unroll
    for (int w = 1; w < kSumWaves; ++w)
#pragma unroll
        for (int j = 0; j < kRowUnit; ++j) sum[j] += parts[w][j][lane];
    finish_unit<AT>(a, row, col, a.cols - col < kRowUnit ? a.cols - col : kRowUnit, sum);
}

// ---- rows without a token ----------------------------------------------------------------------
// A gradient that is written, not added: the other rows become zero. A workgroup owns 64 rows; each
// lane looks its row up among the tokens (binary search in the sorted ones, all of them in a short
// call).
template <int AT>
__global__ __launch_bounds__(256) void embedding_grad_clear_kernel(GradPass a)
{
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t n = a.tokens.n, first = blockIdx.x * kLanes, row = first + lane;
    bool met = false;
    if (a.row_s) {
        uint32_t lo = 0, hi = n;  // the first sorted token of a row not below this one
        while (lo < hi) {
            const uint32_t mid = (lo + hi) >> 1;
            if (a.row_s[mid] < row)
                lo = mid + 1;
            else
                hi = mid;
        }
        met = lo < n && a.row_s[lo] == row;
    } else {
        for (uint32_t i = 0; i < n; ++i) met |= a.tokens.row(i) == row;
    }
    uint64_t clear = __builtin_amdgcn_ballot_w64(!met && row < a.tokens.rows);
    const float zero[kRowUnit] = {};
    for (uint32_t k = 0; clear; ++k, clear &= clear - 1) {
        if ((k & 3u) != wave) continue;
        const uint64_t at = static_cast<uint64_t>(first + __builtin_ctzll(clear)) * a.acc_stride;
        for (uint32_t col = lane * kRowUnit; col < a.cols; col += kBlockCols) {
            if (a.cols - col >= kRowUnit)
                row_store8<AT, true>(a.acc, at + col, zero);
            else
                row_store_some<AT>(a.acc, at + col, zero, a.cols - col);
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------
struct GradPlan {
    uint32_t digit_bits, passes, tiles;
    uint32_t per_wave, groups, padded;
    size_t off_pos_a, off_row_b, off_pos_b, off_count, off_head, off_tail, bytes;  // row_a at 0
};

GradPlan plan_grad(uint64_t n, uint64_t rows, uint64_t cols)
{
    GradPlan p{};
    if (n <= kShortTokens) return p;
    uint32_t bits = 1;
    while (bits < 32 && (rows >> bits) != 0) ++bits;  // values up to `rows`
    p.passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
    p.digit_bits = (bits + p.passes - 1) / p.passes;
    if (p.digit_bits < 6) p.digit_bits = 6;  // at least one counter for each thread of the scan
    p.tiles = static_cast<uint32_t>((n + kSortTile - 1) / kSortTile);
    p.padded = static_cast<uint32_t>((cols + kBlockCols - 1) / kBlockCols * kBlockCols);
    // enough wavefronts to fill the chip, at most 64 tokens each
    const uint64_t blocks = p.padded / kBlockCols;
    uint64_t per_wave = n * blocks / 8192;
    per_wave = per_wave < 4 ? 4 : per_wave > 64 ? 64 : per_wave;
    p.per_wave = static_cast<uint32_t>(per_wave);
    p.groups = static_cast<uint32_t>((n + per_wave * kSumWaves - 1) / (per_wave * kSumWaves));
    auto up = [](size_t x) { return (x + 255) & ~static_cast<size_t>(255); };
    const size_t list = up(n * 4), part = static_cast<size_t>(p.groups) * p.padded * 4;
    p.off_pos_a = list;
    p.off_row_b = 2 * list;
    p.off_pos_b = 3 * list;
    p.off_count = 4 * list;
    p.off_head = p.off_count + up((static_cast<size_t>(p.tiles) << p.digit_bits) * 4);
    p.off_tail = p.off_head + part;
    p.bytes = p.off_tail + part;
    return p;
}

template <typename K>
int allow_lds(K kernel, size_t bytes)
{
    if (bytes > 65536) FT_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
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
    s.count = reinterpret_cast<uint32_t*>(ws + p.off_count);
    const size_t counters = (static_cast<size_t>(kSortWaves) << p.digit_bits) * 4 + kSortWaves * 4;
    if (p.tiles == 1) {
        s.row_out = row_a;
        s.pos_out = pos_a;
        const size_t r_count = (a.tokens.n + kSortThreads - 1) / kSortThreads;
        const size_t lds = counters + 2 * r_count * kSortThreads * 4;
        const int rc = allow_lds(sort_tile_kernel, lds);
        if (rc != FT_OK) return rc;
        hipLaunchKernelGGL(sort_tile_kernel, dim3(1), dim3(kSortThreads), lds, stream, s);
        FT_HIP(hipGetLastError());
    } else {
        for (uint32_t pass = 0; pass < p.passes; ++pass) {
            s.shift = pass * p.digit_bits;
            s.row_out = pass & 1 ? row_b : row_a;
            s.pos_out = pass & 1 ? pos_b : pos_a;
            hipLaunchKernelGGL(sort_count_kernel, dim3(p.tiles), dim3(kSortThreads), counters, stream, s);
            FT_HIP(hipGetLastError());
            hipLaunchKernelGGL(sort_place_kernel, dim3(p.tiles), dim3(kSortThreads), counters, stream, s);
            FT_HIP(hipGetLastError());
            s.row_in = s.row_out;
            s.pos_in = s.pos_out;
        }
    }
    a.row_s = s.row_out;
    a.pos_s = s.pos_out;
    return FT_OK;
}

template <int GT, int AT, bool DROP>
int launch_grad(GradPass a, const GradPlan& p, char* ws, hipStream_t stream)
{
    const bool shorter = a.tokens.n <= kShortTokens;
    if (!shorter) {
        a.head = reinterpret_cast<float*>(ws + p.off_head);
        a.tail = reinterpret_cast<float*>(ws + p.off_tail);
        a.per_wave = p.per_wave;
        a.groups = p.groups;
        a.padded = p.padded;
        const int rc = sort_tokens(a, p, ws, stream);
        if (rc != FT_OK) return rc;
    }
    if (!a.accumulate) {
        hipLaunchKernelGGL((embedding_grad_clear_kernel<AT>), dim3((a.tokens.rows + kLanes - 1) / kLanes), dim3(256), 0, stream, a);
        FT_HIP(hipGetLastError());
    }
    if (a.tokens.n == 0) return FT_OK;
    if (shorter) {
        hipLaunchKernelGGL((embedding_grad_short_kernel<GT, AT, DROP>), dim3(a.tokens.n, (a.cols + kBlockCols - 1) / kBlockCols), dim3(kLanes), 0,
                           stream, a);
        FT_HIP(hipGetLastError());
        return FT_OK;
    }
    const unsigned workgroups = p.groups * (p.padded / kBlockCols);
    hipLaunchKernelGGL((embedding_grad_sum_kernel<GT, AT, DROP>), dim3(workgroups), dim3(kSumWaves * kLanes), 0, stream, a);
    FT_HIP(hipGetLastError());
    hipLaunchKernelGGL((embedding_grad_join_kernel<AT>), dim3(workgroups), dim3(kSumWaves * kLanes), 0, stream, a);
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
    if (t->outer_stride > ftr::kMaxElements >> 31 || t->inner_stride > ftr::kMaxElements >> 31) return fth::fail(FT_EINVAL, "token strides are too large");
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
    return plan_grad(n_tokens, rows, cols).bytes;
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
    const GradPlan plan = plan_grad(a.tokens.n, rows, cols);
    if (rows == 0 || cols == 0 || (a.tokens.n == 0 && accumulate)) return FT_OK;
    if (plan.bytes && (!workspace || workspace_bytes < plan.bytes))
        return fth::fail(FT_EINVAL, "the workspace holds %zu bytes, %zu are needed", workspace ? workspace_bytes : 0, plan.bytes);
    if (plan.bytes && reinterpret_cast<uintptr_t>(workspace) % 16) return fth::fail(FT_EALIGN, "the workspace is not aligned to 16 bytes");
    if (static_cast<uint64_t>(plan.groups) * (plan.padded / kBlockCols) > 0xffffffull)
        return fth::fail(FT_EINVAL, "%u tokens of %zu elements are too many for one call", a.tokens.n, cols);
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
            return masked ? launch_grad<GT, AT, true>(a, plan, ws, s) : launch_grad<GT, AT, false>(a, plan, ws, s);
        });
    });
}

}  // extern "C"
