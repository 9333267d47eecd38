// ft_dropout.hip -- dropout with a mask that is never stored.
//
// out = [residual +] keep(i) * x / (1 - p), keep a pure function of (seed, substream, element index)
// (ft_counter.hpp): the backward pass calls the same kernel on the gradient and finds the same mask.
// HBM-bound: every array is read or written once, 4 bytes per element for a 16-bit x without a residual.
// Measured: 8192 x 4096 bf16 with a residual 32 us = 6.2 TB/s, 16384 x 8192 fp32 166 us = 6.5 TB/s, what
// this GPU's memory gives streaming kernels. The mask costs about nine vector instructions per element, which fit
// beside that traffic. One unit per lane and no loop: the loads of a wavefront are all in flight at once.
//
// The product is rounded to fp32 before the residual is added. A fused multiply-add would keep the factor's own
// rounding: 9 / 0.9 - 10 would not be 0, and sums on the border between two 16-bit numbers (one in a thousand at p = 0.1)
// would all go to the same side.
#include <cmath>
#include <type_traits>

#include "ft_counter.hpp"
#include "ft_internal.hpp"
#include "ft_row_args.hpp"
#include "ft_rows.hpp"

namespace {

using namespace ftk;

constexpr int kBlock = 256;

struct DropoutPass {
    const void* x;
    const void* residual;
    void* out;
    uint64_t x_stride, residual_stride, out_stride;
    uint64_t cols;          // elements of a row
    uint64_t units;         // units of this launch
    uint64_t first_unit;    // flat: unit of the launch's first lane
    uint64_t first_row;     // rows: row of the launch's first lane
    uint32_t units_per_row;
    ftc::DropoutArgs drop;
};

// One unit per lane. FLAT: the arrays are contiguous and count as one row.
template <int XT, int OT, bool RES, bool DROP, bool FLAT>
__global__ __launch_bounds__(kBlock) void dropout_kernel(DropoutPass a)
{
    constexpr int U = row_unit<XT, OT>();
    uint64_t xi, ri, oi, base;  // elements of the arrays; mask index of the unit: base + offset
    uint32_t offset, count = U;
    if constexpr (FLAT) {
        base = (a.first_unit + static_cast<uint64_t>(blockIdx.x) * kBlock) * U;  // wave-uniform
        offset = threadIdx.x * U;
        if (a.cols - base < kBlock * U) {  // the last workgroup
            const uint32_t left = static_cast<uint32_t>(a.cols - base);
            if (offset >= left) return;
            if (left - offset < U) count = left - offset;
        }
        xi = ri = oi = base + offset;
    } else {
        const uint32_t t = blockIdx.x * kBlock + threadIdx.x;
        if (t >= a.units) return;
        const uint32_t r = t / a.units_per_row;
        const uint64_t row = a.first_row + r;
        offset = (t - r * a.units_per_row) * U;
        if (a.cols - offset < U) count = static_cast<uint32_t>(a.cols) - offset;
        xi = row * a.x_stride + offset;
        ri = row * a.residual_stride + offset;
        oi = row * a.out_stride + offset;
        base = row * a.cols;
    }
    RowBits<XT, U> xb;
    RowBits<OT, U> rb;
    if (count == U) {
        xb = row_load<XT, U, true>(a.x, xi);
        if constexpr (RES) rb = row_load<OT, U, true>(a.residual, ri);
    } else {
        xb = row_load_some<XT, U>(a.x, xi, count);
        if constexpr (RES) rb = row_load_some<OT, U>(a.residual, ri, count);
    }
    bool keep[U];
    if constexpr (DROP) {
        const uint64_t b = a.drop.first + base;
        ftc::keep_units<U>(keep, ftc::group_argument(ftc::dropout_key(a.drop), b, offset), static_cast<uint32_t>(b) & 3u, a.drop);
    }
    float x[U], y[U];
    row_floats<XT, U>(x, xb);
    if constexpr (RES) row_floats<OT, U>(y, rb);
#pragma unroll
    for (int k = 0; k < U; ++k) {
        if constexpr (DROP) {  // a dropped element is 0 whatever x holds
            x[k] *= a.drop.factor;
            if constexpr (RES)
                y[k] = keep[k] ? y[k] + x[k] : y[k];
            else
                y[k] = keep[k] ? x[k] : 0.0f;
        } else {
            if constexpr (RES)
                y[k] = x[k] + y[k];
            else
                y[k] = x[k];
        }
    }
    if (count == U)
        row_store<OT, U, true>(a.out, oi, y);
    else
        row_store_some<OT, U>(a.out, oi, y, count);
}

template <int XT, int OT, bool RES, bool DROP>
int launch(DropoutPass a, uint64_t rows, hipStream_t stream)
{
    constexpr int U = row_unit<XT, OT>();
    const bool flat = rows == 1 || (a.x_stride == a.cols && a.out_stride == a.cols && (!RES || a.residual_stride == a.cols));
    if (flat) {
        a.cols *= rows;
        const uint64_t units = (a.cols + U - 1) / U;
        constexpr uint64_t kPiece = 1ull << 31;  // lanes per launch
        for (a.first_unit = 0; a.first_unit < units; a.first_unit += kPiece) {
            a.units = units - a.first_unit < kPiece ? units - a.first_unit : kPiece;
            hipLaunchKernelGGL((dropout_kernel<XT, OT, RES, DROP, true>), dim3(static_cast<unsigned>((a.units + kBlock - 1) / kBlock)),
                               dim3(kBlock), 0, stream, a);
            FT_HIP(hipGetLastError());
        }
        return FT_OK;
    }
    a.units_per_row = static_cast<uint32_t>((a.cols + U - 1) / U);
    const uint64_t piece = (1ull << 31) / a.units_per_row;  // rows per launch; cols is below 2^31
    for (a.first_row = 0; a.first_row < rows; a.first_row += piece) {
        const uint64_t now = rows - a.first_row < piece ? rows - a.first_row : piece;
        a.units = now * a.units_per_row;
        hipLaunchKernelGGL((dropout_kernel<XT, OT, RES, DROP, false>), dim3(static_cast<unsigned>((a.units + kBlock - 1) / kBlock)),
                           dim3(kBlock), 0, stream, a);
        FT_HIP(hipGetLastError());
    }
    return FT_OK;
}

}  // namespace

extern "C" {

int ft_dropout(const void* x, int x_dtype, size_t x_stride, const void* residual, size_t residual_stride, void* out, int out_dtype,
               size_t out_stride, size_t rows, size_t cols, const ft_dropout_t* drop, void* stream)
{
    if (!ftr::valid_dtype(x_dtype) || !ftr::valid_dtype(out_dtype)) return fth::fail(FT_EINVAL, "unknown dtype code %d / %d", x_dtype, out_dtype);
    if (!drop) return fth::fail(FT_EINVAL, "drop must not be NULL");
    DropoutPass a{};
    const int rc = ftr::dropout_args(drop, 1.0, &a.drop);
    if (rc != FT_OK) return rc;
    if (rows == 0 || cols == 0) return FT_OK;
    if (!x || !out) return fth::fail(FT_EINVAL, "x and out must not be NULL");
    const uint64_t most = ftr::kMaxElements / rows;
    if (rows > ftr::kMaxElements || cols > most) return fth::fail(FT_EINVAL, "%zu rows of %zu elements are too many", rows, cols);
    if (rows > 1 && (x_stride > most || out_stride > most || (residual && residual_stride > most)))
        return fth::fail(FT_EINVAL, "the distance of the rows is too large");
    if (rows > 1 && cols >= (1ull << 31) && !(x_stride == cols && out_stride == cols && (!residual || residual_stride == cols)))
        return fth::fail(FT_EINVAL, "rows that lie apart hold at most 2^31 - 1 elements");
    if (rows > 1 && out_stride < cols) return fth::fail(FT_EINVAL, "rows of out overlap: stride %zu, %zu elements", out_stride, cols);
    if (!ftr::aligned_to(x, x_dtype) || !ftr::aligned_to(out, out_dtype) || !ftr::aligned_to(residual, out_dtype))
        return fth::fail(FT_EALIGN, "x, residual and out must be aligned to their element size");
    const ftr::Rows from{x, x_dtype, rows, x_stride, cols}, added{residual, out_dtype, residual ? rows : 0, residual_stride, cols},
        to{out, out_dtype, rows, out_stride, cols};
    if ((!ftr::same_rows(from, to) && ftr::overlap(from, to)) || (!ftr::same_rows(added, to) && ftr::overlap(added, to)))
        return fth::fail(FT_EINVAL, "out overlaps x or residual and is not the same array");
    a.x = x;
    a.residual = residual;
    a.out = out;
    a.x_stride = x_stride;
    a.residual_stride = residual_stride;
    a.out_stride = out_stride;
    a.cols = cols;
    const bool masked = drop->p > 0.0;
    return ftr::with_dtype(x_dtype, [&](auto xt) {
        return ftr::with_dtype(out_dtype, [&](auto ot) {
            constexpr int XT = decltype(xt)::value, OT = decltype(ot)::value;
            const hipStream_t s = static_cast<hipStream_t>(stream);
            if (residual) return masked ? launch<XT, OT, true, true>(a, rows, s) : launch<XT, OT, true, false>(a, rows, s);
            return masked ? launch<XT, OT, false, true>(a, rows, s) : launch<XT, OT, false, false>(a, rows, s);
        });
    });
}

}  // extern "C"
