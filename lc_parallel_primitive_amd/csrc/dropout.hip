// dropout.hip — dropout of rows, with or without a residual added, from a
// counter-based generator (tensor.hpp): no mask is stored, the backward pass is
// the same call on the gradient.
//
//   out = (keep ? in / (1 - p) : 0) [+ residual]
//
// A thread takes octets (eight columns: one block of random bits, one or two
// 16-byte accesses a tensor) at a stride of the whole grid.  Its first octet's
// row and column take one division; every later step adds the grid's stride to
// them, which the host has divided.
//
// Bound by memory: 16384 x 8192 bfloat16 with a residual takes 142 to 145 us, 5.6
// TB/s of the bytes read and written once, where a copy of 512 MiB runs at 5.3.  The
// random bits are 14 wide products for eight elements, hidden behind the loads.
// The grid is what the device holds at once (2048 threads a CU), and the output is
// stored with the streaming policy, which nothing here reads again.
#include <algorithm>

#include "tensor.hpp"

namespace lcpp {
namespace {

struct DropoutArgs {
    const void *in, *residual;
    void *out;
    uint64_t in_stride, residual_stride, out_stride;
    uint64_t items;             // octets of all rows
    uint32_t cols, row_octets;  // of one row
    uint32_t step_rows, step_octets;  // the grid's stride
    DropArgs drop;
};

constexpr int kDropThreads = 256;
template <class T, bool ADD>
__global__ __launch_bounds__(kDropThreads) void dropout_kernel(DropoutArgs a)
{
    uint64_t item = (uint64_t)blockIdx.x * kDropThreads + threadIdx.x;
    if (item >= a.items) return;
    const uint64_t offset = drop_offset(a.drop);
    uint32_t row, octet;
    if (a.items <= 0xFFFFFFFFull) {
        row = (uint32_t)item / a.row_octets;
        octet = (uint32_t)item - row * a.row_octets;
    } else {
        row = (uint32_t)(item / a.row_octets);
        octet = (uint32_t)(item - (uint64_t)row * a.row_octets);
    }
    const uint64_t stride = (uint64_t)gridDim.x * kDropThreads;
    for (; item < a.items; item += stride) {
        const uint32_t col = octet * kOctet;
        const Octet<T> v = load_octet(static_cast<const T *>(a.in) + row * a.in_stride, col, a.cols);
        float x[kOctet];
#pragma unroll
        for (int i = 0; i < kOctet; ++i) x[i] = v[i];
        if (a.drop.cut) drop_octet(x, row, octet, offset, a.drop);
        if constexpr (ADD) {
            const Octet<T> r = load_octet(static_cast<const T *>(a.residual) + row * a.residual_stride, col, a.cols);
#pragma unroll
            for (int i = 0; i < kOctet; ++i) x[i] += r[i];
        }
        T *out = static_cast<T *>(a.out) + row * a.out_stride;
        if (col + kOctet <= a.cols) store_pack_nt<kOctet>(out + col, x);
        else store_octet(out, col, a.cols, x);
        row += a.step_rows;
        octet += a.step_octets;
        if (octet >= a.row_octets) {
            octet -= a.row_octets;
            ++row;
        }
    }
}

}  // namespace
}  // namespace lcpp

using namespace lcpp;

extern "C" int lcpp_dropout(lcpp_dtype t, const void *in, uint64_t in_stride, const void *residual,
                            uint64_t residual_stride, void *out, uint64_t out_stride, uint64_t rows, uint64_t cols,
                            double p, uint64_t seed, uint64_t offset, const uint64_t *offset_dev, void *stream)
{
    const size_t e = float_size(t);
    if (!e) return LCPP_ERR_UNSUPPORTED_DTYPE;
    DropoutArgs a = {};
    if (rows > kMaxRows || cols > kMaxCols || !drop_args(p, seed, offset, offset_dev, &a.drop)) return LCPP_ERR_INVALID_ARG;
    if (rows == 0 || cols == 0) return LCPP_OK;
    if (!elem_ok(in, e) || !elem_ok(out, e) || !rows_apart(out_stride, rows, cols)) return LCPP_ERR_INVALID_ARG;
    if (residual && !elem_ok(residual, e)) return LCPP_ERR_INVALID_ARG;
    a.in = in, a.residual = residual, a.out = out;
    a.in_stride = in_stride, a.residual_stride = residual_stride, a.out_stride = out_stride;
    a.cols = (uint32_t)cols;
    a.row_octets = (uint32_t)ceil_div(cols, kOctet);
    a.items = rows * a.row_octets;
    const uint32_t grid =
        (uint32_t)std::min<uint64_t>(ceil_div(a.items, kDropThreads), (uint64_t)device_cus() * 2048 / kDropThreads);
    const uint64_t step = (uint64_t)grid * kDropThreads;
    a.step_rows = (uint32_t)(step / a.row_octets);
    a.step_octets = (uint32_t)(step % a.row_octets);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return float_dispatch(t, [&](auto x) -> int {
        using T = decltype(x);
        if (a.residual) LCPP_LAUNCH("dropout_add", s, dropout_kernel<T, true><<<grid, kDropThreads, 0, s>>>(a));
        else LCPP_LAUNCH("dropout", s, dropout_kernel<T, false><<<grid, kDropThreads, 0, s>>>(a));
        LCPP_CHECK_LAUNCH();
        return LCPP_OK;
    });
}
