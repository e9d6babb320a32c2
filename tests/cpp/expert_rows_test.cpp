// expert_rows_test.cpp — rows that are only copied, through the C++ classes: the 8-bit rows and scales that an RMS
// norm writes, put in the experts' order for their product.  Built without assertions, so that refusals return.
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <vector>

#include "lcpp/parallel_primitive.h"

using namespace luisa::parallel_primitive;

static int g_failed;
static void report(const char *what, bool ok)
{
    g_failed += !ok;
    std::printf("%s %s\n", ok ? "ok" : "FAIL", what);
    std::fflush(stdout);
}

static_assert(row_dtype_of<const float>() == LCPP_FLOAT32 && row_dtype_of<bfloat16>() == LCPP_BFLOAT16);
static_assert(row_dtype_of<uint8_t>() == LCPP_FLOAT8_E4M3 && row_dtype_of<int32_t>() == LCPP_FLOAT32);

template <class T>
static void copy(CommandList &list, hipStream_t stream, const char *what)
{
    const size_t tokens = 5, choices = 2, cols = 37, rows = tokens * choices;
    std::vector<T> in(tokens * cols), out(rows * cols), got(rows * cols);
    for (size_t i = 0; i < in.size(); ++i) in[i] = (T)(i * 2654435761u >> 7);
    const std::vector<int32_t> positions = {3, 0, -1, 9, 4, 1, 2, 5, 8, 7};
    for (size_t p = 0; p < rows; ++p)
        for (size_t c = 0; c < cols && positions[p] >= 0; ++c) out[positions[p] * cols + c] = in[p / choices * cols + c];
    T *d_in = nullptr, *d_out = nullptr;
    int32_t *d_positions = nullptr;
    bool ok = hipMalloc(reinterpret_cast<void **>(&d_in), in.size() * sizeof(T)) == hipSuccess &&
              hipMalloc(reinterpret_cast<void **>(&d_out), out.size() * sizeof(T)) == hipSuccess &&
              hipMalloc(reinterpret_cast<void **>(&d_positions), rows * 4) == hipSuccess &&
              hipMemcpy(d_in, in.data(), in.size() * sizeof(T), hipMemcpyHostToDevice) == hipSuccess &&
              hipMemcpy(d_out, got.data(), got.size() * sizeof(T), hipMemcpyHostToDevice) == hipSuccess &&
              hipMemcpy(d_positions, positions.data(), rows * 4, hipMemcpyHostToDevice) == hipSuccess;
    if (!ok) std::abort();
    DeviceTokenSort order;
    order.Dispatch<T>(list, {d_in, cols}, d_positions, nullptr, {d_out, cols}, rows, tokens, choices, cols);
    ok = order.last_status() == LCPP_OK && hipStreamSynchronize(stream) == hipSuccess &&
         hipMemcpy(got.data(), d_out, got.size() * sizeof(T), hipMemcpyDeviceToHost) == hipSuccess && got == out;
    report(what, ok);
    float weights[rows] = {};  // (refused before anything is read)
    order.Dispatch<T>(list, {d_in, cols}, d_positions, weights, {d_out, cols}, rows, tokens, choices, cols);
    report("weights of such rows are refused", order.last_status() == LCPP_ERR_UNSUPPORTED_DTYPE);
    (void)hipFree(d_in);
    (void)hipFree(d_out);
    (void)hipFree(d_positions);
}

int main()
{
    hipStream_t stream;
    if (hipStreamCreate(&stream) != hipSuccess) return 1;
    CommandList list{stream};
    copy<uint8_t>(list, stream, "rows of 1 byte");
    copy<uint16_t>(list, stream, "rows of 2 bytes");
    copy<int32_t>(list, stream, "rows of 4 bytes");
    if (hipStreamDestroy(stream) != hipSuccess) return 1;
    std::printf("%s: %d failure(s)\n", g_failed ? "FAILED" : "PASSED", g_failed);
    return g_failed != 0;
}
