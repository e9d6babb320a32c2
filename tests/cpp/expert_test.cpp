// expert_test.cpp — RMS norm, expert router, tokens sorted by expert and the experts'
// products through the C++ classes (include/lcpp/parallel_primitive.h) on a GPU, one
// behind the other, against their definitions in double on the host.  Prints one line
// per check and "PASSED: 0 failure(s)".
#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <vector>

#include "lcpp/parallel_primitive.h"

using namespace luisa::parallel_primitive;

static int g_failed;
static void report(const char *what, double off, double bound)
{
    const bool ok = off <= bound;
    g_failed += !ok;
    std::printf("%s %s (off by %.3g, bound %.3g)\n", ok ? "ok" : "FAIL", what, off, bound);
    std::fflush(stdout);
}

template <class T>
struct Dev {
    T *p = nullptr;
    size_t n;
    explicit Dev(size_t count) : n(count)
    {
        if (hipMalloc(reinterpret_cast<void **>(&p), count * sizeof(T)) != hipSuccess) std::abort();
    }
    explicit Dev(const std::vector<T> &v) : Dev(v.size())
    {
        if (hipMemcpy(p, v.data(), n * sizeof(T), hipMemcpyHostToDevice) != hipSuccess) std::abort();
    }
    std::vector<T> host() const
    {
        std::vector<T> v(n);
        if (hipMemcpy(v.data(), p, n * sizeof(T), hipMemcpyDeviceToHost) != hipSuccess) std::abort();
        return v;
    }
    ~Dev() { (void)hipFree(p); }
    Dev(const Dev &) = delete;
};

static std::vector<float> values(size_t n, unsigned seed, float scale, float shift)
{
    std::vector<float> v(n);
    uint32_t s = seed * 2654435761u + 1;
    for (auto &x : v) {
        s = s * 1664525u + 1013904223u;
        x = ((float)(s >> 8) / 16777216.0f - 0.5f) * scale + shift;
    }
    return v;
}
static double worst(const std::vector<float> &got, const std::vector<double> &want)
{
    double w = 0;
    for (size_t i = 0; i < got.size(); ++i) w = std::fmax(w, std::fabs(got[i] - want[i]));
    return w;
}

int main()
{
    hipStream_t stream;
    if (hipStreamCreate(&stream) != hipSuccess) return 1;
    Device device{0};
    Stream debug{stream};
    CommandList list{stream};
    const size_t tokens = 45, cols = 136, experts = 6, choices = 2, outputs = 72, pairs = tokens * choices;
    const float eps = 1e-6f;
    const double u = 1 / 16777216.0;
    const auto hx = values(tokens * cols, 1, 4.0f, 0.3f), hr = values(tokens * cols, 2, 2.0f, 0.0f), hw = values(cols, 3, 1.0f, 1.0f);
    const auto hl = values(tokens * experts, 4, 6.0f, 0.0f), hm = values(experts * outputs * cols, 5, 0.4f, 0.0f);
    const auto hg = values(tokens * outputs, 6, 2.0f, 0.0f);
    Dev<float> x(hx), r(hr), w(hw), logits(hl), matrices(hm), g(hg);
    Dev<float> s(tokens * cols), y(tokens * cols), rstd(tokens), scales(tokens * 2), weights(pairs);
    Dev<uint8_t> quant(tokens * cols);
    Dev<int32_t> ids(pairs), positions(pairs), offsets(experts + 1), sources(pairs);
    Dev<float> rows(pairs * cols), results(pairs * outputs), out(tokens * outputs);

    DeviceRMSNorm norm;
    DeviceExpertRouter router;
    DeviceTokenSort order;
    DeviceExpertProduct product;
    norm.create(device, &debug);
    router.create(device, &debug);
    order.create(device, &debug);
    product.create(device, &debug);
    const EightBits eight{LCPP_FLOAT8_E4M3, quant.p, cols, scales.p, 2, 1, 128};
    norm.AddForward<float, float>(list, {x.p, cols}, {r.p, cols}, {s.p, cols}, {y.p, cols}, w.p, eps, rstd.p, tokens, cols, eight);
    const RouterScore how{LCPP_SCORE_SOFTMAX, true, 1.0f};
    router.Forward<float>(list, {logits.p, experts}, nullptr, ids.p, weights.p, how, tokens, experts, choices);
    Dev<uint> temp(64);
    order.Sort(list, {temp.p, temp.n}, ids.p, tokens, choices, experts, positions.p, offsets.p, sources.p);
    report("status of the sort", order.last_status(), 0);
    order.Dispatch<float>(list, {y.p, cols}, positions.p, nullptr, {rows.p, cols}, pairs, tokens, choices, cols);
    product.Forward<float>(list, {rows.p, cols}, {matrices.p, cols, outputs * cols}, offsets.p, {results.p, outputs}, pairs, experts,
                           outputs, cols);
    order.Combine<float>(list, {results.p, outputs}, positions.p, weights.p, {out.p, outputs}, {}, pairs, tokens, choices, outputs);
    if (hipStreamSynchronize(stream) != hipSuccess) return 1;

    std::vector<double> wy(tokens * cols), wout(tokens * outputs, 0.0), ww(pairs);
    std::vector<int> best(pairs), count(experts + 1, 0);
    double off_scale = 0;
    const auto sc = scales.host();
    for (size_t t = 0; t < tokens; ++t) {
        double sq = 0;
        for (size_t c = 0; c < cols; ++c) sq += std::pow((double)(hr[t * cols + c] + hx[t * cols + c]), 2);
        const double rs = 1 / std::sqrt(sq / cols + eps);
        double most[2] = {0, 0};
        for (size_t c = 0; c < cols; ++c) {
            wy[t * cols + c] = (double)(hr[t * cols + c] + hx[t * cols + c]) * rs * hw[c];
            most[c / 128] = std::fmax(most[c / 128], std::fabs(wy[t * cols + c]));
        }
        for (int q = 0; q < 2; ++q) off_scale = std::fmax(off_scale, std::fabs(sc[2 * t + q] / (most[q] / 448) - 1));
        double sum = 0;
        for (size_t j = 0; j < choices; ++j) {
            int at = -1;
            for (size_t e = 0; e < experts; ++e)
                if ((j == 0 || (int)e != best[t * choices]) && (at < 0 || hl[t * experts + e] > hl[t * experts + at])) at = (int)e;
            best[t * choices + j] = at;
            ++count[at + 1];
            sum += ww[t * choices + j] = std::exp((double)hl[t * experts + at]);
        }
        for (size_t j = 0; j < choices; ++j) {
            ww[t * choices + j] /= sum;
            for (size_t o = 0; o < outputs; ++o) {
                double d = 0;
                for (size_t c = 0; c < cols; ++c) d += wy[t * cols + c] * hm[(best[t * choices + j] * outputs + o) * cols + c];
                wout[t * outputs + o] += ww[t * choices + j] * d;
            }
        }
    }
    for (size_t e = 0; e < experts; ++e) count[e + 1] += count[e];
    double wrong = 0;
    const auto got_ids = ids.host(), got_pos = positions.host(), got_off = offsets.host(), got_src = sources.host();
    std::vector<int> next(count.begin(), count.end() - 1);
    for (size_t p = 0; p < pairs; ++p) {
        wrong += got_ids[p] != best[p];
        wrong += got_pos[p] != next[best[p]]++;
        wrong += got_src[got_pos[p]] != (int)p;
    }
    for (size_t e = 0; e <= experts; ++e) wrong += got_off[e] != count[e];
    report("choices and places", wrong, 0);
    // values of at most 6 in 50 roundings; sums of 136 of them times 0.2 in 136 roundings more
    report("norm", worst(y.host(), wy), 50 * 6 * u);
    report("scales", off_scale, 50 * u);
    report("weights", worst(weights.host(), ww), 100 * u);
    report("combined products", worst(out.host(), wout), 136 * 6 * 0.2 * 250 * u);

    // backward: through the sum, the products, the copies and the norm
    Dev<float> dres(pairs * outputs), dw(pairs), drows(pairs * cols), dm(experts * outputs * cols), dy(tokens * cols), ds(tokens * cols);
    Dev<float> dlogits(tokens * experts), dnw(cols);
    order.CombineBackward<float>(list, {g.p, outputs}, {results.p, outputs}, positions.p, weights.p, {dres.p, outputs}, dw.p, pairs,
                                 tokens, choices, outputs);
    product.Backward<float, float>(list, {dres.p, outputs}, {rows.p, cols}, {matrices.p, cols, outputs * cols}, offsets.p,
                                   {drows.p, cols}, {dm.p, cols, outputs * cols}, pairs, experts, outputs, cols);
    order.DispatchBackward<float>(list, {drows.p, cols}, positions.p, nullptr, {dy.p, cols}, {}, nullptr, pairs, tokens, choices, cols);
    Dev<uint> norm_temp(bytes_to_uint_count(DeviceRMSNorm::GetBackwardTempStorageBytes<float>(tokens, cols)));
    norm.Backward<float, float>(list, {norm_temp.p, norm_temp.n}, {dy.p, cols}, {}, {s.p, cols}, w.p, rstd.p, {ds.p, cols}, dnw.p,
                                tokens, cols);
    report("status of the norm's gradient", norm.last_status(), 0);
    router.Backward<float>(list, {logits.p, experts}, ids.p, dw.p, {dlogits.p, experts}, how, tokens, experts, choices);
    if (hipStreamSynchronize(stream) != hipSuccess) return 1;
    std::vector<double> wdm(experts * outputs * cols, 0.0), wdw(pairs), wdy(tokens * cols, 0.0), wdl(tokens * experts, 0.0);
    for (size_t t = 0; t < tokens; ++t) {
        double mean = 0;
        for (size_t j = 0; j < choices; ++j) {
            const size_t p = t * choices + j, e = best[p];
            for (size_t o = 0; o < outputs; ++o) {
                const double gw = hg[t * outputs + o] * ww[p];
                double d = 0;
                for (size_t c = 0; c < cols; ++c) {
                    const double m = hm[(e * outputs + o) * cols + c];
                    d += wy[t * cols + c] * m;
                    wdm[(e * outputs + o) * cols + c] += gw * wy[t * cols + c];
                    wdy[t * cols + c] += gw * m;
                }
                wdw[p] += hg[t * outputs + o] * d;
            }
            mean += wdw[p] * ww[p];
        }
        for (size_t j = 0; j < choices; ++j) wdl[t * experts + best[t * choices + j]] = ww[t * choices + j] * (wdw[t * choices + j] - mean);
    }
    report("gradient of the matrices", worst(dm.host(), wdm), 45 * 6 * 200 * u);
    report("gradient of the weights", worst(dw.host(), wdw), 72 * 136 * 6 * 0.2 * 300 * u);
    report("gradient of the rows", worst(dy.host(), wdy), 2 * 72 * 0.2 * 200 * u);
    report("gradient of the logits", worst(dlogits.host(), wdl), 72 * 136 * 6 * 0.2 * 300 * u);
    if (hipStreamDestroy(stream) != hipSuccess) return 1;
    std::printf("%s: %d failure(s)\n", g_failed ? "FAILED" : "PASSED", g_failed);
    return g_failed != 0;
}
