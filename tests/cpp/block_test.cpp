// block_test.cpp — layer norm, dropout and the gated recurrence through the C++
// classes (include/lcpp/parallel_primitive.h) on a GPU, against their definitions
// in double on the host.  Prints one line per check and "PASSED: 0 failure(s)".
#include <hip/hip_runtime_api.h>

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
    const size_t rows = 37, cols = 203;
    const float eps = 1e-5f;
    const auto hx = values(rows * cols, 1, 4.0f, 0.5f), hw = values(cols, 2, 1.0f, 1.0f), hb = values(cols, 3, 1.0f, 0.0f);
    const auto hdy = values(rows * cols, 4, 2.0f, 0.0f);
    {
        DeviceLayerNorm norm;
        norm.create(device, &debug);
        Dev<float> x(hx), w(hw), b(hb), dy(hdy), y(rows * cols), dx(rows * cols), dw(cols), db(cols), mean(rows), rstd(rows);
        Dev<uint> temp(bytes_to_uint_count(DeviceLayerNorm::GetBackwardTempStorageBytes<float>(rows, cols)));
        norm.Forward<float, float>(list, {x.p, cols}, {y.p, cols}, w.p, b.p, eps, mean.p, rstd.p, rows, cols);
        norm.Backward<float, float>(list, {temp.p, temp.n}, {dy.p, cols}, {x.p, cols}, w.p, mean.p, rstd.p, {dx.p, cols}, dw.p,
                                    db.p, rows, cols);
        report("status of the layer norm", norm.last_status(), 0);
        std::vector<double> wy(rows * cols), wdx(rows * cols), wdw(cols, 0.0), wdb(cols, 0.0);
        for (size_t r = 0; r < rows; ++r) {
            double m = 0, v = 0, c1 = 0, c2 = 0;
            for (size_t c = 0; c < cols; ++c) m += hx[r * cols + c];
            m /= cols;
            for (size_t c = 0; c < cols; ++c) v += (hx[r * cols + c] - m) * (hx[r * cols + c] - m);
            const double rs = 1 / std::sqrt(v / cols + eps);
            for (size_t c = 0; c < cols; ++c) {
                const double u = (hx[r * cols + c] - m) * rs, g = hdy[r * cols + c];
                wy[r * cols + c] = u * hw[c] + hb[c];
                c1 += g * hw[c], c2 += g * hw[c] * u;
                wdw[c] += g * u, wdb[c] += g;
            }
            for (size_t c = 0; c < cols; ++c) {
                const double u = (hx[r * cols + c] - m) * rs;
                wdx[r * cols + c] = rs * (hdy[r * cols + c] * hw[c] - c1 / cols - u * c2 / cols);
            }
        }
        // values of at most 5 and sums of 203 and 37 of them, in under 100 roundings of 2^-24
        report("layer norm", worst(y.host(), wy), 100 * 5 / 16777216.0);
        report("layer norm dx", worst(dx.host(), wdx), 100 * 5 / 16777216.0);
        report("layer norm dweight", worst(dw.host(), wdw), 100 * 37 * 3 / 16777216.0);
        report("layer norm dbias", worst(db.host(), wdb), 100 * 37 / 16777216.0);
    }
    {
        DeviceDropout drop;
        DeviceLayerNorm norm;
        drop.create(device, &debug);
        norm.create(device, &debug);
        Dev<float> x(hx), r(hdy), y(rows * cols), s(rows * cols), n(rows * cols), back(rows * cols);
        const DropoutState state{0.25, 77, 5, nullptr};
        drop.Forward<float>(list, {x.p, cols}, {y.p, cols}, state, rows, cols, {r.p, cols});
        norm.AddForward<float, float>(list, {x.p, cols}, {r.p, cols}, state, {s.p, cols}, {n.p, cols}, nullptr, nullptr, eps,
                                      nullptr, nullptr, rows, cols);
        drop.Backward<float>(list, {x.p, cols}, {back.p, cols}, state, rows, cols);
        const auto a = y.host(), c = s.host(), g = back.host();
        double off = 0, share = 0;
        for (size_t i = 0; i < a.size(); ++i) {
            off = std::fmax(off, std::fabs(a[i] - c[i]));
            share += g[i] != 0;
            off = std::fmax(off, std::fabs(a[i] - (g[i] + hdy[i])));
        }
        report("dropout alone, in the layer norm and backward", off, 0);
        const double n_all = (double)a.size();
        report("dropout's share", std::fabs(share / n_all - 0.75), 6 * std::sqrt(0.75 * 0.25 / n_all));
    }
    {
        DeviceGatedRecurrence mix;
        mix.create(device, &debug);
        const size_t n = 2, t = 300, c = 70;
        const auto hg = values(n * t * c, 5, 6.0f, 1.5f), hv = values(n * t * c, 6, 2.0f, 0.0f), hd = values(n * t * c, 7, 2.0f, 0.0f);
        Dev<float> g(hg), v(hv), dy(hd), y(n * t * c), dg(n * t * c), dv(n * t * c), last(n * c), first(n * c);
        Dev<float> saved(n * DeviceGatedRecurrence::GetCheckpointRows(t) * c);
        Dev<uint> temp(bytes_to_uint_count(DeviceGatedRecurrence::GetTempStorageBytes(n, t, c)));
        const Sequences seq{n, t, c};
        const RowsView<float> vg{g.p, c, t * c}, vv{v.p, c, t * c}, vy{y.p, c, t * c}, vd{dy.p, c, t * c};
        mix.Forward<float>(list, {temp.p, temp.n}, LCPP_GATE_SIGMOID, vg, vv, vy, nullptr, last.p, saved.p, seq);
        mix.Backward<float>(list, {temp.p, temp.n}, LCPP_GATE_SIGMOID, vg, vv, saved.p, vd, {dg.p, c, t * c}, {dv.p, c, t * c},
                            nullptr, first.p, seq);
        report("status of the recurrence", mix.last_status(), 0);
        std::vector<double> wy(n * t * c), wg(n * t * c), wv(n * t * c);
        for (size_t s = 0; s < n; ++s)
            for (size_t k = 0; k < c; ++k) {
                double h = 0, e = 0;
                for (size_t i = 0; i < t; ++i) {
                    const size_t at = (s * t + i) * c + k;
                    const double a = 1 / (1 + std::exp(-(double)hg[at]));
                    wy[at] = h = a * h + (1 - a) * hv[at];
                }
                for (size_t i = t; i-- > 0;) {
                    const size_t at = (s * t + i) * c + k;
                    const double a = 1 / (1 + std::exp(-(double)hg[at])), before = i ? wy[at - c] : 0.0, d = hd[at] + e;
                    wg[at] = d * (before - hv[at]) * a * (1 - a);
                    wv[at] = d * (1 - a);
                    e = a * d;
                }
            }
        // values of at most 1 with a memory of at most 90 steps of 20 roundings each, gradients of sums of 90
        report("recurrence", worst(y.host(), wy), 90 * 20 / 16777216.0);
        report("recurrence dgate", worst(dg.host(), wg), 90 * 90 * 20 / 16777216.0);
        report("recurrence dinput", worst(dv.host(), wv), 90 * 90 * 20 / 16777216.0);
        Dev<float> pool(n * c), out(n * c);
        if (hipMemcpy(pool.p, last.p, n * c * 4, hipMemcpyDeviceToDevice) != hipSuccess) return 1;
        mix.Step<float>(list, LCPP_GATE_SIGMOID, {g.p, t * c}, {v.p, t * c}, pool.p, pool.p, nullptr, n, {out.p, c}, n, c);
        std::vector<double> ws(n * c);
        for (size_t s = 0; s < n; ++s)
            for (size_t k = 0; k < c; ++k) {
                const double a = 1 / (1 + std::exp(-(double)hg[s * t * c + k]));
                ws[s * c + k] = a * wy[(s * t + t - 1) * c + k] + (1 - a) * hv[s * t * c + k];
            }
        if (hipStreamSynchronize(stream) != hipSuccess) return 1;
        report("recurrence step", worst(out.host(), ws), 91 * 20 / 16777216.0);
    }
    if (hipStreamDestroy(stream) != hipSuccess) return 1;
    std::printf("%s: %d failure(s)\n", g_failed ? "FAILED" : "PASSED", g_failed);
    return g_failed != 0;
}
