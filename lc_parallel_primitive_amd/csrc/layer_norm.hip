// layer_norm.hip — layer norm over rows, forward and backward, alone or with
// the residual sum and dropout before it.
//
//   s = x, or s = residual + dropout(x), stored in the rows' type
//   mean = sum(s) / n,  rstd = 1 / sqrt(sum((s - mean)^2) / n + eps)
//   y = (s - mean) rstd w + b
//
// With u = (s - mean) rstd and v = dy w, the gradients are
//   ds = rstd (v - sum(v) / n - u sum(v u) / n)   [+ the gradient that reaches s elsewhere]
//   dw = sum over rows of dy u,  db = sum over rows of dy
//   dresidual = ds,  dx = dropout(ds) with the forward pass's random bits
//
// What bounds it is memory: a row is read once, into registers, and its sums, the
// outputs and the columns' sums are made from there, with no more than ten or so
// operations an element.  So a row belongs to as few threads as hold it (16 lanes
// to 1024 threads), a workgroup keeps several short rows, takes one set of rows
// after the other and has the next ones on their way meanwhile.  dw and db are
// sums in the same registers, one partial sum per workgroup, and a second launch
// adds these in a fixed order: no atomics, the same result at every call.
//
// Measured (us by kernel traces and what that makes of the bytes read and written once;
// TB/s): 16384 x 4096 bfloat16 forward 51 (5.3), backward 68 (6.0), the partial sums 5;
// 16384 x 2048 with the sum and dropout, forward 45 (5.9), backward 60 (5.6), the partial
// sums 5.  A copy of 512 MiB runs at 5.3; what the pass before has left in the
// last-level cache makes up the rest.  16 x 1024 forward 3: a launch.
#include <algorithm>

#include "tensor.hpp"

namespace lcpp {
namespace {

// A barrier for what waves exchange in LDS.  __syncthreads() would also wait for
// the global loads in flight, which here are those of the next rows.
__device__ __forceinline__ void group_barrier()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// A row's columns: eight at a time (an octet) in the lanes of its group of
// threads, K octets a thread, and the last `rem` < 8 columns one to a thread, so
// that no octet is partly valid.
template <int NT, int K>
struct Columns {
    uint32_t t, full, rem, cols;
    __device__ __forceinline__ Columns(uint32_t n) : t(threadIdx.x % NT), full(n & ~7u), rem(n & 7u), cols(n) {}
    __device__ __forceinline__ uint32_t col(int k) const { return (t + k * NT) * kOctet; }
    __device__ __forceinline__ bool has(int k) const { return col(k) < full; }
    __device__ __forceinline__ bool has_tail() const { return t < rem; }
    __device__ __forceinline__ uint32_t tail() const { return full + t; }
};

// A thread's part of a row as it lies in memory.
template <class T, int K>
struct RowPart {
    Octet<T> o[K];
    T tail;
    template <int NT>
    __device__ __forceinline__ void load(const T *row, const Columns<NT, K> &c)
    {
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (c.has(k)) o[k] = load_pack<kOctet>(row + c.col(k));
        if (c.has_tail()) tail = row[c.tail()];
    }
    // a vector of weights, or one value everywhere
    template <int NT>
    __device__ __forceinline__ void load_or(const T *p, const Columns<NT, K> &c, float value)
    {
        tail = (T)value;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < kOctet; ++i) o[k].v[i] = (T)value;
        if (p) load(p, c);
    }
};

// Sum over a row's threads within a wave: all 64 lanes, or the 16 or 32 of a
// narrow row, whose wave works on several rows.
template <int NT>
__device__ __forceinline__ float lanes_sum(float x)
{
    if constexpr (NT >= kWave) {
        return wave_reduce_dpp(x, SumOp());
    } else {
        static_assert(NT == 16 || NT == 32, "rows of a wave");
        x += dpp_perm<kDppQuadXor1>(x);
        x += dpp_perm<kDppQuadXor2>(x);
        x += dpp_perm<kDppRowHalfMirror>(x);
        x += dpp_perm<kDppRowMirror>(x);
        if constexpr (NT == 32) x += shfl_xor(x, 16);
        return x;
    }
}

// Sums of V values over the NT threads of a row's group; every thread of the
// group gets them.  A group of several waves meets in LDS, all groups of the
// workgroup at the same barrier; `slot` alternates from row to row, so one
// barrier a row is enough.
template <int NT, int WAVES, int V>
__device__ __forceinline__ void group_sum(float (&x)[V], float (*lds)[WAVES][2], int slot)
{
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = lanes_sum<NT>(x[v]);
    if constexpr (NT > kWave) {
        constexpr int GW = NT / kWave;
        const uint32_t wave = threadIdx.x / kWave;
        if (lane_id() == 0) {
#pragma unroll
            for (int v = 0; v < V; ++v) lds[slot][wave][v] = x[v];
        }
        group_barrier();
        const uint32_t first = wave / GW * GW;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < GW; ++w) s += lds[slot][first + w][v];
            x[v] = s;
        }
    }
}

// A product as it is rounded, fused with no later sum: every difference from a mean
// has to be from the same mean.
__device__ __forceinline__ float rounded(float x)
{
    asm("" : "+v"(x));
    return x;
}
// x, or 0 in the place of infinities and NaN.
__device__ __forceinline__ float finite_or_0(float x)
{
    return fabsf(x) <= std::numeric_limits<float>::max() ? x : 0.0f;
}
// An infinite mean has no rest, and the difference of squares is not below 0 (a NaN
// stays one).
__device__ __forceinline__ void norm_rest(float &rest, float &sq)
{
    rest = finite_or_0(rest);
    sq = sq < 0.0f ? 0.0f : sq;
}

// Mean and mean square deviation of a row.  The mean of a first sum is off by some
// roundings of its size, which is much where a row lies far from 0 and varies
// little, so the second pass sums the differences from it as well as their squares:
// the mean is `mean` + `rest`, known to roundings of the differences alone, and the
// squares around it are those around `mean` less n rest^2.  A wave does this for
// its columns; the waves' values meet in LDS at one barrier, one wave's in each of
// 16 lanes, and combine as distances from the first wave's mean.  (16384 x 4096 bfloat16
// 52.6 us, with the first sum alone and each thread adding up the waves 53.0.)
// `count`, `lane_count`: columns of the wave, and of the wave whose values the lane
// combines (0: none); `each` gives f(x) for each of the thread's columns.
template <int NT, int WAVES, class F>
__device__ __forceinline__ void group_moments(F each, float count, float lane_count, float (*lds)[WAVES][3], int slot,
                                              float cols, float inv_cols, float &mean, float &rest, float &var)
{
    float sum = 0.0f;
    each([&](float x) { sum += x; });
    const float inv = count > 0.0f ? 1.0f / count : 0.0f;
    mean = rounded(lanes_sum<NT>(sum) * inv);
    float off = 0.0f, sq = 0.0f;
    each([&](float x) {
        const float d = x - mean;
        off += d;
        sq += d * d;
    });
    rest = lanes_sum<NT>(off) * inv;
    sq = lanes_sum<NT>(sq) - count * (rest * rest);
    norm_rest(rest, sq);
    if constexpr (NT > kWave) {
        constexpr uint32_t GW = NT / kWave;
        const uint32_t wave = threadIdx.x / kWave, from = lane_id() % 16;
        if (lane_id() == 0) lds[slot][wave][0] = mean, lds[slot][wave][1] = rest, lds[slot][wave][2] = sq;
        group_barrier();
        const bool has = from < GW;
        const float(*w)[3] = &lds[slot][wave / GW * GW];
        // (the first lane's sum for all: a product that is fused with a sum's first addition
        // is rounded differently in two lanes, and `rest` has to belong to `mean`)
        auto waves_sum = [](float x) { return read_lane(lanes_sum<16>(x), 0); };
        const float base = finite_or_0(w[0][0]);
        const float d = has ? (w[has ? from : 0][0] - base) + w[has ? from : 0][1] : 0.0f;
        const float nd = lane_count * d;
        const float shift = rounded(waves_sum(nd) * inv_cols);
        sq = waves_sum((has ? w[has ? from : 0][2] : 0.0f) + nd * d) - cols * (shift * shift);
        mean = base + shift;
        rest = (base - mean) + shift;
        norm_rest(rest, sq);
    }
    var = sq * inv_cols;
}

// One octet of a vector of weights, or one value everywhere.
template <class W>
__device__ __forceinline__ Octet<W> octet_or(const void *p, uint32_t col, float value)
{
    if (p) return load_pack<kOctet>(static_cast<const W *>(p) + col);
    Octet<W> o;
#pragma unroll
    for (int i = 0; i < kOctet; ++i) o.v[i] = (W)value;
    return o;
}

struct NormArgs {
    const void *in, *residual, *weight, *bias;
    void *sum, *out;
    uint64_t in_stride, residual_stride, sum_stride, out_stride;
    float *mean, *rstd;
    uint32_t rows, cols;
    float eps;
    DropArgs drop;
};

// One element's dropout, for the last columns of a row.
__device__ __forceinline__ float drop_one(float x, uint32_t row, uint32_t col, uint64_t offset, const DropArgs &d)
{
    float v[kOctet] = {x, x, x, x, x, x, x, x};
    drop_octet(v, row, col / kOctet, offset, d);
    float r = v[0];
#pragma unroll
    for (int i = 1; i < kOctet; ++i) r = (int)(col % kOctet) == i ? v[i] : r;
    return r;
}

// Rows that the registers of NT threads hold, K octets each; THREADS / NT rows at
// a time, each workgroup several one after the other, the next ones on their way
// while these are worked on, and the weights in registers too (AHEAD: where the
// registers hold that).
template <class T, class W, int NT, int K, int THREADS, bool ADD, bool AHEAD>
__global__ __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(AHEAD ? 1 : ADD && sizeof(T) == 4 ? 2 : 4))) void norm_forward_kernel(NormArgs a)
{
    constexpr int WAVES = THREADS / kWave, RG = THREADS / NT;
    constexpr uint32_t GW = NT > kWave ? NT / kWave : 1;
    constexpr uint32_t kLaneCols = (NT < kWave ? NT : kWave) * kOctet;
    __shared__ float lds[2][WAVES][3];
    const Columns<NT, K> c(a.cols);
    const uint32_t group = threadIdx.x / NT;
    const uint64_t offset = ADD ? drop_offset(a.drop) : 0;
    // columns of a wave of the group
    auto wave_cols = [&](uint32_t w) {
        uint32_t n = w == 0 ? c.rem : 0;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const uint32_t from = (w * kWave + k * NT) * kOctet;
            n += from < c.full ? (c.full - from < kLaneCols ? c.full - from : kLaneCols) : 0;
        }
        return (float)n;
    };
    const float inv_cols = 1.0f / (float)a.cols;
    const float count = wave_cols(threadIdx.x / kWave % GW);
    const float lane_count = lane_id() % 16 < GW ? wave_cols(lane_id() % 16) : 0.0f;

    RowPart<W, K> w, b;
    if constexpr (AHEAD) {
        w.load_or(static_cast<const W *>(a.weight), c, 1.0f);
        b.load_or(static_cast<const W *>(a.bias), c, 0.0f);
    }
    const T *in = static_cast<const T *>(a.in), *residual = static_cast<const T *>(a.residual);
    RowPart<T, K> next, next_r;
    auto load = [&](uint64_t row) {
        if (row >= a.rows) return;
        next.load(in + row * a.in_stride, c);
        if constexpr (ADD && AHEAD) next_r.load(residual + row * a.residual_stride, c);
    };
    uint64_t row = (uint64_t)blockIdx.x * RG + group;
    if constexpr (AHEAD) load(row);
    // (the workgroup's groups make the same number of rounds: they share barriers)
    const uint64_t stride = (uint64_t)gridDim.x * RG;
    int slot = 0;
    for (uint64_t base = (uint64_t)blockIdx.x * RG; base < a.rows; base += stride, row += stride, slot ^= 1) {
        if constexpr (!AHEAD) load(row);
        RowPart<T, K> x = next, r = next_r;
        const bool live = row < a.rows;
        if constexpr (AHEAD) load(row + stride);
        if constexpr (ADD) {
            // s in the place of x, rounded as it is stored
            if (live) {
                T *sum = static_cast<T *>(a.sum) + row * a.sum_stride;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (!c.has(k)) continue;
                    float v[kOctet];
                    if constexpr (!AHEAD) r.o[k] = load_pack<kOctet>(residual + row * a.residual_stride + c.col(k));
#pragma unroll
                    for (int i = 0; i < kOctet; ++i) v[i] = x.o[k][i];
                    if (a.drop.cut) drop_octet(v, (uint32_t)row, c.col(k) / kOctet, offset, a.drop);
#pragma unroll
                    for (int i = 0; i < kOctet; ++i) {
                        v[i] += r.o[k][i];
                        x.o[k].v[i] = (T)v[i];
                    }
                    store_pack<kOctet>(sum + c.col(k), v);
                }
                if (c.has_tail()) {
                    float v = (float)x.tail;
                    if constexpr (!AHEAD) r.tail = residual[row * a.residual_stride + c.tail()];
                    if (a.drop.cut) v = drop_one(v, (uint32_t)row, c.tail(), offset, a.drop);
                    x.tail = (T)(v + (float)r.tail);
                    sum[c.tail()] = x.tail;
                }
            }
        }
        float mean, rest, var;
        group_moments<NT, WAVES>(
            [&](auto f) {
                if (!live) return;
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (c.has(k))
#pragma unroll
                        for (int i = 0; i < kOctet; ++i) f(x.o[k][i]);
                if (c.has_tail()) f((float)x.tail);
            },
            count, lane_count, lds, slot, (float)a.cols, inv_cols, mean, rest, var);
        const float rstd = 1.0f / sqrtf(var + a.eps), shift = rest * rstd;
        if (!live) continue;
        T *out = static_cast<T *>(a.out) + row * a.out_stride;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (!c.has(k)) continue;
            if constexpr (!AHEAD) {
                w.o[k] = octet_or<W>(a.weight, c.col(k), 1.0f);
                b.o[k] = octet_or<W>(a.bias, c.col(k), 0.0f);
            }
            float y[kOctet];
#pragma unroll
            for (int i = 0; i < kOctet; ++i) y[i] = ((x.o[k][i] - mean) * rstd - shift) * w.o[k][i] + b.o[k][i];
            store_pack_nt<kOctet>(out + c.col(k), y);
        }
        if constexpr (!AHEAD) {
            if (c.has_tail()) {
                w.tail = a.weight ? static_cast<const W *>(a.weight)[c.tail()] : (W)1.0f;
                b.tail = a.bias ? static_cast<const W *>(a.bias)[c.tail()] : (W)0.0f;
            }
        }
        if (c.has_tail()) out[c.tail()] = (T)((((float)x.tail - mean) * rstd - shift) * (float)w.tail + (float)b.tail);
        if (c.t == 0) {
            if (a.mean) a.mean[row] = mean + rest;
            if (a.rstd) a.rstd[row] = rstd;
        }
    }
}

// ---- longer rows
constexpr int kLongThreads = 1024;
constexpr int kLongWaves = kLongThreads / kWave;

// s of one octet: the input, or residual + dropout(input) rounded to the rows'
// type, which is also stored.
template <class T, bool ADD>
__device__ __forceinline__ Octet<T> norm_input(const NormArgs &a, uint64_t offset, uint64_t row, uint32_t col)
{
    Octet<T> x = load_octet(static_cast<const T *>(a.in) + row * a.in_stride, col, a.cols);
    if constexpr (ADD) {
        const Octet<T> r = load_octet(static_cast<const T *>(a.residual) + row * a.residual_stride, col, a.cols);
        float v[kOctet];
#pragma unroll
        for (int i = 0; i < kOctet; ++i) v[i] = x[i];
        if (a.drop.cut) drop_octet(v, (uint32_t)row, col / kOctet, offset, a.drop);
#pragma unroll
        for (int i = 0; i < kOctet; ++i) {
            v[i] += r[i];
            x.v[i] = (T)v[i];
        }
        store_octet(static_cast<T *>(a.sum) + row * a.sum_stride, col, a.cols, v);
    }
    return x;
}
template <class W>
__device__ __forceinline__ void norm_weight(const void *weight, uint32_t col, uint32_t cols, float value, float (&w)[kOctet])
{
    if (weight) {
        const Octet<W> o = load_octet(static_cast<const W *>(weight), col, cols);
#pragma unroll
        for (int i = 0; i < kOctet; ++i) w[i] = o[i];
    } else {
#pragma unroll
        for (int i = 0; i < kOctet; ++i) w[i] = value;
    }
}

// A workgroup reads its row three times (from the caches).
template <class T, class W, bool ADD>
__global__ __launch_bounds__(kLongThreads) void norm_forward_long_kernel(NormArgs a)
{
    __shared__ float lds[2][kLongWaves][2];
    const uint64_t offset = ADD ? drop_offset(a.drop) : 0;
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *s = ADD ? static_cast<const T *>(a.sum) + row * a.sum_stride
                         : static_cast<const T *>(a.in) + row * a.in_stride;
        float sum[1] = {0.0f};
        for (uint32_t col = threadIdx.x * kOctet; col < a.cols; col += kLongThreads * kOctet) {
            const Octet<T> x = norm_input<T, ADD>(a, offset, row, col);
#pragma unroll
            for (int i = 0; i < kOctet; ++i) sum[0] += x[i];
        }
        group_sum<kLongThreads, kLongWaves>(sum, lds, 0);
        const float mean = sum[0] / (float)a.cols;
        float off[2] = {0.0f, 0.0f};  // sums of the differences and of their squares, as in group_moments
        // (each thread reads back the sums that it stored itself)
        for (uint32_t col = threadIdx.x * kOctet; col < a.cols; col += kLongThreads * kOctet) {
            const Octet<T> x = load_octet(s, col, a.cols);
#pragma unroll
            for (int i = 0; i < kOctet; ++i) {
                const float d = x[i] - mean;
                if (col + i < a.cols) off[0] += d, off[1] += d * d;
            }
        }
        group_sum<kLongThreads, kLongWaves>(off, lds, 1);
        float rest = off[0] / (float)a.cols, sq = off[1] - off[0] * rest;
        norm_rest(rest, sq);
        const float rstd = 1.0f / sqrtf(sq / (float)a.cols + a.eps), shift = rest * rstd;
        for (uint32_t col = threadIdx.x * kOctet; col < a.cols; col += kLongThreads * kOctet) {
            const Octet<T> x = load_octet(s, col, a.cols);
            float w[kOctet], b[kOctet];
            norm_weight<W>(a.weight, col, a.cols, 1.0f, w);
            norm_weight<W>(a.bias, col, a.cols, 0.0f, b);
#pragma unroll
            for (int i = 0; i < kOctet; ++i) w[i] = ((x[i] - mean) * rstd - shift) * w[i] + b[i];
            store_octet(static_cast<T *>(a.out) + row * a.out_stride, col, a.cols, w);
        }
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[row] = mean + rest;
            if (a.rstd) a.rstd[row] = rstd;
        }
    }
}

// ---------------------------------------------------------------- backward
struct NormGradArgs {
    const void *grad_out, *grad_sum, *in, *weight;
    void *grad_in, *grad_branch;  // ds, and dx where it is not ds
    uint64_t go_stride, gs_stride, in_stride, gi_stride, gb_stride;
    const float *mean, *rstd;
    float *partial;    // [workgroup][dw, db][cols]; null: neither is wanted
    uint32_t *status;  // the temp storage's status word, cleared here (may be null)
    uint32_t rows, cols;
    DropArgs drop;
};

// THREADS / NT rows at a time; a thread keeps the same columns for all of its
// workgroup's rows, so dw and db are sums in its registers, one partial sum per
// workgroup at the end.  The next rows are on their way while these are worked on.
template <class T, class W, int NT, int K, int THREADS, bool ADD, bool AHEAD, bool ACC>
__global__ __launch_bounds__(THREADS) void norm_backward_kernel(NormGradArgs a)
{
    constexpr int WAVES = THREADS / kWave, RG = THREADS / NT;
    __shared__ float lds[2][WAVES][2];
    // (a wave with several rows adds their sums up first)
    constexpr int FOLD = NT < kWave ? WAVES : RG;
    __shared__ float fold[FOLD > 1 ? NT * K * kOctet : 1], fold_tail[FOLD > 1 ? kOctet : 1];
    const Columns<NT, K> c(a.cols);
    const uint32_t group = threadIdx.x / NT;
    const uint64_t offset = ADD ? drop_offset(a.drop) : 0;
    const float inv = 1.0f / (float)a.cols;
    float dw[K][kOctet] = {}, db[K][kOctet] = {}, dw_tail = 0.0f, db_tail = 0.0f;
    if (a.status && blockIdx.x == 0 && threadIdx.x == 0) *a.status = 0;
    RowPart<W, K> w;
    if constexpr (AHEAD) w.load_or(static_cast<const W *>(a.weight), c, 1.0f);
    const T *grad_out = static_cast<const T *>(a.grad_out), *in = static_cast<const T *>(a.in);
    const T *grad_sum = static_cast<const T *>(a.grad_sum);
    RowPart<T, K> next_dy, next_s, next_g;
    float next_mean = 0.0f, next_rstd = 0.0f;
    auto load = [&](uint64_t row) {
        if (row >= a.rows) return;
        next_dy.load(grad_out + row * a.go_stride, c);
        next_s.load(in + row * a.in_stride, c);
        if constexpr (ADD && AHEAD) {
            if (grad_sum) next_g.load(grad_sum + row * a.gs_stride, c);
        }
        next_mean = a.mean[row];
        next_rstd = a.rstd[row];
    };
    uint64_t row = (uint64_t)blockIdx.x * RG + group;
    if constexpr (AHEAD) load(row);
    // (the workgroup's groups make the same number of rounds: they share barriers)
    const uint64_t stride = (uint64_t)gridDim.x * RG;
    int slot = 0;
    for (uint64_t base = (uint64_t)blockIdx.x * RG; base < a.rows; base += stride, row += stride, slot ^= 1) {
        if constexpr (!AHEAD) load(row);
        RowPart<T, K> dy = next_dy, s = next_s, g = next_g;
        const float mean = next_mean, rstd = next_rstd;
        const bool live = row < a.rows;
        if constexpr (AHEAD) load(row + stride);
        float sums[2] = {0.0f, 0.0f};
        if (live) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (!c.has(k)) continue;
                if constexpr (!AHEAD) w.o[k] = octet_or<W>(a.weight, c.col(k), 1.0f);
#pragma unroll
                for (int i = 0; i < kOctet; ++i) {
                    const float u = (s.o[k][i] - mean) * rstd, v = dy.o[k][i] * w.o[k][i];
                    sums[0] += v;
                    sums[1] += v * u;
                    if constexpr (ACC) {
                        dw[k][i] += dy.o[k][i] * u;
                        db[k][i] += dy.o[k][i];
                    }
                }
            }
            if (c.has_tail()) {
                if constexpr (!AHEAD) w.tail = a.weight ? static_cast<const W *>(a.weight)[c.tail()] : (W)1.0f;
                const float u = ((float)s.tail - mean) * rstd, v = (float)dy.tail * (float)w.tail;
                sums[0] += v;
                sums[1] += v * u;
                dw_tail += (float)dy.tail * u;
                db_tail += (float)dy.tail;
            }
        }
        group_sum<NT, WAVES>(sums, lds, slot);
        if (!live) continue;
        const float mean_v = sums[0] * inv, mean_vu = sums[1] * inv;
        T *gi = static_cast<T *>(a.grad_in) + row * a.gi_stride, *gb = static_cast<T *>(a.grad_branch) + row * a.gb_stride;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (!c.has(k)) continue;
            float d[kOctet];
            if constexpr (!AHEAD) {
                w.o[k] = octet_or<W>(a.weight, c.col(k), 1.0f);
                if constexpr (ADD) {
                    if (grad_sum) g.o[k] = load_pack<kOctet>(grad_sum + row * a.gs_stride + c.col(k));
                }
            }
#pragma unroll
            for (int i = 0; i < kOctet; ++i) {
                const float u = (s.o[k][i] - mean) * rstd, v = dy.o[k][i] * w.o[k][i];
                d[i] = rstd * (v - mean_v - u * mean_vu);
            }
            if constexpr (ADD) {
                if (grad_sum) {
#pragma unroll
                    for (int i = 0; i < kOctet; ++i) d[i] += g.o[k][i];
                }
            }
            if (a.grad_in) store_pack_nt<kOctet>(gi + c.col(k), d);
            if constexpr (ADD) {
                if (a.grad_branch) {
                    if (a.drop.cut) drop_octet(d, (uint32_t)row, c.col(k) / kOctet, offset, a.drop);
                    store_pack_nt<kOctet>(gb + c.col(k), d);
                }
            }
        }
        if (c.has_tail()) {
            const float u = ((float)s.tail - mean) * rstd, v = (float)dy.tail * (float)w.tail;
            float d = rstd * (v - mean_v - u * mean_vu);
            if constexpr (ADD) {
                if constexpr (!AHEAD) {
                    if (grad_sum) g.tail = grad_sum[row * a.gs_stride + c.tail()];
                }
                if (grad_sum) d += (float)g.tail;
            }
            if (a.grad_in) gi[c.tail()] = (T)d;
            if constexpr (ADD) {
                if (a.grad_branch) {
                    if (a.drop.cut) d = drop_one(d, (uint32_t)row, c.tail(), offset, a.drop);
                    gb[c.tail()] = (T)d;
                }
            }
        }
    }
    if (!ACC || !a.partial) return;
    float *part = a.partial + (uint64_t)blockIdx.x * 2 * a.cols;
#pragma unroll
    for (int half = 0; half < 2; ++half, part += a.cols) {
        float(&x)[K][kOctet] = half ? db : dw;
        float &tail = half ? db_tail : dw_tail;
        uint32_t turn = group;
        bool writes = group == RG - 1;
        if constexpr (NT < kWave) {
#pragma unroll
            for (int step = NT; step < kWave; step *= 2) {
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < kOctet; ++i) x[k][i] += shfl_xor(x[k][i], step);
                tail += shfl_xor(tail, step);
            }
            const bool first = lane_id() < NT;
            turn = first ? threadIdx.x / kWave : WAVES;
            writes = first && turn == WAVES - 1;
        }
        if constexpr (FOLD > 1) {
            // the groups add to the columns' sums one after the other, in a fixed order
            for (uint32_t g = 0; g < FOLD; ++g) {
                if (turn == g) {
#pragma unroll
                    for (int k = 0; k < K; ++k)
#pragma unroll
                        for (int i = 0; i < kOctet; ++i) {
                            float &f = fold[(i * K + k) * NT + c.t];
                            f = g ? f + x[k][i] : x[k][i];
                            x[k][i] = f;
                        }
                    if (c.has_tail()) {
                        float &f = fold_tail[c.t];
                        f = g ? f + tail : tail;
                        tail = f;
                    }
                }
                __syncthreads();
            }
        }
        if (writes) {
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (c.has(k)) store_pack<kOctet>(part + c.col(k), x[k]);
            if (c.has_tail()) part[c.tail()] = tail;
        }
    }
}

// Longer rows, ds: a workgroup reads its row twice (the second time from the caches).
template <class T, class W, bool ADD>
__global__ __launch_bounds__(kLongThreads) void norm_backward_long_kernel(NormGradArgs a)
{
    __shared__ float lds[2][kLongWaves][2];
    const uint64_t offset = ADD ? drop_offset(a.drop) : 0;
    const float inv = 1.0f / (float)a.cols;
    if (a.status && blockIdx.x == 0 && threadIdx.x == 0) *a.status = 0;
    int slot = 0;
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x, slot ^= 1) {
        const float mean = a.mean[row], rstd = a.rstd[row];
        const T *dy = static_cast<const T *>(a.grad_out) + row * a.go_stride;
        const T *s = static_cast<const T *>(a.in) + row * a.in_stride;
        float sums[2] = {0.0f, 0.0f};
        // v and u of an octet (past the row's end dy and so v are 0)
        auto terms = [&](uint32_t col, float(&v)[kOctet], float(&u)[kOctet]) {
            const Octet<T> d = load_octet(dy, col, a.cols), x = load_octet(s, col, a.cols);
            float w[kOctet];
            norm_weight<W>(a.weight, col, a.cols, 1.0f, w);
#pragma unroll
            for (int i = 0; i < kOctet; ++i) {
                u[i] = (x[i] - mean) * rstd;
                v[i] = d[i] * w[i];
            }
        };
        for (uint32_t col = threadIdx.x * kOctet; col < a.cols; col += kLongThreads * kOctet) {
            float v[kOctet], u[kOctet];
            terms(col, v, u);
#pragma unroll
            for (int i = 0; i < kOctet; ++i) {
                sums[0] += v[i];
                sums[1] += v[i] * u[i];
            }
        }
        group_sum<kLongThreads, kLongWaves>(sums, lds, slot);
        for (uint32_t col = threadIdx.x * kOctet; col < a.cols; col += kLongThreads * kOctet) {
            float v[kOctet], u[kOctet], d[kOctet];
            terms(col, v, u);
#pragma unroll
            for (int i = 0; i < kOctet; ++i) d[i] = rstd * (v[i] - sums[0] * inv - u[i] * (sums[1] * inv));
            if constexpr (ADD) {
                if (a.grad_sum) {
                    const Octet<T> g = load_octet(static_cast<const T *>(a.grad_sum) + row * a.gs_stride, col, a.cols);
#pragma unroll
                    for (int i = 0; i < kOctet; ++i) d[i] += g[i];
                }
            }
            if (a.grad_in) store_octet(static_cast<T *>(a.grad_in) + row * a.gi_stride, col, a.cols, d);
            if constexpr (ADD) {
                if (a.grad_branch) {
                    if (a.drop.cut) drop_octet(d, (uint32_t)row, col / kOctet, offset, a.drop);
                    store_octet(static_cast<T *>(a.grad_branch) + row * a.gb_stride, col, a.cols, d);
                }
            }
        }
    }
}
// Longer rows, dw and db: a workgroup takes 2048 columns of every gridDim.y-th
// row.
constexpr int kColThreads = 256;
constexpr uint32_t kColGroups = 1024;  // workgroups that these partial sums are split over
template <class T>
__global__ __launch_bounds__(kColThreads) void norm_backward_cols_kernel(NormGradArgs a)
{
    const uint32_t col = (blockIdx.x * kColThreads + threadIdx.x) * kOctet;
    if (col >= a.cols) return;
    float dw[kOctet] = {}, db[kOctet] = {};
    for (uint64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const Octet<T> dy = load_octet(static_cast<const T *>(a.grad_out) + row * a.go_stride, col, a.cols);
        const Octet<T> s = load_octet(static_cast<const T *>(a.in) + row * a.in_stride, col, a.cols);
        const float mean = a.mean[row], rstd = a.rstd[row];
#pragma unroll
        for (int i = 0; i < kOctet; ++i) {
            dw[i] += dy[i] * ((s[i] - mean) * rstd);
            db[i] += dy[i];
        }
    }
    float *part = a.partial + (uint64_t)blockIdx.y * 2 * a.cols;
    store_octet(part, col, a.cols, dw);
    store_octet(part + a.cols, col, a.cols, db);
}

// dw and db from the partial sums: 64 columns per workgroup at a time, each wave
// every 16th partial sum, always in the same order.  Bound by the latency of one
// round of loads: 4 us for 256 sums of 2 x 5001 columns, 3.9 TB/s of last-level cache.
constexpr int kFoldWaves = 16;
template <class W>
__global__ __launch_bounds__(kFoldWaves *kWave) void norm_fold_kernel(const float *partial, uint32_t parts, uint32_t cols,
                                                                      W *grad_weight, W *grad_bias)
{
    __shared__ float lds[kFoldWaves][kWave];
    const uint32_t wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    W *out = blockIdx.y ? grad_bias : grad_weight;
    if (!out) return;
    for (uint32_t base = blockIdx.x * kWave; base < cols; base += gridDim.x * kWave) {
        const uint32_t col = base + lane;
        float sum = 0.0f;
        if (col < cols) {
            const float *p = partial + (uint64_t)blockIdx.y * cols + col;
#pragma unroll 16
            for (uint32_t i = wave; i < parts; i += kFoldWaves) sum += p[(uint64_t)i * 2 * cols];
        }
        lds[wave][lane] = sum;
        __syncthreads();
        if (wave == 0 && col < cols) {
#pragma unroll
            for (int w = 1; w < kFoldWaves; ++w) sum += lds[w][lane];
            out[col] = (W)sum;
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- launches
// (a launch has less than 2^32 threads: with more rows, workgroups take several)
constexpr uint64_t kMaxGroups = 1u << 20;
// Threads of a workgroup whose rows take nt each: as many rows as fit `atleast`.
constexpr int norm_threads(int nt, int atleast) { return nt >= atleast ? nt : atleast / nt * nt; }
// Workgroups that the device holds at once: all get the same number of rows, give
// or take one (one more per CU than is resident runs alone in the end: 16384 x 4096
// bfloat16 forward 53 us, 59 with one more).
template <class Kernel>
uint64_t resident_groups(DeviceCache &cache, Kernel kernel, int threads)
{
    return (uint64_t)device_cus() * device_cached(cache, [&] {
               int n = 0;
               const hipError_t e = hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0);
               return e == hipSuccess && n > 0 ? n : 1;
           });
}

// NT threads with K octets each for a row of `octets`: the smallest group of
// waves that holds it.  f(NT, K) as integral constants; false if the row is longer
// or f has no kernel of that shape.  PER: octets of a thread in rows of several
// waves.  Two are better for the forward pass of 2-byte types, one for 4-byte types
// (us between events, one -> two: 16384 x 4096 bfloat16 55.6 -> 52.6, 16384 x 5120 87 -> 77,
// 3000 x 4608 19 -> 15; 2000 x 4096 float32 15.0 -> 17.5).  The backward pass keeps sums
// for each octet; two lose with few rows or full groups (1777 x 5001 float16 with the sum 27.2
// -> 29.7, 8000 x 7000 bfloat16 56 -> 60) and win with many rows of 5120 columns (104 -> 89).
// FINE: a group for 640 octets too, for the forward pass without the sum (16384 x 5120
// bfloat16 83 -> 77, 8000 x 5001 50 -> 45, 3000 x 4608 19 -> 15); with the sum (113 -> 117 at
// 16384 x 5120) and backward (60.5 -> 63 at 8000 x 5001, 21.0 -> 23.4 at 3000 x 4608) the larger
// group's waves fill the CU better.
template <int NT, int K, class F>
bool norm_shape_of(F f)
{
    return f(std::integral_constant<int, NT>{}, std::integral_constant<int, K>{});
}
template <int PER, bool FINE, class F>
bool norm_shape(uint32_t octets, F f)
{
    if (octets <= 16) return norm_shape_of<16, 1>(f);
    if (octets <= 32) return norm_shape_of<32, 1>(f);
    if (octets <= 64) return norm_shape_of<64, 1>(f);
    if (octets <= 128) return norm_shape_of<64, 2>(f);
    if (octets <= 192) return norm_shape_of<192, 1>(f);
    if (octets <= 256) return norm_shape_of<256 / PER, PER>(f);
    if (octets <= 384) return norm_shape_of<384 / PER, PER>(f);
    if (octets <= 512) return norm_shape_of<512 / PER, PER>(f);
    if constexpr (FINE) {
        if (octets <= 640) return norm_shape_of<640 / PER, PER>(f);
    }
    if (octets <= 768) return norm_shape_of<768 / PER, PER>(f);
    if (octets <= 1024) return norm_shape_of<1024 / PER, PER>(f);
    if (octets <= 2048) return norm_shape_of<512, 4>(f);
    if (octets <= 4096) return norm_shape_of<1024, 4>(f);
    return false;
}

template <class T, class W, bool ADD>
int norm_forward_launch(const NormArgs &a, hipStream_t s)
{
    const uint32_t octets = a.cols / kOctet;
    const char *name = ADD ? "layer_norm_add_forward" : "layer_norm_forward";
    const bool fits = norm_shape<sizeof(T) == 2 ? 2 : 1, !ADD>(octets, [&](auto nt, auto k) {
        constexpr int NT = decltype(nt)::value, K = decltype(k)::value;
        constexpr int THREADS = norm_threads(NT, 256);
        if constexpr (ADD && NT * K > 2048) {
            return false;  // (the registers do not hold it: it would spill)
        } else {
            const auto kernel = norm_forward_kernel<T, W, NT, K, THREADS, ADD, K <= 2>;
            static DeviceCache cache;
            const uint32_t grid =
                (uint32_t)std::min(ceil_div(a.rows, THREADS / NT), resident_groups(cache, kernel, THREADS));
            LCPP_LAUNCH(name, s, kernel<<<grid, THREADS, 0, s>>>(a));
            return true;
        }
    });
    if (!fits)
        LCPP_LAUNCH(name, s,
                    norm_forward_long_kernel<T, W, ADD>
                    <<<(uint32_t)std::min<uint64_t>(a.rows, kMaxGroups), kLongThreads, 0, s>>>(a));
    LCPP_CHECK_LAUNCH();
    return LCPP_OK;
}

// Partial sums of dw and db: at most one for each of two workgroups per CU.
constexpr uint64_t kMaxParts = 512;
uint64_t norm_parts(uint64_t rows) { return rows < kMaxParts ? rows : kMaxParts; }
uint64_t norm_backward_temp(uint64_t rows, uint64_t cols)
{
    return rows && cols ? kStatusBytes + align_up(norm_parts(rows) * 2 * cols * sizeof(float), 256) : 0;
}

template <class T, class W, bool ADD>
int norm_backward_launch(const NormGradArgs &a, W *grad_weight, W *grad_bias, hipStream_t s)
{
    const uint32_t octets = a.cols / kOctet;
    const char *name = ADD ? "layer_norm_add_backward" : "layer_norm_backward";
    uint32_t parts = 0;
    // rows whose columns' sums do not fit the registers: these are summed first (ds may go where dy or s lies)
    auto columns = [&] {
        if (!a.partial) return;
        const uint32_t blocks = (uint32_t)ceil_div(a.cols, kColThreads * kOctet);
        parts = (uint32_t)std::min<uint64_t>(ceil_div(a.rows, 8), std::min(std::max(kColGroups / blocks, 8u), (uint32_t)kMaxParts));
        LCPP_LAUNCH("layer_norm_backward_cols", s,
                    norm_backward_cols_kernel<T><<<dim3(blocks, parts), kColThreads, 0, s>>>(a));
    };
    const bool fits = norm_shape<1, false>(octets, [&](auto nt, auto k) {
        constexpr int NT = decltype(nt)::value, K = decltype(k)::value;
        constexpr int THREADS = norm_threads(NT, 512);
        constexpr bool kAcc = NT * K <= 2048;
        constexpr bool kAhead = K < 4 ? NT < 1024 || sizeof(T) == 2 || !ADD : kAcc && sizeof(T) == 2 && !ADD;
        if constexpr (ADD && !kAcc) {
            return false;  // (the registers do not hold it: it would spill)
        } else {
            const auto kernel = norm_backward_kernel<T, W, NT, K, THREADS, ADD, kAhead, kAcc>;
            static DeviceCache cache;
            uint32_t grid = (uint32_t)std::min(ceil_div(a.rows, THREADS / NT), resident_groups(cache, kernel, THREADS));
            if (kAcc) parts = grid = std::min<uint32_t>(grid, kMaxParts);
            else columns();
            LCPP_LAUNCH(name, s, kernel<<<grid, THREADS, 0, s>>>(a));
            return true;
        }
    });
    if (!fits) {
        columns();
        LCPP_LAUNCH(name, s,
                    norm_backward_long_kernel<T, W, ADD>
                    <<<(uint32_t)std::min<uint64_t>(a.rows, kMaxGroups), kLongThreads, 0, s>>>(a));
    }
    if (a.partial)
        LCPP_LAUNCH("layer_norm_fold", s,
                    norm_fold_kernel<W><<<dim3((uint32_t)std::min<uint64_t>(ceil_div(a.cols, kWave), kMaxGroups), 2), kFoldWaves * kWave, 0, s>>>(
                        a.partial, parts, a.cols, grad_weight, grad_bias));
    LCPP_CHECK_LAUNCH();
    return LCPP_OK;
}

template <class W>
__global__ void norm_zero_kernel(W *x, W *y, uint32_t n, uint32_t *status)
{
    if (status && blockIdx.x == 0 && threadIdx.x == 0) *status = 0;
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) {
        if (x) x[i] = (W)0.0f;
        if (y) y[i] = (W)0.0f;
    }
}

// The rows' type, and the weights' type, which is the same or float32.
template <class F>
int norm_dispatch(lcpp_dtype t, lcpp_dtype wt, F f)
{
    if (wt != t && wt != LCPP_FLOAT32) return LCPP_ERR_UNSUPPORTED_DTYPE;
    return float_dispatch(t, [&](auto x) -> int {
        using T = decltype(x);
        if (wt == t) return f(x, x);
        if constexpr (!std::is_same_v<T, float>) return f(x, float());
        return LCPP_ERR_UNSUPPORTED_DTYPE;
    });
}

bool norm_pointer(const void *p, size_t size, bool needed) { return p ? elem_ok(p, size) : !needed; }

int norm_forward(lcpp_dtype t, lcpp_dtype wt, bool add, const NormArgs &a, uint64_t rows, uint64_t cols, hipStream_t s)
{
    const size_t e = float_size(t), we = float_size(wt);
    if (!e || !we || (wt != t && wt != LCPP_FLOAT32)) return LCPP_ERR_UNSUPPORTED_DTYPE;
    if (rows > kMaxRows || cols > kMaxCols) return LCPP_ERR_INVALID_ARG;
    if (rows == 0 || cols == 0) return LCPP_OK;
    if (!elem_ok(a.in, e) || !elem_ok(a.out, e) || !rows_apart(a.out_stride, rows, cols)) return LCPP_ERR_INVALID_ARG;
    if (!norm_pointer(a.weight, we, false) || !norm_pointer(a.bias, we, false)) return LCPP_ERR_INVALID_ARG;
    if (!norm_pointer(a.mean, 4, false) || !norm_pointer(a.rstd, 4, false)) return LCPP_ERR_INVALID_ARG;
    if (!(a.eps >= 0.0f)) return LCPP_ERR_INVALID_ARG;
    if (add && (!elem_ok(a.residual, e) || !elem_ok(a.sum, e) || !rows_apart(a.sum_stride, rows, cols)))
        return LCPP_ERR_INVALID_ARG;
    if (same_place(a.mean, a.rstd) || (add && same_place(a.sum, a.out))) return LCPP_ERR_INVALID_ARG;
    return norm_dispatch(t, wt, [&](auto x, auto w) -> int {
        using T = decltype(x);
        using W = decltype(w);
        return add ? norm_forward_launch<T, W, true>(a, s) : norm_forward_launch<T, W, false>(a, s);
    });
}

int norm_backward(lcpp_dtype t, lcpp_dtype wt, bool add, void *temp, size_t temp_bytes, NormGradArgs &a,
                  void *grad_weight, void *grad_bias, uint64_t rows, uint64_t cols, hipStream_t s)
{
    const size_t e = float_size(t), we = float_size(wt);
    if (!e || !we || (wt != t && wt != LCPP_FLOAT32)) return LCPP_ERR_UNSUPPORTED_DTYPE;
    if (rows > kMaxRows || cols > kMaxCols) return LCPP_ERR_INVALID_ARG;
    if (cols == 0) return LCPP_OK;
    if (!norm_pointer(grad_weight, we, false) || !norm_pointer(grad_bias, we, false)) return LCPP_ERR_INVALID_ARG;
    if (temp && temp_bytes >= kStatusBytes && !(reinterpret_cast<uintptr_t>(temp) & 255))
        a.status = static_cast<uint32_t *>(temp);
    if (rows == 0) {  // sums over no rows
        if (!grad_weight && !grad_bias) return LCPP_OK;
        return norm_dispatch(t, wt, [&](auto, auto w) -> int {
            using W = decltype(w);
            LCPP_LAUNCH("layer_norm_zero", s,
                        norm_zero_kernel<W><<<(uint32_t)std::min<uint64_t>(ceil_div(cols, 256), 1024), 256, 0, s>>>(
                            static_cast<W *>(grad_weight), static_cast<W *>(grad_bias), (uint32_t)cols, a.status));
            LCPP_CHECK_LAUNCH();
            return LCPP_OK;
        });
    }
    if (!elem_ok(a.grad_out, e) || !elem_ok(a.in, e) || !elem_ok(a.mean, 4) || !elem_ok(a.rstd, 4))
        return LCPP_ERR_INVALID_ARG;
    if (!norm_pointer(a.weight, we, false) || !norm_pointer(a.grad_sum, e, false)) return LCPP_ERR_INVALID_ARG;
    if (!norm_pointer(a.grad_in, e, !add) || !norm_pointer(a.grad_branch, e, false)) return LCPP_ERR_INVALID_ARG;
    if (a.grad_in && !rows_apart(a.gi_stride, rows, cols)) return LCPP_ERR_INVALID_ARG;
    if (a.grad_branch && !rows_apart(a.gb_stride, rows, cols)) return LCPP_ERR_INVALID_ARG;
    if (grad_weight || grad_bias) {
        if (temp_bytes < norm_backward_temp(rows, cols)) return LCPP_ERR_TEMP_TOO_SMALL;
        if (!temp || (reinterpret_cast<uintptr_t>(temp) & 255)) return LCPP_ERR_INVALID_ARG;
        a.partial = reinterpret_cast<float *>(static_cast<char *>(temp) + kStatusBytes);
    }
    // (without dropout the two gradients of rows are the same)
    if (same_place(grad_weight, grad_bias) || (a.drop.cut && same_place(a.grad_in, a.grad_branch))) return LCPP_ERR_INVALID_ARG;
    return norm_dispatch(t, wt, [&](auto x, auto w) -> int {
        using T = decltype(x);
        using W = decltype(w);
        W *gw = static_cast<W *>(grad_weight), *gb = static_cast<W *>(grad_bias);
        return add ? norm_backward_launch<T, W, true>(a, gw, gb, s) : norm_backward_launch<T, W, false>(a, gw, gb, s);
    });
}

}  // namespace
}  // namespace lcpp

using namespace lcpp;

extern "C" int lcpp_layer_norm_forward(lcpp_dtype t, lcpp_dtype wt, const void *in, uint64_t in_stride,
                                       const void *weight, const void *bias, float eps, void *out, uint64_t out_stride,
                                       float *mean, float *rstd, uint64_t rows, uint64_t cols, void *stream)
{
    NormArgs a = {};
    a.in = in, a.weight = weight, a.bias = bias, a.out = out;
    a.in_stride = in_stride, a.out_stride = out_stride;
    a.mean = mean, a.rstd = rstd, a.rows = (uint32_t)rows, a.cols = (uint32_t)cols, a.eps = eps;
    return norm_forward(t, wt, false, a, rows, cols, static_cast<hipStream_t>(stream));
}

extern "C" int lcpp_layer_norm_add_forward(lcpp_dtype t, lcpp_dtype wt, const void *in, uint64_t in_stride,
                                           const void *residual, uint64_t residual_stride, double p, uint64_t seed,
                                           uint64_t offset, const uint64_t *offset_dev, const void *weight,
                                           const void *bias, float eps, void *sum, uint64_t sum_stride, void *out,
                                           uint64_t out_stride, float *mean, float *rstd, uint64_t rows, uint64_t cols,
                                           void *stream)
{
    NormArgs a = {};
    if (!drop_args(p, seed, offset, offset_dev, &a.drop)) return LCPP_ERR_INVALID_ARG;
    a.in = in, a.residual = residual, a.weight = weight, a.bias = bias, a.sum = sum, a.out = out;
    a.in_stride = in_stride, a.residual_stride = residual_stride, a.sum_stride = sum_stride, a.out_stride = out_stride;
    a.mean = mean, a.rstd = rstd, a.rows = (uint32_t)rows, a.cols = (uint32_t)cols, a.eps = eps;
    return norm_forward(t, wt, true, a, rows, cols, static_cast<hipStream_t>(stream));
}

extern "C" int lcpp_layer_norm_backward_temp_bytes(lcpp_dtype t, uint64_t rows, uint64_t cols, size_t *bytes)
{
    if (!bytes || rows > kMaxRows || cols > kMaxCols) return LCPP_ERR_INVALID_ARG;
    if (!float_size(t)) return LCPP_ERR_UNSUPPORTED_DTYPE;
    *bytes = norm_backward_temp(rows, cols);
    return LCPP_OK;
}

extern "C" int lcpp_layer_norm_backward(lcpp_dtype t, lcpp_dtype wt, void *temp, size_t temp_bytes, const void *grad_out,
                                        uint64_t grad_out_stride, const void *in, uint64_t in_stride, const void *weight,
                                        const float *mean, const float *rstd, void *grad_in, uint64_t grad_in_stride,
                                        void *grad_weight, void *grad_bias, uint64_t rows, uint64_t cols, void *stream)
{
    NormGradArgs a = {};
    a.grad_out = grad_out, a.in = in, a.weight = weight, a.grad_in = grad_in;
    a.go_stride = grad_out_stride, a.in_stride = in_stride, a.gi_stride = grad_in_stride;
    a.mean = mean, a.rstd = rstd, a.rows = (uint32_t)rows, a.cols = (uint32_t)cols;
    return norm_backward(t, wt, false, temp, temp_bytes, a, grad_weight, grad_bias, rows, cols,
                         static_cast<hipStream_t>(stream));
}

extern "C" int lcpp_layer_norm_add_backward(lcpp_dtype t, lcpp_dtype wt, void *temp, size_t temp_bytes,
                                            const void *grad_out, uint64_t grad_out_stride, const void *grad_sum,
                                            uint64_t grad_sum_stride, const void *sum, uint64_t sum_stride,
                                            const void *weight, const float *mean, const float *rstd, double p,
                                            uint64_t seed, uint64_t offset, const uint64_t *offset_dev,
                                            void *grad_residual, uint64_t grad_residual_stride, void *grad_in,
                                            uint64_t grad_in_stride, void *grad_weight, void *grad_bias, uint64_t rows,
                                            uint64_t cols, void *stream)
{
    NormGradArgs a = {};
    if (!drop_args(p, seed, offset, offset_dev, &a.drop)) return LCPP_ERR_INVALID_ARG;
    a.grad_out = grad_out, a.grad_sum = grad_sum, a.in = sum, a.weight = weight;
    a.grad_in = grad_residual, a.grad_branch = grad_in;
    a.go_stride = grad_out_stride, a.gs_stride = grad_sum_stride, a.in_stride = sum_stride;
    a.gi_stride = grad_residual_stride, a.gb_stride = grad_in_stride;
    a.mean = mean, a.rstd = rstd, a.rows = (uint32_t)rows, a.cols = (uint32_t)cols;
    return norm_backward(t, wt, true, temp, temp_bytes, a, grad_weight, grad_bias, rows, cols,
                         static_cast<hipStream_t>(stream));
}
