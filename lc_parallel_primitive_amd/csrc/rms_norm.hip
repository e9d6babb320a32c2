// rms_norm.hip — root-mean-square norm over rows, alone or with the residual's sum
// before it, with an output in the rows' type, in 8-bit floating point with scales,
// or both; and its gradient.
//
//   s = x, or s = residual + x, stored in the rows' type
//   rstd = 1 / sqrt(sum(s^2) / n + eps)
//   y = s rstd w
//   8 bits: for each group of columns amax = max |y|, scale = max(amax, 2^-100) / m with
//   m the format's largest value, q = y / scale, a quotient of 32 bits rounded to nearest
//   even.  A group with a y that is not finite has the scale NaN and values NaN.
//
// With v = dy w the gradients are
//   ds = rstd (v - s rstd^2 sum(v s) / n)   [+ the gradient that reaches s elsewhere]
//   dw = sum over rows of dy s rstd
// and both x and the residual have the gradient ds.
//
// Bound by memory, and laid out as the layer norm is: a row in the registers of as few
// threads as hold it, several rows of a workgroup one after the other with the next
// ones on their way, dw in registers over all of a workgroup's rows and one partial sum
// per workgroup, which a second launch adds in a fixed order.  A group's columns lie in
// neighbouring lanes, so its maximum takes two to six lane exchanges and no LDS.
// 32768 x 2048 bfloat16 with the sum and 8 bits in groups of 128: 91 us, 5.2 TB/s; 16384 x
// 4096 with the sum, forward 87 us, 6.2 TB/s, backward 108 + 5, 5.1 TB/s; a copy of 512 MiB
// runs at 5.2 to 5.35.
#include "row_group.hpp"

namespace lcpp {
namespace {

struct RmsArgs {
    const void *in, *residual, *weight;
    void *sum, *out, *quant;
    uint64_t in_stride, residual_stride, sum_stride, out_stride, quant_stride;
    float *scales, *rstd;
    uint64_t scale_row, scale_col;  // strides of the scales
    uint32_t rows, cols;
    uint32_t group;    // octets of a group of columns, 0: the whole row
    uint32_t log2_lanes;  // of the lanes that hold a group
    float eps, qmax;
    bool wide_weight;  // weights are float32
    bool e5m2;
};

// Eight weights as floats, or ones.
template <class T>
__device__ __forceinline__ void weight_octet(const void *p, bool wide, uint32_t col, float (&w)[kOctet])
{
    if (!p) {
#pragma unroll
        for (int i = 0; i < kOctet; ++i) w[i] = 1.0f;
    } else if (wide) {
        const Octet<float> o = load_pack<kOctet>(static_cast<const float *>(p) + col);
#pragma unroll
        for (int i = 0; i < kOctet; ++i) w[i] = o[i];
    } else {
        const Octet<T> o = load_pack<kOctet>(static_cast<const T *>(p) + col);
#pragma unroll
        for (int i = 0; i < kOctet; ++i) w[i] = o[i];
    }
}
template <class T>
__device__ __forceinline__ float weight_one(const void *p, bool wide, uint32_t col)
{
    if (!p) return 1.0f;
    return wide ? static_cast<const float *>(p)[col] : (float)static_cast<const T *>(p)[col];
}
template <class T>
__device__ __forceinline__ void weight_octet_part(const void *p, bool wide, uint32_t col, uint32_t cols, float (&w)[kOctet])
{
    if (col + kOctet <= cols) return weight_octet<T>(p, wide, col, w);
#pragma unroll
    for (int i = 0; i < kOctet; ++i) w[i] = col + i < cols ? weight_one<T>(p, wide, col + i) : 0.0f;
}

// ---------------------------------------------------------------- 8 bits
// |y| as bits: ordered like the values, with NaN above infinity, so that the maximum of
// a group shows a NaN.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu; }
struct UMax {
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return a > b ? a : b; }
};
// The maximum over 2^n neighbouring lanes (n uniform, 0 to 6), in each of them.
__device__ __forceinline__ uint32_t lanes_max(uint32_t x, uint32_t n)
{
    const UMax m;
    if (n > 0) x = m(x, dpp_perm<kDppQuadXor1>(x));
    if (n > 1) x = m(x, dpp_perm<kDppQuadXor2>(x));
    if (n > 2) x = m(x, dpp_perm<kDppRowHalfMirror>(x));
    if (n > 3) x = m(x, dpp_perm<kDppRowMirror>(x));
    if (n > 4) x = m(x, shfl_xor(x, 16));
    if (n > 5) x = m(x, shfl_xor(x, 32));
    return x;
}
constexpr float kSmallestMax = 7.888609052210118e-31f;  // 2^-100: 1 / scale stays finite
struct Scale {
    float scale, inverse;
};
__device__ __forceinline__ Scale make_scale(uint32_t amax, float qmax)
{
    // (infinite or NaN: a NaN for both)
    const float a = amax < 0x7F800000u ? __builtin_bit_cast(float, amax) : std::numeric_limits<float>::quiet_NaN();
    Scale s;
    s.scale = (a < kSmallestMax ? kSmallestMax : a) / qmax;
    s.inverse = 1.0f / s.scale;
    return s;
}
// x / scale rounded to 32 bits.  The product with the rounded reciprocal is off by up to two units in its last place, which
// turns one of 14 quotients half way between two 8-bit values to the wrong side; what it leaves of x is a number of 32
// bits, which corrects it.  (The signs are those that keep a zero's.)
__device__ __forceinline__ float quotient(float x, const Scale &s)
{
    const float r = x * s.inverse;
    return fmaf(-fmaf(r, s.scale, -x), s.inverse, r);
}
// Two numbers in 8 bits: no more than the largest value and a rounding of 32 bits, which rounds to it.
__device__ __forceinline__ uint32_t quant_pair(float x, float y, bool e5m2, uint32_t old, bool high)
{
    if (e5m2) return high ? __builtin_amdgcn_cvt_pk_bf8_f32(x, y, (int)old, true) : __builtin_amdgcn_cvt_pk_bf8_f32(x, y, (int)old, false);
    return high ? __builtin_amdgcn_cvt_pk_fp8_f32(x, y, (int)old, true) : __builtin_amdgcn_cvt_pk_fp8_f32(x, y, (int)old, false);
}
__device__ __forceinline__ void quant_octet(const float (&y)[kOctet], const Scale &s, bool e5m2, uint8_t (&q)[kOctet])
{
    uint32_t w[2] = {};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        w[h] = quant_pair(quotient(y[4 * h], s), quotient(y[4 * h + 1], s), e5m2, 0, false);
        w[h] = quant_pair(quotient(y[4 * h + 2], s), quotient(y[4 * h + 3], s), e5m2, w[h], true);
    }
    __builtin_memcpy(q, w, sizeof(w));
}
__device__ __forceinline__ void store_bytes(uint8_t *p, const uint8_t (&q)[kOctet])
{
    typedef uint8_t vec __attribute__((ext_vector_type(kOctet)));
    typedef vec vec_u __attribute__((aligned(1)));
    vec v;
    __builtin_memcpy(&v, q, sizeof(v));
    *reinterpret_cast<vec_u *>(p) = v;
}

// The maximum over the NT threads of a row's group of threads.
template <int NT, int WAVES>
__device__ __forceinline__ uint32_t group_max(uint32_t x, uint32_t (*lds)[WAVES], int slot)
{
    x = lanes_max(x, NT >= kWave ? 6 : NT == 32 ? 5 : 4);
    if constexpr (NT > kWave) {
        constexpr int GW = NT / kWave;
        const uint32_t wave = threadIdx.x / kWave;
        if (lane_id() == 0) lds[slot][wave] = x;
        group_barrier();
        const uint32_t first = wave / GW * GW;
#pragma unroll
        for (int w = 0; w < GW; ++w) x = UMax()(x, lds[slot][first + w]);
    }
    return x;
}

// ---------------------------------------------------------------- forward
template <class T, int NT, int K, int THREADS, bool ADD, bool Q, bool AHEAD>
__global__ __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(AHEAD ? 1 : 2))) void rms_forward_kernel(RmsArgs a)
{
    constexpr int WAVES = THREADS / kWave, RG = THREADS / NT;
    constexpr uint32_t kRowLanes = NT >= kWave ? 6 : NT == 32 ? 5 : 4;  // (a row's lanes in a wave, as a power of 2)
    __shared__ float lds[2][WAVES][2];
    __shared__ uint32_t lds_max[2][WAVES];
    __shared__ uint32_t lds_tail[2][RG][2];
    const Columns<NT, K> c(a.cols);
    const uint32_t group = threadIdx.x / NT;
    const float inv_cols = 1.0f / (float)a.cols;
    float w[K][kOctet], w_tail = 1.0f;
    auto weights = [&](int k) {
        if (c.has(k)) weight_octet<T>(a.weight, a.wide_weight, c.col(k), w[k]);
    };
    if constexpr (AHEAD) {
#pragma unroll
        for (int k = 0; k < K; ++k) weights(k);
    }
    if (c.has_tail()) w_tail = weight_one<T>(a.weight, a.wide_weight, c.tail());
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
                    for (int i = 0; i < kOctet; ++i) {
                        v[i] = x.o[k][i] + r.o[k][i];
                        x.o[k].v[i] = (T)v[i];
                    }
                    store_pack<kOctet>(sum + c.col(k), v);
                }
                if (c.has_tail()) {
                    if constexpr (!AHEAD) r.tail = residual[row * a.residual_stride + c.tail()];
                    x.tail = (T)((float)x.tail + (float)r.tail);
                    sum[c.tail()] = x.tail;
                }
            }
        }
        float sq[1] = {0.0f};
        if (live) {
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (c.has(k))
#pragma unroll
                    for (int i = 0; i < kOctet; ++i) sq[0] += x.o[k][i] * x.o[k][i];
            if (c.has_tail()) sq[0] += (float)x.tail * (float)x.tail;
        }
        group_sum<NT, WAVES>(sq, lds, slot);
        const float rstd = 1.0f / sqrtf(sq[0] * inv_cols + a.eps);
        if (live && c.t == 0 && a.rstd) a.rstd[row] = rstd;
        auto y_octet = [&](int k, float(&y)[kOctet]) {
#pragma unroll
            for (int i = 0; i < kOctet; ++i) y[i] = x.o[k][i] * rstd * w[k][i];
        };
        const float y_tail = (float)x.tail * rstd * w_tail;
        if (live && (!Q || a.out)) {
            T *out = static_cast<T *>(a.out) + row * a.out_stride;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (!c.has(k)) continue;
                if constexpr (!AHEAD) weights(k);
                float y[kOctet];
                y_octet(k, y);
                store_pack_nt<kOctet>(out + c.col(k), y);
            }
            if (c.has_tail()) out[c.tail()] = (T)y_tail;
        }
        if constexpr (Q) {
            uint32_t most[K];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                most[k] = 0;
                if (!live || !c.has(k)) continue;
                if constexpr (!AHEAD) weights(k);
                float y[kOctet];
                y_octet(k, y);
#pragma unroll
                for (int i = 0; i < kOctet; ++i) most[k] = UMax()(most[k], abs_bits(y[i]));
            }
            uint32_t tail_most = live && c.has_tail() ? abs_bits(y_tail) : 0;
            const uint32_t octets = c.full / kOctet;
            uint32_t tail_group = 0;
            if (a.group == 0) {
                uint32_t all = tail_most;
#pragma unroll
                for (int k = 0; k < K; ++k) all = UMax()(all, most[k]);
                all = group_max<NT, WAVES>(all, lds_max, slot);
#pragma unroll
                for (int k = 0; k < K; ++k) most[k] = all;
                tail_most = all;
            } else {
#pragma unroll
                for (int k = 0; k < K; ++k) most[k] = lanes_max(most[k], std::min(a.log2_lanes, kRowLanes));
                if (c.rem) {
                    // the last columns lie in other lanes than their group's octets: both maxima meet in LDS
                    tail_group = octets >> a.log2_lanes;
                    const bool shared = octets & (a.group - 1);
                    tail_most = lanes_max(tail_most, 3);  // (of the first lanes, which hold them)
                    if (c.t == 0) {
                        lds_tail[slot][group][0] = tail_most;
                        if (!shared) lds_tail[slot][group][1] = 0;
                    }
#pragma unroll
                    for (int k = 0; k < K; ++k)
                        if (shared && c.t + k * NT == octets - 1) lds_tail[slot][group][1] = most[k];
                    group_barrier();
                    tail_most = UMax()(lds_tail[slot][group][0], lds_tail[slot][group][1]);
#pragma unroll
                    for (int k = 0; k < K; ++k)
                        if ((c.t + k * NT) >> a.log2_lanes == tail_group) most[k] = tail_most;
                }
            }
            if (live) {
                uint8_t *q = static_cast<uint8_t *>(a.quant) + row * a.quant_stride;
                float *scales = a.scales + row * a.scale_row;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (!c.has(k)) continue;
                    const Scale s = make_scale(most[k], a.qmax);
                    float y[kOctet];
                    uint8_t b[kOctet];
                    y_octet(k, y);
                    quant_octet(y, s, a.e5m2, b);
                    store_bytes(q + c.col(k), b);
                    const uint32_t octet = c.t + k * NT;
                    const uint32_t g = a.group ? octet >> a.log2_lanes : 0;
                    if (octet == g * a.group) scales[g * a.scale_col] = s.scale;
                }
                if (c.has_tail()) {
                    const Scale s = make_scale(tail_most, a.qmax);
                    q[c.tail()] = (uint8_t)quant_pair(quotient(y_tail, s), 0.0f, a.e5m2, 0, false);
                    // (a group of these columns alone)
                    if (c.t == 0 && octets == tail_group * a.group) scales[tail_group * a.scale_col] = s.scale;
                }
            }
        }
    }
}

// Longer rows: a workgroup reads its row two or three times (from the caches).
template <class T, bool ADD, bool Q>
__global__ __launch_bounds__(kLongThreads) void rms_forward_long_kernel(RmsArgs a)
{
    __shared__ float lds[2][kLongWaves][2];
    __shared__ uint32_t lds_max[2][kLongWaves];
    int slot = 0;
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x, slot ^= 1) {
        const T *in = static_cast<const T *>(a.in) + row * a.in_stride;
        const T *s = ADD ? static_cast<const T *>(a.sum) + row * a.sum_stride : in;
        float sq[1] = {0.0f};
        for (uint32_t col = threadIdx.x * kOctet; col < a.cols; col += kLongThreads * kOctet) {
            Octet<T> x = load_octet(in, col, a.cols);
            if constexpr (ADD) {
                const Octet<T> r = load_octet(static_cast<const T *>(a.residual) + row * a.residual_stride, col, a.cols);
                float v[kOctet];
#pragma unroll
                for (int i = 0; i < kOctet; ++i) {
                    v[i] = x[i] + r[i];
                    x.v[i] = (T)v[i];
                }
                store_octet(static_cast<T *>(a.sum) + row * a.sum_stride, col, a.cols, v);
            }
#pragma unroll
            for (int i = 0; i < kOctet; ++i) sq[0] += x[i] * x[i];
        }
        group_sum<kLongThreads, kLongWaves>(sq, lds, slot);
        const float rstd = 1.0f / sqrtf(sq[0] / (float)a.cols + a.eps);
        if (threadIdx.x == 0 && a.rstd) a.rstd[row] = rstd;
        // (each thread reads back the sums that it stored itself; past the row's end y is 0)
        auto y_octet = [&](uint32_t col, float(&y)[kOctet]) {
            const Octet<T> x = load_octet(s, col, a.cols);
            float w[kOctet];
            weight_octet_part<T>(a.weight, a.wide_weight, col, a.cols, w);
#pragma unroll
            for (int i = 0; i < kOctet; ++i) y[i] = col + i < a.cols ? x[i] * rstd * w[i] : 0.0f;
        };
        auto max_octet = [&](const float(&y)[kOctet]) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < kOctet; ++i) m = UMax()(m, abs_bits(y[i]));
            return m;
        };
        uint32_t all = 0;
        if constexpr (Q) {
            if (a.group == 0) {
                for (uint32_t col = threadIdx.x * kOctet; col < a.cols; col += kLongThreads * kOctet) {
                    float y[kOctet];
                    y_octet(col, y);
                    all = UMax()(all, max_octet(y));
                }
                all = group_max<kLongThreads, kLongWaves>(all, lds_max, slot);
                if (threadIdx.x == 0) a.scales[row * a.scale_row] = make_scale(all, a.qmax).scale;
            }
        }
        // (all lanes of a wave make the rounds that one makes: they exchange maxima)
        const uint32_t wave_col = threadIdx.x / kWave * kWave * kOctet;
        for (uint32_t from = wave_col; from < a.cols; from += kLongThreads * kOctet) {
            const uint32_t col = from + lane_id() * kOctet;
            float y[kOctet];
            if (col < a.cols) {
                y_octet(col, y);
                if (!Q || a.out) store_octet(static_cast<T *>(a.out) + row * a.out_stride, col, a.cols, y);
            } else {
#pragma unroll
                for (int i = 0; i < kOctet; ++i) y[i] = 0.0f;
            }
            if constexpr (Q) {
                const uint32_t most = a.group ? lanes_max(max_octet(y), a.log2_lanes) : all;
                if (col < a.cols) {
                    const Scale sc = make_scale(most, a.qmax);
                    uint8_t b[kOctet];
                    quant_octet(y, sc, a.e5m2, b);
                    uint8_t *q = static_cast<uint8_t *>(a.quant) + row * a.quant_stride + col;
                    if (col + kOctet <= a.cols) {
                        store_bytes(q, b);
                    } else {
#pragma unroll
                        for (int i = 0; i < kOctet; ++i)
                            if (col + i < a.cols) q[i] = b[i];
                    }
                    const uint32_t octet = col / kOctet;
                    if (a.group && (octet & (a.group - 1)) == 0)
                        a.scales[row * a.scale_row + (octet >> a.log2_lanes) * a.scale_col] = sc.scale;
                }
            }
        }
    }
}

// ---------------------------------------------------------------- backward
struct RmsGradArgs {
    const void *grad_out, *grad_sum, *in, *weight;
    void *grad_in;
    uint64_t go_stride, gs_stride, in_stride, gi_stride;
    const float *rstd;
    float *partial;    // [workgroup][cols] sums of dw, or null
    uint32_t *status;  // the status word of the temp storage, cleared here (may be null)
    uint32_t rows, cols;
    bool wide_weight;
};

// As the forward pass; a thread keeps the same columns for all of its workgroup's
// rows, so dw is a sum in its registers.
template <class T, int NT, int K, int THREADS, bool ADD, bool AHEAD, bool ACC>
__global__ __launch_bounds__(THREADS) void rms_backward_kernel(RmsGradArgs a)
{
    constexpr int WAVES = THREADS / kWave, RG = THREADS / NT;
    constexpr int FOLD = !ACC ? 1 : NT < kWave ? WAVES : RG;  // turns of the fold below
    __shared__ float lds[2][WAVES][2];
    __shared__ float fold[FOLD > 1 ? NT * K * kOctet : 1], fold_tail[FOLD > 1 ? NT : 1];
    const Columns<NT, K> c(a.cols);
    const uint32_t group = threadIdx.x / NT;
    const float inv = 1.0f / (float)a.cols;
    if (a.status && blockIdx.x == 0 && threadIdx.x == 0) *a.status = 0;
    float w[K][kOctet], w_tail = 1.0f;
    auto weights = [&](int k) {
        if (c.has(k)) weight_octet<T>(a.weight, a.wide_weight, c.col(k), w[k]);
    };
    if constexpr (AHEAD) {
#pragma unroll
        for (int k = 0; k < K; ++k) weights(k);
    }
    if (c.has_tail()) w_tail = weight_one<T>(a.weight, a.wide_weight, c.tail());
    float dw[K][kOctet], dw_tail = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < kOctet; ++i) dw[k][i] = 0.0f;
    const T *grad_out = static_cast<const T *>(a.grad_out), *in = static_cast<const T *>(a.in);
    const T *grad_sum = static_cast<const T *>(a.grad_sum);
    RowPart<T, K> next_dy, next_s, next_g;
    float next_rstd = 0.0f;
    auto load = [&](uint64_t row) {
        if (row >= a.rows) return;
        next_dy.load(grad_out + row * a.go_stride, c);
        next_s.load(in + row * a.in_stride, c);
        if constexpr (ADD && AHEAD) next_g.load(grad_sum + row * a.gs_stride, c);
        next_rstd = a.rstd[row];
    };
    uint64_t row = (uint64_t)blockIdx.x * RG + group;
    if constexpr (AHEAD) load(row);
    const uint64_t stride = (uint64_t)gridDim.x * RG;
    int slot = 0;
    for (uint64_t base = (uint64_t)blockIdx.x * RG; base < a.rows; base += stride, row += stride, slot ^= 1) {
        if constexpr (!AHEAD) load(row);
        RowPart<T, K> dy = next_dy, s = next_s, g = next_g;
        const float rstd = next_rstd;
        const bool live = row < a.rows;
        if constexpr (AHEAD) load(row + stride);
        float sums[1] = {0.0f};
        if (live) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (!c.has(k)) continue;
                if constexpr (!AHEAD) weights(k);
#pragma unroll
                for (int i = 0; i < kOctet; ++i) {
                    const float t = dy.o[k][i] * (s.o[k][i] * rstd);
                    sums[0] += t * w[k][i];
                    if constexpr (ACC) dw[k][i] += t;
                }
            }
            if (c.has_tail()) {
                const float t = (float)dy.tail * ((float)s.tail * rstd);
                sums[0] += t * w_tail;
                dw_tail += t;
            }
        }
        group_sum<NT, WAVES>(sums, lds, slot);
        if (!live) continue;
        const float mean = sums[0] * inv;  // of v u, u = s rstd
        T *gi = static_cast<T *>(a.grad_in) + row * a.gi_stride;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (!c.has(k)) continue;
            if constexpr (!AHEAD) {
                weights(k);
                if constexpr (ADD) g.o[k] = load_pack<kOctet>(grad_sum + row * a.gs_stride + c.col(k));
            }
            float d[kOctet];
#pragma unroll
            for (int i = 0; i < kOctet; ++i) {
                d[i] = rstd * (dy.o[k][i] * w[k][i] - (s.o[k][i] * rstd) * mean);
                if constexpr (ADD) d[i] += g.o[k][i];
            }
            store_pack_nt<kOctet>(gi + c.col(k), d);
        }
        if (c.has_tail()) {
            float d = rstd * ((float)dy.tail * w_tail - ((float)s.tail * rstd) * mean);
            if constexpr (ADD) {
                if constexpr (!AHEAD) g.tail = grad_sum[row * a.gs_stride + c.tail()];
                d += (float)g.tail;
            }
            gi[c.tail()] = (T)d;
        }
    }
    if (!ACC || !a.partial) return;
    uint32_t turn = group;
    bool writes = group == RG - 1;
    if constexpr (NT < kWave) {
#pragma unroll
        for (int step = NT; step < kWave; step *= 2) {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < kOctet; ++i) dw[k][i] += shfl_xor(dw[k][i], step);
            dw_tail += shfl_xor(dw_tail, step);
        }
        const bool first = lane_id() < NT;
        turn = first ? threadIdx.x / kWave : WAVES;
        writes = first && turn == WAVES - 1;
    }
    if constexpr (FOLD > 1) {
        // the groups add to the columns' sums one after the other, in a fixed order
        for (uint32_t f = 0; f < FOLD; ++f) {
            if (turn == f) {
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < kOctet; ++i) {
                        float &at = fold[(i * K + k) * NT + c.t];
                        at = f ? at + dw[k][i] : dw[k][i];
                        dw[k][i] = at;
                    }
                if (c.has_tail()) {
                    float &at = fold_tail[c.t];
                    at = f ? at + dw_tail : dw_tail;
                    dw_tail = at;
                }
            }
            __syncthreads();
        }
    }
    if (writes) {
        float *part = a.partial + (uint64_t)blockIdx.x * a.cols;
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (c.has(k)) store_pack<kOctet>(part + c.col(k), dw[k]);
        if (c.has_tail()) part[c.tail()] = dw_tail;
    }
}

// Longer rows, ds: a workgroup reads its row twice (the second time from the caches).
template <class T, bool ADD>
__global__ __launch_bounds__(kLongThreads) void rms_backward_long_kernel(RmsGradArgs a)
{
    __shared__ float lds[2][kLongWaves][2];
    const float inv = 1.0f / (float)a.cols;
    if (a.status && blockIdx.x == 0 && threadIdx.x == 0) *a.status = 0;
    int slot = 0;
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x, slot ^= 1) {
        const float rstd = a.rstd[row];
        const T *dy = static_cast<const T *>(a.grad_out) + row * a.go_stride;
        const T *s = static_cast<const T *>(a.in) + row * a.in_stride;
        // v and u of an octet (past the row's end 0)
        auto terms = [&](uint32_t col, float(&v)[kOctet], float(&u)[kOctet]) {
            const Octet<T> d = load_octet(dy, col, a.cols), x = load_octet(s, col, a.cols);
            float w[kOctet];
            weight_octet_part<T>(a.weight, a.wide_weight, col, a.cols, w);
#pragma unroll
            for (int i = 0; i < kOctet; ++i) {
                u[i] = col + i < a.cols ? x[i] * rstd : 0.0f;
                v[i] = d[i] * w[i];
            }
        };
        float sums[1] = {0.0f};
        for (uint32_t col = threadIdx.x * kOctet; col < a.cols; col += kLongThreads * kOctet) {
            float v[kOctet], u[kOctet];
            terms(col, v, u);
#pragma unroll
            for (int i = 0; i < kOctet; ++i) sums[0] += v[i] * u[i];
        }
        group_sum<kLongThreads, kLongWaves>(sums, lds, slot);
        const float mean = sums[0] * inv;
        for (uint32_t col = threadIdx.x * kOctet; col < a.cols; col += kLongThreads * kOctet) {
            float v[kOctet], u[kOctet], d[kOctet];
            terms(col, v, u);
#pragma unroll
            for (int i = 0; i < kOctet; ++i) d[i] = rstd * (v[i] - u[i] * mean);
            if constexpr (ADD) {
                const Octet<T> g = load_octet(static_cast<const T *>(a.grad_sum) + row * a.gs_stride, col, a.cols);
#pragma unroll
                for (int i = 0; i < kOctet; ++i) d[i] += g[i];
            }
            store_octet(static_cast<T *>(a.grad_in) + row * a.gi_stride, col, a.cols, d);
        }
    }
}

// Longer rows, dw: a workgroup takes 2048 columns of every gridDim.y-th row.
constexpr int kRmsColThreads = 256;
constexpr uint32_t kRmsColGroups = 1024;  // workgroups that these partial sums are split over
template <class T>
__global__ __launch_bounds__(kRmsColThreads) void rms_backward_cols_kernel(RmsGradArgs a)
{
    const uint32_t col = (blockIdx.x * kRmsColThreads + threadIdx.x) * kOctet;
    if (col >= a.cols) return;
    float dw[kOctet] = {};
    for (uint64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const Octet<T> dy = load_octet(static_cast<const T *>(a.grad_out) + row * a.go_stride, col, a.cols);
        const Octet<T> s = load_octet(static_cast<const T *>(a.in) + row * a.in_stride, col, a.cols);
        const float rstd = a.rstd[row];
#pragma unroll
        for (int i = 0; i < kOctet; ++i)
            if (col + i < a.cols) dw[i] += dy[i] * (s[i] * rstd);
    }
    store_octet(a.partial + (uint64_t)blockIdx.y * a.cols, col, a.cols, dw);
}

// dw from the partial sums: 64 columns per workgroup at a time, each wave every 16th
// partial sum, always in the same order.
constexpr int kRmsFoldWaves = 16;
template <class W>
__global__ __launch_bounds__(kRmsFoldWaves *kWave) void rms_fold_kernel(const float *partial, uint32_t parts, uint32_t cols,
                                                                        W *grad_weight)
{
    __shared__ float lds[kRmsFoldWaves][kWave];
    const uint32_t wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    for (uint32_t base = blockIdx.x * kWave; base < cols; base += gridDim.x * kWave) {
        const uint32_t col = base + lane;
        float sum = 0.0f;
        if (col < cols) {
#pragma unroll 16
            for (uint32_t i = wave; i < parts; i += kRmsFoldWaves) sum += partial[(uint64_t)i * cols + col];
        }
        lds[wave][lane] = sum;
        __syncthreads();
        if (wave == 0 && col < cols) {
#pragma unroll
            for (int w = 1; w < kRmsFoldWaves; ++w) sum += lds[w][lane];
            grad_weight[col] = (W)sum;
        }
        __syncthreads();
    }
}
template <class W>
__global__ void rms_zero_kernel(W *x, uint32_t n, uint32_t *status)
{
    if (status && blockIdx.x == 0 && threadIdx.x == 0) *status = 0;
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) x[i] = (W)0.0f;
}

// ---------------------------------------------------------------- launches
template <class T, bool ADD, bool Q>
int rms_forward_launch(const RmsArgs &a, hipStream_t s)
{
    const char *name = Q ? ADD ? "rms_norm_add_quant" : "rms_norm_quant" : ADD ? "rms_norm_add_forward" : "rms_norm_forward";
    const bool fits = norm_shape<sizeof(T) == 2 ? 2 : 1, !ADD>(a.cols / kOctet, [&](auto nt, auto k) {
        constexpr int NT = decltype(nt)::value, K = decltype(k)::value;
        constexpr int THREADS = norm_threads(NT, 256);
        if constexpr ((ADD || Q) && NT * K > 2048) {
            return false;  // (the registers do not hold it: it would spill)
        } else {
            const auto kernel = rms_forward_kernel<T, NT, K, THREADS, ADD, Q, K <= 2>;
            static DeviceCache cache;
            const uint32_t grid =
                (uint32_t)std::min(ceil_div(a.rows, THREADS / NT), resident_groups(cache, kernel, THREADS));
            LCPP_LAUNCH(name, s, kernel<<<grid, THREADS, 0, s>>>(a));
            return true;
        }
    });
    if (!fits)
        LCPP_LAUNCH(name, s,
                    rms_forward_long_kernel<T, ADD, Q>
                    <<<(uint32_t)std::min<uint64_t>(a.rows, kMaxGroups), kLongThreads, 0, s>>>(a));
    LCPP_CHECK_LAUNCH();
    return LCPP_OK;
}

// Partial sums of dw: at most one for each of two workgroups per CU.
constexpr uint64_t kRmsMaxParts = 512;
uint64_t rms_backward_temp(uint64_t rows, uint64_t cols)
{
    return rows && cols ? kStatusBytes + align_up(std::min(rows, kRmsMaxParts) * cols * sizeof(float), 256) : 0;
}

template <class T, bool ADD>
int rms_backward_launch(const RmsGradArgs &a, void *grad_weight, hipStream_t s)
{
    uint32_t parts = 0;
    // rows whose columns' sums do not fit the registers: these are summed first (ds may go where dy or s lies)
    auto columns = [&] {
        if (!a.partial) return;
        const uint32_t blocks = (uint32_t)ceil_div(a.cols, kRmsColThreads * kOctet);
        parts = (uint32_t)std::min<uint64_t>(ceil_div(a.rows, 8),
                                             std::min(std::max(kRmsColGroups / blocks, 8u), (uint32_t)kRmsMaxParts));
        LCPP_LAUNCH("rms_norm_backward_cols", s,
                    rms_backward_cols_kernel<T><<<dim3(blocks, parts), kRmsColThreads, 0, s>>>(a));
    };
    const bool fits = norm_shape<1, false>(a.cols / kOctet, [&](auto nt, auto k) {
        constexpr int NT = decltype(nt)::value, K = decltype(k)::value;
        constexpr int THREADS = norm_threads(NT, 512);
        constexpr bool kAcc = NT * K <= 2048;
        constexpr bool kAhead = K < 4 ? NT < 1024 || sizeof(T) == 2 || !ADD : kAcc && sizeof(T) == 2 && !ADD;
        if constexpr (ADD && !kAcc) {
            return false;  // (the registers do not hold it: it would spill)
        } else {
            const auto kernel = rms_backward_kernel<T, NT, K, THREADS, ADD, kAhead, kAcc>;
            static DeviceCache cache;
            uint32_t grid = (uint32_t)std::min(ceil_div(a.rows, THREADS / NT), resident_groups(cache, kernel, THREADS));
            if (kAcc) parts = grid = std::min<uint32_t>(grid, kRmsMaxParts);
            else columns();
            LCPP_LAUNCH("rms_norm_backward", s, kernel<<<grid, THREADS, 0, s>>>(a));
            return true;
        }
    });
    if (!fits) {
        columns();
        LCPP_LAUNCH("rms_norm_backward", s,
                    rms_backward_long_kernel<T, ADD>
                    <<<(uint32_t)std::min<uint64_t>(a.rows, kMaxGroups), kLongThreads, 0, s>>>(a));
    }
    if (a.partial) {
        const uint32_t grid = (uint32_t)std::min<uint64_t>(ceil_div(a.cols, kWave), kMaxGroups);
        if (a.wide_weight)
            LCPP_LAUNCH("rms_norm_fold", s,
                        rms_fold_kernel<float><<<grid, kRmsFoldWaves * kWave, 0, s>>>(a.partial, parts, a.cols,
                                                                                      static_cast<float *>(grad_weight)));
        else
            LCPP_LAUNCH("rms_norm_fold", s,
                        rms_fold_kernel<T><<<grid, kRmsFoldWaves * kWave, 0, s>>>(a.partial, parts, a.cols,
                                                                                  static_cast<T *>(grad_weight)));
    }
    LCPP_CHECK_LAUNCH();
    return LCPP_OK;
}

}  // namespace
}  // namespace lcpp

using namespace lcpp;

extern "C" int lcpp_rms_norm_forward(lcpp_dtype t, lcpp_dtype wt, const void *in, uint64_t in_stride, const void *residual,
                                     uint64_t residual_stride, const void *weight, float eps, void *sum,
                                     uint64_t sum_stride, void *out, uint64_t out_stride, float *rstd, lcpp_dtype qt,
                                     void *quant, uint64_t quant_stride, float *scales, uint64_t scale_row_stride,
                                     uint64_t scale_group_stride, uint32_t group, uint64_t rows, uint64_t cols,
                                     void *stream)
{
    const size_t e = float_size(t), we = float_size(wt);
    if (!e || !we || (wt != t && wt != LCPP_FLOAT32)) return LCPP_ERR_UNSUPPORTED_DTYPE;
    if (quant && qt != LCPP_FLOAT8_E4M3 && qt != LCPP_FLOAT8_E5M2) return LCPP_ERR_UNSUPPORTED_DTYPE;
    if (rows > kMaxRows || cols > kMaxCols || !(eps >= 0.0f)) return LCPP_ERR_INVALID_ARG;
    // groups of 4 to 64 octets: what neighbouring lanes of a wave hold
    if (quant && group && (group < 32 || group > 512 || (group & (group - 1)))) return LCPP_ERR_INVALID_ARG;
    if (rows == 0 || cols == 0) return LCPP_OK;
    if (!elem_ok(in, e) || (!out && !quant)) return LCPP_ERR_INVALID_ARG;
    if (out && (!elem_ok(out, e) || !rows_apart(out_stride, rows, cols))) return LCPP_ERR_INVALID_ARG;
    if (!norm_pointer(weight, we, false) || !norm_pointer(rstd, 4, false)) return LCPP_ERR_INVALID_ARG;
    if (residual && (!elem_ok(residual, e) || !elem_ok(sum, e) || !rows_apart(sum_stride, rows, cols)))
        return LCPP_ERR_INVALID_ARG;
    if (!residual && sum) return LCPP_ERR_INVALID_ARG;
    const uint64_t groups = group ? ceil_div(cols, group) : 1;
    if (quant) {
        if (!elem_ok(scales, 4) || !rows_apart(quant_stride, rows, cols)) return LCPP_ERR_INVALID_ARG;
        // no two scales in one place, whichever dimension is the outer one
        const bool apart = (scale_group_stride >= 1 || groups == 1) && rows_apart(scale_row_stride, rows, 1);
        const bool outer_rows = rows == 1 || groups == 1 || scale_row_stride > (groups - 1) * scale_group_stride;
        const bool outer_groups = rows == 1 || groups == 1 || scale_group_stride > (rows - 1) * scale_row_stride;
        if (!apart || (!outer_rows && !outer_groups)) return LCPP_ERR_INVALID_ARG;
        // (8-bit rows would be written over inputs that other threads have yet to read)
        if (same_place(quant, in) || same_place(quant, residual)) return LCPP_ERR_INVALID_ARG;
    }
    if (same_place(sum, out) || same_place(sum, quant) || same_place(out, quant) || same_place(rstd, scales))
        return LCPP_ERR_INVALID_ARG;
    RmsArgs a = {};
    a.in = in, a.residual = residual, a.weight = weight;
    a.sum = sum, a.out = out, a.quant = quant;
    a.in_stride = in_stride, a.residual_stride = residual_stride, a.sum_stride = sum_stride;
    a.out_stride = out_stride, a.quant_stride = quant_stride;
    a.scales = quant ? scales : nullptr, a.rstd = rstd;
    a.scale_row = scale_row_stride, a.scale_col = scale_group_stride;
    a.rows = (uint32_t)rows, a.cols = (uint32_t)cols;
    a.group = quant ? group / kOctet : 0;
    for (uint32_t g = a.group; g > 1; g /= 2) ++a.log2_lanes;
    a.eps = eps;
    a.e5m2 = qt == LCPP_FLOAT8_E5M2;
    a.qmax = a.e5m2 ? 57344.0f : 448.0f;
    a.wide_weight = wt == LCPP_FLOAT32;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return float_dispatch(t, [&](auto x) -> int {
        using T = decltype(x);
        if (quant) return residual ? rms_forward_launch<T, true, true>(a, s) : rms_forward_launch<T, false, true>(a, s);
        return residual ? rms_forward_launch<T, true, false>(a, s) : rms_forward_launch<T, false, false>(a, s);
    });
}

extern "C" int lcpp_rms_norm_backward_temp_bytes(lcpp_dtype t, uint64_t rows, uint64_t cols, size_t *bytes)
{
    if (!bytes) return LCPP_ERR_INVALID_ARG;
    if (!float_size(t)) return LCPP_ERR_UNSUPPORTED_DTYPE;
    if (rows > kMaxRows || cols > kMaxCols) return LCPP_ERR_INVALID_ARG;
    *bytes = (size_t)rms_backward_temp(rows, cols);
    return LCPP_OK;
}

extern "C" int lcpp_rms_norm_backward(lcpp_dtype t, lcpp_dtype wt, void *temp, size_t temp_bytes, const void *grad_out,
                                      uint64_t grad_out_stride, const void *grad_sum, uint64_t grad_sum_stride,
                                      const void *in, uint64_t in_stride, const void *weight, const float *rstd,
                                      void *grad_in, uint64_t grad_in_stride, void *grad_weight, uint64_t rows,
                                      uint64_t cols, void *stream)
{
    const size_t e = float_size(t), we = float_size(wt);
    if (!e || !we || (wt != t && wt != LCPP_FLOAT32)) return LCPP_ERR_UNSUPPORTED_DTYPE;
    if (rows > kMaxRows || cols > kMaxCols) return LCPP_ERR_INVALID_ARG;
    if (cols == 0) return LCPP_OK;
    if (!norm_pointer(grad_weight, we, false)) return LCPP_ERR_INVALID_ARG;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (temp && temp_bytes >= kStatusBytes && reinterpret_cast<uintptr_t>(temp) % 256) return LCPP_ERR_INVALID_ARG;
    uint32_t *status = temp && temp_bytes >= kStatusBytes ? static_cast<uint32_t *>(temp) : nullptr;
    if (rows == 0) {
        // (no rows, no gradient of the weights)
        if (!grad_weight && !status) return LCPP_OK;
        const uint32_t n = grad_weight ? (uint32_t)cols : 0, grid = std::max(1u, std::min(4096u, (n + 255) / 256));
        if (we == 4) LCPP_LAUNCH("rms_norm_zero", s, rms_zero_kernel<float><<<grid, 256, 0, s>>>(static_cast<float *>(grad_weight), n, status));
        else LCPP_LAUNCH("rms_norm_zero", s, rms_zero_kernel<uint16_t><<<grid, 256, 0, s>>>(static_cast<uint16_t *>(grad_weight), n, status));
        LCPP_CHECK_LAUNCH();
        return LCPP_OK;
    }
    if (!elem_ok(grad_out, e) || !elem_ok(in, e) || !elem_ok(rstd, 4) || !elem_ok(grad_in, e)) return LCPP_ERR_INVALID_ARG;
    if (!norm_pointer(grad_sum, e, false) || !norm_pointer(weight, we, false)) return LCPP_ERR_INVALID_ARG;
    if (!rows_apart(grad_in_stride, rows, cols) || same_place(grad_in, grad_weight)) return LCPP_ERR_INVALID_ARG;
    if (grad_weight) {
        if (!temp) return LCPP_ERR_INVALID_ARG;
        if (temp_bytes < rms_backward_temp(rows, cols)) return LCPP_ERR_TEMP_TOO_SMALL;
    }
    RmsGradArgs a = {};
    a.grad_out = grad_out, a.grad_sum = grad_sum, a.in = in, a.weight = weight, a.grad_in = grad_in;
    a.go_stride = grad_out_stride, a.gs_stride = grad_sum_stride, a.in_stride = in_stride, a.gi_stride = grad_in_stride;
    a.rstd = rstd;
    a.partial = grad_weight ? reinterpret_cast<float *>(static_cast<char *>(temp) + kStatusBytes) : nullptr;
    a.status = status;
    a.rows = (uint32_t)rows, a.cols = (uint32_t)cols;
    a.wide_weight = wt == LCPP_FLOAT32;
    return float_dispatch(t, [&](auto x) -> int {
        using T = decltype(x);
        return grad_sum ? rms_backward_launch<T, true>(a, grad_weight, s) : rms_backward_launch<T, false>(a, grad_weight, s);
    });
}
