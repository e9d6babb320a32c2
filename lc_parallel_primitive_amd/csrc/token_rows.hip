// token_rows.hip — rows of tokens copied to the rows of their (token, choice) pairs, and
// the pairs' rows summed back, token by token; each with the weights' gradient.
//
//   spread   out[pos[t, j]] = w[t, j] in[t]            (pairs of position -1: nothing)
//   sum      out[t] = [residual[t] +] sum over j of w[t, j] in[pos[t, j]]
//   dots     d[t, j] = sum over columns of few[t] many[pos[t, j]]
//
// The gradient of a spread is a sum, that of a sum a spread, and the weights' gradients
// are the dots, made in the same pass over the same rows.  Sums run over j in order, in 32
// bits, and there are no atomics: the same bits at every call.
//
// Bound by memory.  A wave takes one token's chunk of 64 octets (one or two 16-byte
// accesses a lane and row), so the positions and weights are scalars and a pair without a
// row costs nothing; a token's row is read once for all its pairs.  Of rows of fewer
// octets a wave takes two to eight tokens at once.  With dots a token belongs to no more
// than one wave or to four.
// bfloat16: 8192 tokens x 4 rows of 2048 copied in 31.5 us and summed back in 31.7, 5.3
// TB/s; 16384 x 4 rows of 4096 summed with weights in 117 us, 5.8 TB/s, their gradients
// with the dots 241, 5.0; 8192 x 4 of 2048 summed with weights and the dots in 34.6, 5.8 (float32
// 79, 5.1); 37 x 8 rows of 2048 float16 in 4.5, the launch and two loads one after the other.
#include <algorithm>

#include "tensor.hpp"

namespace lcpp {
namespace {

constexpr int kRowThreads = 256, kRowWaves = kRowThreads / kWave;
constexpr uint64_t kMaxRowGroups = 1u << 20;
constexpr int kBatch = 8;  // pairs of a token whose rows are on their way at once

struct TokenArgs {
    const void *few, *many, *residual;  // [token], [pair], [token]
    void *few_out, *many_out;
    uint64_t few_stride, many_stride, residual_stride, few_out_stride, many_out_stride;
    const int32_t *positions;
    const float *weights;
    float *dots;
    uint64_t tokens, many_rows;
    uint32_t choices, cols, chunks;
};

// The eight columns that a lane works on: at the row's end the octet is moved back to lie
// inside the row, and only its columns from `lo` on are the lane's.
struct Place {
    uint32_t col, lo, hi;
    bool active;
};
__device__ __forceinline__ Place octet_place(uint32_t octet, uint32_t cols)
{
    Place p;
    p.col = octet * kOctet, p.lo = 0, p.hi = kOctet;
    p.active = p.col < cols;
    if (p.active && p.col + kOctet > cols) {
        if (cols >= kOctet) {
            p.lo = p.col + kOctet - cols;
            p.col = cols - kOctet;
        } else {
            p.hi = cols;  // (a row of less than eight columns)
        }
    }
    return p;
}
template <class T>
__device__ __forceinline__ Octet<T> load_place(const T *row, const Place &p)
{
    return p.hi == kOctet ? load_pack<kOctet>(row + p.col) : load_pack_part<kOctet>(row, (int)p.hi);
}
template <class T>
__device__ __forceinline__ void store_place(T *row, const Place &p, const float (&x)[kOctet])
{
    if (p.lo == 0 && p.hi == kOctet) {
        // (two accesses of a 4-byte type's octet meet in the L2: 8192 tokens x 4 x 2048 with weights 118 us past it, 70 so)
        if constexpr (sizeof(T) == 4) store_pack<kOctet>(row + p.col, x);
        else store_pack_nt<kOctet>(row + p.col, x);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < kOctet; ++i)
            if (i >= p.lo && i < p.hi) row[p.col + i] = (T)x[i];
    }
}

// The pairs first .. first + kBatch of a token: their rows (-1: none) and weights, the same
// in all lanes where LT, the lanes of a token, are a wave.
struct Pairs {
    int64_t row[kBatch];
    float w[kBatch];
};
template <int LT>
__device__ __forceinline__ Pairs token_pairs(const TokenArgs &a, uint64_t token, uint32_t first)
{
    Pairs p;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
        p.row[j] = -1;
        p.w[j] = 1.0f;
        if (first + j >= a.choices) continue;
        const uint64_t at = token * a.choices + first + j;
        int32_t row = a.positions[at];
        if constexpr (LT == kWave) row = __builtin_amdgcn_readfirstlane(row);
        if (row >= 0 && (uint64_t)row < a.many_rows) p.row[j] = row;
        if (a.weights) p.w[j] = a.weights[at];
    }
    return p;
}

// ---------------------------------------------------------------- without dots
// What a wave works on: a chunk of one token's row, or, with fewer lanes LT for a token,
// the whole rows of several.
template <int LT>
struct Items {
    uint64_t at;
    __device__ __forceinline__ Items(const TokenArgs &)
        : at((uint64_t)blockIdx.x * kRowWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave))
    {
    }
    __device__ __forceinline__ bool more(const TokenArgs &a) const
    {
        return LT == kWave ? at < a.tokens * a.chunks : at * (kWave / LT) < a.tokens;
    }
    __device__ __forceinline__ void next() { at += (uint64_t)gridDim.x * kRowWaves; }
    __device__ __forceinline__ uint64_t token(const TokenArgs &a) const
    {
        return LT == kWave ? at / a.chunks : at * (kWave / LT) + lane_id() / LT;
    }
    // the lane's part of the row, in octets or vectors
    __device__ __forceinline__ uint32_t part(const TokenArgs &a, uint64_t token) const
    {
        return LT == kWave ? (uint32_t)(at - token * a.chunks) * kWave + lane_id() : lane_id() % LT;
    }
};

template <class T, int LT>
__global__ __launch_bounds__(kRowThreads) void token_sum_kernel(TokenArgs a)
{
    Items<LT> item(a);
    for (; item.more(a); item.next()) {
        const uint64_t token = item.token(a);
        const Place at = octet_place(item.part(a, token), token < a.tokens ? a.cols : 0);
        float acc[kOctet] = {};
        if (a.residual && at.active) {
            const Octet<T> r = load_place(static_cast<const T *>(a.residual) + token * a.residual_stride, at);
#pragma unroll
            for (int i = 0; i < kOctet; ++i) acc[i] = r[i];
        }
        for (uint32_t first = 0; first < a.choices; first += kBatch) {
            if (LT < kWave && !at.active) continue;
            const Pairs p = token_pairs<LT>(a, token, first);
            if (!at.active) continue;
            Octet<T> x[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
                if (p.row[j] >= 0) x[j] = load_place(static_cast<const T *>(a.many) + p.row[j] * a.many_stride, at);
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
                if (p.row[j] >= 0)
#pragma unroll
                    for (int i = 0; i < kOctet; ++i) acc[i] += p.w[j] * x[j][i];
        }
        if (at.active) store_place(static_cast<T *>(a.few_out) + token * a.few_out_stride, at, acc);
    }
}

template <class T, int LT>
__global__ __launch_bounds__(kRowThreads) void token_spread_kernel(TokenArgs a)
{
    Items<LT> item(a);
    for (; item.more(a); item.next()) {
        const uint64_t token = item.token(a);
        const Place at = octet_place(item.part(a, token), token < a.tokens ? a.cols : 0);
        Octet<T> x;
        if (at.active) x = load_place(static_cast<const T *>(a.few) + token * a.few_stride, at);
        for (uint32_t first = 0; first < a.choices; first += kBatch) {
            if (LT < kWave && !at.active) continue;
            const Pairs p = token_pairs<LT>(a, token, first);
            if (!at.active) continue;
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                if (p.row[j] < 0) continue;
                float y[kOctet];
#pragma unroll
                for (int i = 0; i < kOctet; ++i) y[i] = p.w[j] * x[i];
                store_place(static_cast<T *>(a.many_out) + p.row[j] * a.many_out_stride, at, y);
            }
        }
    }
}

// Rows of any type as they are: V elements of U a lane, 16 bytes.
template <class U, int LT>
__global__ __launch_bounds__(kRowThreads) void token_copy_kernel(TokenArgs a)
{
    constexpr uint32_t V = 16 / sizeof(U);
    typedef U vec __attribute__((ext_vector_type(V)));
    typedef vec vec_u __attribute__((aligned(sizeof(U))));
    Items<LT> item(a);
    for (; item.more(a); item.next()) {
        const uint64_t token = item.token(a);
        uint32_t col = item.part(a, token) * V;
        const bool active = col < a.cols && token < a.tokens, whole = a.cols >= V;
        if (active && whole && col + V > a.cols) col = a.cols - V;  // (copied twice, the same values)
        const U *in = static_cast<const U *>(a.few) + token * a.few_stride + col;
        vec x = {};
        if (active) {
            if (whole) x = *reinterpret_cast<const vec_u *>(in);
            else
#pragma unroll
                for (uint32_t i = 0; i < V; ++i)
                    if (i < a.cols) x[i] = in[i];
        }
        for (uint32_t first = 0; first < a.choices; first += kBatch) {
            if (LT < kWave && !active) continue;
            const Pairs p = token_pairs<LT>(a, token, first);
            if (!active) continue;
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                if (p.row[j] < 0) continue;
                U *out = static_cast<U *>(a.many_out) + p.row[j] * a.many_out_stride + col;
                if (whole) __builtin_nontemporal_store(x, reinterpret_cast<vec_u *>(out));
                else
#pragma unroll
                    for (uint32_t i = 0; i < V; ++i)
                        if (i < a.cols) out[i] = x[i];
            }
        }
    }
}

// ---------------------------------------------------------------- with dots
// Sum over the LT lanes of a token, in each of them (LT 8 to 64).
template <int LT>
__device__ __forceinline__ float lanes_total(float x)
{
    if constexpr (LT == kWave) return wave_reduce_dpp(x, SumOp());
    x += dpp_perm<kDppQuadXor1>(x);
    x += dpp_perm<kDppQuadXor2>(x);
    x += dpp_perm<kDppRowHalfMirror>(x);
    if constexpr (LT > 8) x += dpp_perm<kDppRowMirror>(x);
    if constexpr (LT > 16) x += shfl_xor(x, 16);
    return x;
}
// NT threads (8 to 256) for a token, B batches of its pairs at a time, so that the sums of their dots
// stay in registers while its columns are gone through.  SPREAD: many_out[pos] = w few as
// well (where it is wanted), else few_out = sum of w many, of all pairs at once.
template <class T, int NT, int B, bool SPREAD>
__global__ __launch_bounds__(kRowThreads) void token_dots_kernel(TokenArgs a)
{
    constexpr int RG = kRowThreads / NT, GW = NT > kWave ? NT / kWave : 1, LT = NT < kWave ? NT : kWave;
    __shared__ float lds[2][kRowThreads / LT][B * kBatch];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t t = threadIdx.x % NT, group = NT < kWave ? threadIdx.x / NT : wave / GW;
    const uint32_t part = NT < kWave ? group : wave;  // of the workgroup, that sums its dots
    const uint32_t octets = (a.cols + kOctet - 1) / kOctet;
    int slot = 0;
    auto some_pairs = [&](uint64_t token, uint32_t first) {
        const bool live = token < a.tokens;
        float dot[B][kBatch] = {};
        if (live)
            for (uint32_t octet = t; octet < octets; octet += NT) {
                const Place at = octet_place(octet, a.cols);
                const Octet<T> x = load_place(static_cast<const T *>(a.few) + token * a.few_stride, at);
                float acc[kOctet] = {};
#pragma unroll
                for (int b = 0; b < B; ++b) {
                    const Pairs p = token_pairs<LT>(a, token, first + b * kBatch);
                    Octet<T> y[kBatch];
#pragma unroll
                    for (int j = 0; j < kBatch; ++j)
                        if (p.row[j] >= 0) y[j] = load_place(static_cast<const T *>(a.many) + p.row[j] * a.many_stride, at);
#pragma unroll
                    for (int j = 0; j < kBatch; ++j) {
                        if (p.row[j] < 0) continue;
#pragma unroll
                        for (uint32_t i = 0; i < kOctet; ++i)
                            if (i >= at.lo) dot[b][j] += x[i] * y[j][i];
                        if constexpr (SPREAD) {
                            if (!a.many_out) continue;
                            float v[kOctet];
#pragma unroll
                            for (int i = 0; i < kOctet; ++i) v[i] = p.w[j] * x[i];
                            store_place(static_cast<T *>(a.many_out) + p.row[j] * a.many_out_stride, at, v);
                        } else {
#pragma unroll
                            for (int i = 0; i < kOctet; ++i) acc[i] += p.w[j] * y[j][i];
                        }
                    }
                }
                if constexpr (!SPREAD) store_place(static_cast<T *>(a.few_out) + token * a.few_out_stride, at, acc);
            }
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
            for (int j = 0; j < kBatch; ++j) dot[b][j] = lanes_total<LT>(dot[b][j]);
        if (lane_id() % LT == 0)
#pragma unroll
            for (int b = 0; b < B; ++b)
#pragma unroll
                for (int j = 0; j < kBatch; ++j) lds[slot][part][b * kBatch + j] = dot[b][j];
        if constexpr (GW > 1) __syncthreads();
        else wave_lds_sync();
        for (uint32_t j = t; j < B * kBatch; j += NT) {
            if (!live || first + j >= a.choices) break;
            float d = 0.0f;
#pragma unroll
            for (int w = 0; w < GW; ++w) d += lds[slot][group * GW + w][j];
            a.dots[token * a.choices + first + j] = d;
        }
        slot ^= 1;
    };
    // (the workgroup's tokens make the same number of rounds: they share barriers)
    for (uint64_t base = (uint64_t)blockIdx.x * RG; base < a.tokens; base += (uint64_t)gridDim.x * RG) {
        if constexpr (SPREAD) {
            for (uint32_t first = 0; first < a.choices; first += B * kBatch) some_pairs(base + group, first);
        } else {
            some_pairs(base + group, 0);
        }
    }
}

size_t row_elem_size(lcpp_dtype t)
{
    switch (t) {
    case LCPP_INT32:
    case LCPP_UINT32:
    case LCPP_FLOAT32: return 4;
    case LCPP_BFLOAT16:
    case LCPP_FLOAT16: return 2;
    case LCPP_FLOAT8_E4M3:
    case LCPP_FLOAT8_E5M2: return 1;
    default: return 0;
    }
}
constexpr uint64_t kSumDots = 2 * kBatch;   // pairs whose sum and dots are made in one pass
constexpr uint64_t kMaxPairs = 8 * kBatch;  // of a token
bool row_sizes(uint64_t tokens, uint64_t choices, uint64_t cols, uint64_t rows)
{
    return tokens <= 0x7FFFFFFFull && choices <= kMaxPairs && tokens * choices <= 0x7FFFFFFFull && cols <= kMaxCols && rows <= 0x7FFFFFFFull;
}
uint32_t row_grid(uint64_t items, int each) { return (uint32_t)std::min(ceil_div(items, each), kMaxRowGroups); }
bool pointer_or_null(const void *p, size_t size) { return !p || elem_ok(p, size); }

// f(lanes) as an integral constant: as few as hold a token's row of so many parts, 8 to 64.
template <class F>
int lanes_of(uint64_t parts, F f)
{
    if (parts <= 8) return f(std::integral_constant<int, 8>{});
    if (parts <= 16) return f(std::integral_constant<int, 16>{});
    if (parts <= 32) return f(std::integral_constant<int, 32>{});
    return f(std::integral_constant<int, 64>{});
}
// A token in one wave or less where its columns are few, else in four.
template <class T, int B, bool SPREAD>
int dots_launch_of(const TokenArgs &a, const char *name, hipStream_t s)
{
    const uint64_t octets = ceil_div(a.cols, kOctet);
    if (octets > 128) {
        LCPP_LAUNCH(name, s, token_dots_kernel<T, kRowThreads, B, SPREAD><<<row_grid(a.tokens, 1), kRowThreads, 0, s>>>(a));
        LCPP_CHECK_LAUNCH();
        return LCPP_OK;
    }
    return lanes_of(octets, [&](auto lanes) -> int {
        constexpr int LT = decltype(lanes)::value;
        LCPP_LAUNCH(name, s,
                    token_dots_kernel<T, LT, B, SPREAD><<<row_grid(a.tokens, kRowThreads / LT), kRowThreads, 0, s>>>(a));
        LCPP_CHECK_LAUNCH();
        return LCPP_OK;
    });
}
template <bool SPREAD>
int dots_launch(lcpp_dtype t, const TokenArgs &a, const char *name, hipStream_t s)
{
    return float_dispatch(t, [&](auto x) -> int {
        using T = decltype(x);
        return a.choices <= kBatch ? dots_launch_of<T, 1, SPREAD>(a, name, s) : dots_launch_of<T, 2, SPREAD>(a, name, s);
    });
}

}  // namespace
}  // namespace lcpp

using namespace lcpp;

extern "C" int lcpp_token_spread(lcpp_dtype t, const void *in, uint64_t in_stride, const int32_t *positions,
                                 const float *weights, void *out, uint64_t out_stride, const void *other,
                                 uint64_t other_stride, float *dots, uint64_t rows, uint64_t tokens, uint64_t choices,
                                 uint64_t cols, void *stream)
{
    const size_t e = row_elem_size(t);
    if (!e || ((weights || dots) && !float_size(t))) return LCPP_ERR_UNSUPPORTED_DTYPE;
    if (!row_sizes(tokens, choices, cols, rows)) return LCPP_ERR_INVALID_ARG;
    if (tokens == 0 || choices == 0 || (!dots && (cols == 0 || rows == 0))) return LCPP_OK;
    if (!elem_ok(positions, 4) || !pointer_or_null(weights, 4) || !pointer_or_null(dots, 4) || (!out && !dots)) return LCPP_ERR_INVALID_ARG;
    if (cols && (!elem_ok(in, e) || !pointer_or_null(out, e) || (out && !rows_apart(out_stride, rows, cols)))) return LCPP_ERR_INVALID_ARG;
    if (cols && dots && rows && !elem_ok(other, e)) return LCPP_ERR_INVALID_ARG;
    if (same_place(out, dots) || same_place(out, in)) return LCPP_ERR_INVALID_ARG;
    TokenArgs a = {};
    a.few = in, a.few_stride = in_stride, a.many_out = out, a.many_out_stride = out_stride;
    a.many = other, a.many_stride = other_stride, a.dots = dots;
    a.positions = positions, a.weights = weights;
    a.tokens = tokens, a.many_rows = rows, a.choices = (uint32_t)choices, a.cols = (uint32_t)cols;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dots) return dots_launch<true>(t, a, "token_spread_dots", s);
    if (weights)
        return float_dispatch(t, [&](auto x) -> int {
            using T = decltype(x);
            return lanes_of(ceil_div(cols, kOctet), [&](auto lanes) -> int {
                constexpr int LT = decltype(lanes)::value;
                a.chunks = (uint32_t)ceil_div(cols, LT * kOctet);
                LCPP_LAUNCH("token_spread", s,
                            token_spread_kernel<T, LT>
                            <<<row_grid(tokens * a.chunks, kRowThreads / LT), kRowThreads, 0, s>>>(a));
                LCPP_CHECK_LAUNCH();
                return LCPP_OK;
            });
        });
    return lanes_of(ceil_div(cols, 16 / e), [&](auto lanes) -> int {
        constexpr int LT = decltype(lanes)::value;
        a.chunks = (uint32_t)ceil_div(cols, LT * 16 / e);
        const uint32_t grid = row_grid(tokens * a.chunks, kRowThreads / LT);
        if (e == 4) LCPP_LAUNCH("token_copy", s, token_copy_kernel<uint32_t, LT><<<grid, kRowThreads, 0, s>>>(a));
        else if (e == 2) LCPP_LAUNCH("token_copy", s, token_copy_kernel<uint16_t, LT><<<grid, kRowThreads, 0, s>>>(a));
        else LCPP_LAUNCH("token_copy", s, token_copy_kernel<uint8_t, LT><<<grid, kRowThreads, 0, s>>>(a));
        LCPP_CHECK_LAUNCH();
        return LCPP_OK;
    });
}

extern "C" int lcpp_token_sum(lcpp_dtype t, const void *in, uint64_t in_stride, uint64_t rows, const int32_t *positions,
                              const float *weights, const void *residual, uint64_t residual_stride, void *out,
                              uint64_t out_stride, const void *other, uint64_t other_stride, float *dots, uint64_t tokens,
                              uint64_t choices, uint64_t cols, void *stream)
{
    const size_t e = float_size(t);
    if (!e) return LCPP_ERR_UNSUPPORTED_DTYPE;
    if (!row_sizes(tokens, choices, cols, rows)) return LCPP_ERR_INVALID_ARG;
    if (residual && dots) return LCPP_ERR_INVALID_ARG;  // (no gradient needs both)
    if (tokens == 0 || (cols == 0 && !dots)) return LCPP_OK;
    if (choices && (!elem_ok(positions, 4) || !pointer_or_null(weights, 4) || !pointer_or_null(dots, 4))) return LCPP_ERR_INVALID_ARG;
    if (cols && (!elem_ok(out, e) || !pointer_or_null(residual, e) || !rows_apart(out_stride, tokens, cols))) return LCPP_ERR_INVALID_ARG;
    if (cols && rows && choices && !elem_ok(in, e)) return LCPP_ERR_INVALID_ARG;
    if (cols && dots && !elem_ok(other, e)) return LCPP_ERR_INVALID_ARG;
    if (same_place(out, dots) || same_place(out, in)) return LCPP_ERR_INVALID_ARG;
    TokenArgs a = {};
    a.many = in, a.many_stride = in_stride, a.many_rows = rows;
    a.residual = residual, a.residual_stride = residual_stride;
    a.few_out = out, a.few_out_stride = out_stride;
    a.few = other, a.few_stride = other_stride, a.dots = dots;
    a.positions = positions, a.weights = weights;
    a.tokens = tokens, a.choices = (uint32_t)choices, a.cols = (uint32_t)cols;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dots && choices && choices <= kSumDots) return dots_launch<false>(t, a, "token_sum_dots", s);
    if (dots && choices) {
        // (more dots than registers hold: a pass of their own over the same rows)
        const int status = dots_launch<true>(t, a, "token_dots", s);
        if (status || cols == 0) return status;
    }
    return float_dispatch(t, [&](auto x) -> int {
        using T = decltype(x);
        return lanes_of(ceil_div(cols, kOctet), [&](auto lanes) -> int {
            constexpr int LT = decltype(lanes)::value;
            a.chunks = (uint32_t)ceil_div(cols, LT * kOctet);
            LCPP_LAUNCH("token_sum", s,
                        token_sum_kernel<T, LT><<<row_grid(tokens * a.chunks, kRowThreads / LT), kRowThreads, 0, s>>>(a));
            LCPP_CHECK_LAUNCH();
            return LCPP_OK;
        });
    });
}
