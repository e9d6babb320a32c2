// expert_product.hip — the products of each expert's rows with its own matrix, and their
// gradients, on the matrix cores.
//
// Rows offsets[e] .. offsets[e + 1] belong to expert e, whose matrix W has a row for each
// output.  Every one of the three products is O[m][n] = sum over c of R(m, c) L(n, c):
//
//   forward     y[r][o]  = sum over i of x[r][i] W[o][i]     m = row,    n = output, c = input
//   grad rows   dx[r][i] = sum over o of dy[r][o] W[o][i]    m = row,    n = input,  c = output
//   grad matrix dW[o][i] = sum over r of dy[r][o] x[r][i]    m = output, n = input,  c = row
//
// L is the left operand of a 32 x 32 matrix instruction and R the right one, so that a lane
// ends up with four neighbouring n of one m and stores them at once.  An operand lies in
// memory either with c along its rows (x and W forward, dy) or across them (W and x and dy
// of a grad matrix); either way it is staged in LDS as it lies, by loads that go there
// directly, 128 bytes of c deep, twice: one stage is on its way while the other is
// multiplied, with one barrier a stage.  Operands with c across are read through the LDS'
// transposing loads.  16-byte chunks are permuted inside rows so that the 64 lanes of a read
// meet all banks evenly.
//
// 8-bit operands have a scale for each row's 128 inputs and for 128 outputs x 128 inputs of
// a matrix: a stage is 128 inputs deep, its product is made from 0 and then added to the
// sums in 32 bits, times both scales.
#include <algorithm>

#include "tensor.hpp"

namespace lcpp {
namespace {

struct fp8 {
    uint8_t v;
};

enum class Product { kForward, kGradRows, kGradMatrix };

struct ProductArgs {
    const void *r, *l;        // operands
    void *o;
    uint64_t r_stride, l_stride, o_stride;  // of their rows, in elements
    uint64_t l_expert, o_expert;            // from one expert's matrix to the next (l of forward and grad rows, o of grad matrix)
    const int32_t *offsets;
    uint64_t rows;            // of the tensors
    uint32_t experts, m, n, c;  // sizes that are no expert's (m of grad matrix; c of the others)
    const float *r_scales, *l_scales;
    uint64_t r_scale_row, r_scale_col, l_scale_expert;
    uint32_t l_scale_row;
};

constexpr uint32_t kChunk = 16;         // bytes
constexpr uint32_t kStageBytes = 128;   // of c
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------- loads to LDS
// 16 bytes for each lane, from base + voff (0 where voff is outside) to lds + 16 lane.  In
// assembly because the compiler takes every later read of LDS to wait for it; what reads
// the stage waits explicitly (stage_barrier).
constexpr uint32_t kOutside = 0xFFFFFF00u;
__device__ __forceinline__ void load_to_lds(u32x4 rsrc, uint32_t voff, uint32_t lds)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc) : "memory");
}
__device__ __forceinline__ u32x4 stage_rsrc(const void *p)
{
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    u32x4 r;
    r.x = __builtin_amdgcn_readfirstlane((uint32_t)a);
    r.y = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xFFFFu);
    r.z = 0x7FFFFFFFu;
    r.w = (uint32_t)kRawBufferWord3;
    return r;
}
// Every wave's loads to LDS have arrived, and every wave has read what it needed before.
__device__ __forceinline__ void stage_barrier()
{
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// ---------------------------------------------------------------- an operand's stage
// X elements (rows or columns of the operand) x 128 bytes of c.  ACROSS: c runs from row to
// row, X columns in each; else X rows with c along them.
template <class T, uint32_t X, uint32_t THREADS, bool ACROSS>
struct Stage {
    static constexpr uint32_t kElems = kChunk / sizeof(T);         // of a chunk
    static constexpr uint32_t kDepth = kStageBytes / sizeof(T);    // of c
    static constexpr uint32_t kRowChunks = ACROSS ? X / kElems : kStageBytes / kChunk;
    static constexpr uint32_t kBytes = X * kStageBytes;
    static constexpr uint32_t kLoads = kBytes / kChunk / THREADS;  // of a thread
    static_assert(kBytes % (kChunk * THREADS) == 0, "whole loads");
    // where chunk c of a row is kept
    static __device__ __forceinline__ uint32_t swizzle(uint32_t row) { return ACROSS ? (row & 3) << 2 : (row >> 1) & 7; }

    const T *base;     // of the tile
    uint64_t stride;   // of rows, in elements
    uint32_t valid;    // of X
    uint32_t depth;    // of c in all
    uint32_t row[kLoads], chunk[kLoads], off[kLoads];

    __device__ __forceinline__ Stage(const T *p, uint64_t s, uint32_t x, uint32_t c) : base(p), stride(s), valid(x), depth(c)
    {
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            const uint32_t slot = i * THREADS + threadIdx.x;
            row[i] = slot / kRowChunks;
            chunk[i] = (slot % kRowChunks) ^ swizzle(row[i]);
            if constexpr (ACROSS) {
                off[i] = chunk[i] * kElems < valid ? (uint32_t)(row[i] * stride * sizeof(T)) + chunk[i] * kChunk : kOutside;
            } else {
                // (rows past the last one are the last one again, and are not stored)
                const uint32_t r = row[i] < valid ? row[i] : valid - 1;
                off[i] = (uint32_t)(r * stride * sizeof(T)) + chunk[i] * kChunk;
            }
        }
    }
    // The stage from c = from on, all of whose chunks are aligned and whole.
    __device__ __forceinline__ void issue(uint32_t from, uint32_t lds) const
    {
        const u32x4 rsrc = stage_rsrc(base + (ACROSS ? from * stride : from));
        const bool last = from + kDepth > depth;
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            uint32_t v = off[i];
            if (last && from + (ACROSS ? row[i] : chunk[i] * kElems) >= depth) v = kOutside;
            load_to_lds(rsrc, v, lds + (i * THREADS + wave * kWave) * kChunk);
        }
    }
    // The same by way of registers, for any stride, size and alignment.
    struct Held {
        u32x4 v[kLoads];
    };
    __device__ __forceinline__ void fetch(uint32_t from, Held &h) const
    {
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            const uint32_t c = from + (ACROSS ? row[i] : chunk[i] * kElems);
            const uint32_t r = ACROSS ? 0 : row[i] < valid ? row[i] : valid - 1;
            const uint32_t inside = ACROSS ? valid : depth, at = ACROSS ? chunk[i] * kElems : c;
            const bool there = c < depth && at < inside;
            const T *p = base + (ACROSS ? c * stride + at : r * stride + c);
            typedef T vec __attribute__((ext_vector_type(kElems)));
            typedef vec vec_u __attribute__((aligned(sizeof(T))));
            vec v = {};
            if (there && at + kElems <= inside) {
                v = *reinterpret_cast<const vec_u *>(p);
            } else if (there) {
#pragma unroll
                for (uint32_t j = 0; j < kElems; ++j)
                    if (at + j < inside) v[j] = p[j];
            }
            __builtin_memcpy(&h.v[i], &v, sizeof(v));
        }
    }
    __device__ __forceinline__ void put(const Held &h, char *lds) const
    {
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i)
            *reinterpret_cast<u32x4 *>(lds + (i * THREADS + threadIdx.x) * kChunk) = h.v[i];
    }

    // A lane's part of step k for the 32 elements from x on: 32 bytes of c (8-bit), 16 (16-bit)
    // or 4 values one instruction apart (32-bit); the order of c within a stage is the
    // same for both operands.
    static __device__ __forceinline__ u32x4 along(const char *lds, uint32_t x, uint32_t chunk)
    {
        const uint32_t r = x + lane_id() % 32;
        return *reinterpret_cast<const u32x4 *>(lds + r * kStageBytes + ((chunk ^ swizzle(r)) * kChunk));
    }
    static __device__ __forceinline__ uint32_t across_at(uint32_t row, uint32_t col)
    {
        const uint32_t byte = col * (uint32_t)sizeof(T);
        return row * (X * (uint32_t)sizeof(T)) + ((byte / kChunk ^ swizzle(row)) * kChunk) + byte % kChunk;
    }
    static __device__ __forceinline__ u32x4 fragment(const char *lds, uint32_t x, uint32_t k)
    {
        const uint32_t lane = lane_id();
        if constexpr (!ACROSS) {
            return along(lds, x, k * 2 + lane / 32);
        } else if constexpr (sizeof(T) == 2) {
            // 16 lanes give the places of 4 rows x 16 columns and get 4 rows of one column each
            u32x4 v;
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                const uint32_t row = k * 16 + lane / 32 * 8 + h * 4 + lane % 16 / 4;
                const uint32_t at = across_at(row, x + lane % 32 / 16 * 16 + lane % 4 * 4);
                typedef __attribute__((address_space(3))) s16x4 *place;
                const s16x4 q = __builtin_amdgcn_ds_read_tr16_b64_v4i16((place)(lds + at));
                uint2 w;
                __builtin_memcpy(&w, &q, 8);
                v[2 * h] = w.x, v[2 * h + 1] = w.y;
            }
            return v;
        } else {
            u32x4 v;
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
                v[j] = *reinterpret_cast<const uint32_t *>(lds + across_at(k * 8 + lane / 32 * 4 + j, x + lane % 32));
            return v;
        }
    }
};

__device__ __forceinline__ f32x16 multiply(u32x4 l, u32x4 r, f32x16 acc, bf16)
{
    typedef bf16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, l), __builtin_bit_cast(v8, r), acc, 0, 0, 0);
}
__device__ __forceinline__ f32x16 multiply(u32x4 l, u32x4 r, f32x16 acc, f16)
{
    typedef f16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, l), __builtin_bit_cast(v8, r), acc, 0, 0, 0);
}
__device__ __forceinline__ f32x16 multiply(u32x4 l, u32x4 r, f32x16 acc, float)
{
    typedef float v4 __attribute__((ext_vector_type(4)));
    const v4 a = __builtin_bit_cast(v4, l), b = __builtin_bit_cast(v4, r);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], acc, 0, 0, 0);
    return acc;
}

// ---------------------------------------------------------------- tiles
// The tile of a workgroup.  Those of one expert lie one behind the other, m fastest; each
// XCD, which get the workgroups in turn, works on neighbouring ones, which share operands in
// its L2.
struct Tile {
    uint32_t expert, m, n;  // numbers of the tile's first row and column, in tiles
    int64_t first;          // the expert's rows
    uint32_t count;
};
template <Product P>
__device__ __forceinline__ bool find_tile(const ProductArgs &a, uint32_t tm, uint32_t tn, Tile &t)
{
    const uint32_t nt = (a.n + tn - 1) / tn;
    constexpr uint32_t kXcds = 8;
    const uint32_t lane = lane_id();
    auto span = [&](uint32_t e, int64_t &first, uint32_t &count) {
        int64_t b = a.offsets[e], z = a.offsets[e + 1];
        b = b < 0 ? 0 : b;
        z = z > (int64_t)a.rows ? (int64_t)a.rows : z;
        first = b;
        count = z > b ? (uint32_t)(z - b) : 0;
    };
    uint32_t all = 0, id = blockIdx.x;
    if constexpr (P == Product::kGradMatrix) {
        const uint32_t mt = (a.m + tm - 1) / tm, each = mt * nt;
        const uint32_t per = (a.experts * each + kXcds - 1) / kXcds;
        id = id % kXcds * per + id / kXcds;
        if (blockIdx.x / kXcds >= per || id >= a.experts * each) return false;
        t.expert = id / each;
        const uint32_t in = id - t.expert * each;
        t.n = in / mt;
        t.m = in - t.n * mt;
        span(t.expert, t.first, t.count);
        return true;
    }
    for (uint32_t e = 0; e < a.experts; e += kWave) {
        int64_t first;
        uint32_t count = 0;
        if (e + lane < a.experts) span(e + lane, first, count);
        all += wave_reduce_dpp((count + tm - 1) / tm, SumOp());
    }
    const uint32_t per = (all * nt + kXcds - 1) / kXcds;
    id = id % kXcds * per + id / kXcds;
    if (blockIdx.x / kXcds >= per || id >= all * nt) return false;
    uint32_t before = 0;
    for (uint32_t e = 0; e < a.experts; e += kWave) {
        int64_t first = 0;
        uint32_t count = 0;
        if (e + lane < a.experts) span(e + lane, first, count);
        const uint32_t tiles = (count + tm - 1) / tm;
        const uint32_t sum = wave_inclusive_scan(tiles, SumOp());
        const uint64_t past = ballot((before + sum) * nt > id);
        if (past) {
            const int at = __builtin_ctzll(past);
            t.expert = e + at;
            t.first = read_lane(first, at);
            t.count = read_lane(count, at);
            const uint32_t mt = read_lane(tiles, at), in = id - (before + read_lane(sum, at) - mt) * nt;
            t.n = in / mt;
            t.m = in - t.n * mt;
            return true;
        }
        before += read_lane(sum, kWave - 1);
    }
    return false;
}

template <class T, class O>
__device__ __forceinline__ void store_four(O *row, uint32_t col, uint32_t cols, const float (&x)[4])
{
    if (col + 4 <= cols) store_pack<4>(row + col, x);
    else
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (col + i < cols) row[col + i] = (O)x[i];
}

// A workgroup of WM x WN waves makes TM x TN outputs.  ALIGNED: chunks are whole and aligned.
template <class T, class O, Product P, int TM, int TN, int WM, int WN, bool ALIGNED>
__global__ __launch_bounds__(WM *WN *kWave) void product_kernel(ProductArgs a)
{
    constexpr uint32_t THREADS = WM * WN * kWave;
    constexpr int FM = TM / WM / 32, FN = TN / WN / 32;
    constexpr bool kQuant = std::is_same_v<T, fp8>;
    using E = std::conditional_t<kQuant, uint8_t, T>;
    constexpr bool kLeftAcross = P != Product::kForward, kRightAcross = P == Product::kGradMatrix;
    using Left = Stage<E, TN, THREADS, kLeftAcross>;
    using Right = Stage<E, TM, THREADS, kRightAcross>;
    constexpr uint32_t kBytes = Left::kBytes + Right::kBytes;
    __shared__ __attribute__((aligned(256))) char lds[2 * kBytes];

    Tile t;
    if (!find_tile<P>(a, TM, TN, t)) return;
    const uint32_t m0 = t.m * TM, n0 = t.n * TN;
    const uint32_t rows = P == Product::kGradMatrix ? a.m : t.count;  // of the output
    const uint32_t depth = P == Product::kGradMatrix ? t.count : a.c;
    const E *lp = static_cast<const E *>(a.l), *rp = static_cast<const E *>(a.r);
    if constexpr (P == Product::kForward) lp += t.expert * a.l_expert + n0 * a.l_stride;
    else if constexpr (P == Product::kGradRows) lp += t.expert * a.l_expert + n0;
    else lp += t.first * a.l_stride + n0;
    if constexpr (P == Product::kGradMatrix) rp += t.first * a.r_stride + m0;
    else rp += (t.first + m0) * a.r_stride;
    const Left left(lp, a.l_stride, a.n - n0, depth);
    const Right right(rp, a.r_stride, rows - m0, depth);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id();
    const uint32_t wm = wave % WM * (TM / WM), wn = wave / WM * (TN / WN);

    f32x16 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = f32x16{};

    const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)lds);
    const uint32_t stages = (depth + Left::kDepth - 1) / Left::kDepth;
    typename Left::Held held_l;
    typename Right::Held held_r;
    // scales: of the lane's rows of m and of the wave's block of n
    float scale_m[FM], scale_n = 0.0f;
    auto scales = [&](uint32_t s) {
        if constexpr (kQuant) {
#pragma unroll
            for (int j = 0; j < FM; ++j) {
                const uint32_t m = m0 + wm + j * 32 + lane % 32;
                scale_m[j] = a.r_scales[(t.first + (m < rows ? m : rows - 1)) * a.r_scale_row + s * a.r_scale_col];
            }
            const uint32_t n = n0 + wn < a.n ? n0 + wn : a.n - 1;
            scale_n = a.l_scales[t.expert * a.l_scale_expert + (uint64_t)(n / 128) * a.l_scale_row + s];
        }
    };
    auto begin = [&](uint32_t s) {
        if constexpr (ALIGNED) {
            const uint32_t at = lds0 + (s & 1) * kBytes;
            left.issue(s * Left::kDepth, at);
            right.issue(s * Left::kDepth, at + Left::kBytes);
        } else {
            left.fetch(s * Left::kDepth, held_l);
            right.fetch(s * Left::kDepth, held_r);
        }
    };
    auto finish = [&](uint32_t s) {
        if constexpr (!ALIGNED) {
            left.put(held_l, lds + (s & 1) * kBytes);
            right.put(held_r, lds + (s & 1) * kBytes + Left::kBytes);
        }
    };
    if (stages) {
        begin(0);
        finish(0);
        scales(0);
    }
    for (uint32_t s = 0; s < stages; ++s) {
        stage_barrier();
        float now_m[FM], now_n = scale_n;
#pragma unroll
        for (int j = 0; j < FM; ++j) now_m[j] = scale_m[j];
        if (s + 1 < stages) {
            begin(s + 1);
            scales(s + 1);
        }
        const char *ll = lds + (s & 1) * kBytes, *lr = ll + Left::kBytes;
        if constexpr (kQuant) {
            static_assert(TN / WN <= 128 && 128 % (TN / WN) == 0, "a wave's columns have one scale");
            u32x8 x[FM][2];
            auto wide = [&](const char *p, uint32_t from, uint32_t k) {
                u32x8 v;
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    const u32x4 q = Left::along(p, from, k * 4 + lane / 32 * 2 + h);
#pragma unroll
                    for (int b = 0; b < 4; ++b) v[4 * h + b] = q[b];
                }
                return v;
            };
#pragma unroll
            for (int j = 0; j < FM; ++j)
#pragma unroll
                for (int k = 0; k < 2; ++k) x[j][k] = wide(lr, wm + j * 32, k);
#pragma unroll
            for (int i = 0; i < FN; ++i) {
                u32x8 w[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) w[k] = wide(ll, wn + i * 32, k);
#pragma unroll
                for (int j = 0; j < FM; ++j) {
                    f32x16 part = {};
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        part = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[k], x[j][k], part, 0, 0, 0, 0x7F7F7F7F, 0, 0x7F7F7F7F);
                    const float f = now_m[j] * now_n;
#pragma unroll
                    for (int q = 0; q < 16; ++q) acc[i][j][q] += part[q] * f;
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                u32x4 x[FM], w[FN];
#pragma unroll
                for (int j = 0; j < FM; ++j) x[j] = Right::fragment(lr, wm + j * 32, k);
#pragma unroll
                for (int i = 0; i < FN; ++i) w[i] = Left::fragment(ll, wn + i * 32, k);
#pragma unroll
                for (int i = 0; i < FN; ++i)
#pragma unroll
                    for (int j = 0; j < FM; ++j) acc[i][j] = multiply(w[i], x[j], acc[i][j], T());
            }
        }
        if (s + 1 < stages) finish(s + 1);
    }

    // a lane has column m of the instruction's result and rows 8 q + 4 (lane / 32) .. + 4 of n
    O *out = static_cast<O *>(a.o);
    if constexpr (P == Product::kGradMatrix) out += t.expert * a.o_expert;
    else out += t.first * a.o_stride;
#pragma unroll
    for (int j = 0; j < FM; ++j) {
        const uint32_t m = m0 + wm + j * 32 + lane % 32;
        if (m >= rows) continue;
        O *row = out + m * a.o_stride;
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint32_t n = n0 + wn + i * 32 + q * 8 + lane / 32 * 4;
                const float v[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                if (n < a.n) store_four<T>(row, n, a.n, v);
            }
    }
}

template <class T, class O, Product P, int TM, int TN, int WM, int WN, bool ALIGNED>
int product_launch_of(const ProductArgs &a, hipStream_t s)
{
    // no more tiles of rows than one for each TM of them and one for each expert
    const uint64_t mt = P == Product::kGradMatrix ? a.experts * ceil_div(a.m, TM) : a.rows / TM + std::min<uint64_t>(a.experts, a.rows);
    const uint64_t tiles = mt * ceil_div(a.n, TN) + 8;  // (each XCD's share is rounded up)
    if (tiles > 0x7FFFFFFFull) return LCPP_ERR_SIZE_LIMIT;
    const char *name = P == Product::kForward ? "expert_product" : P == Product::kGradRows ? "expert_product_rows" : "expert_product_matrix";
    LCPP_LAUNCH(name, s, product_kernel<T, O, P, TM, TN, WM, WN, ALIGNED><<<(uint32_t)tiles, WM * WN * kWave, 0, s>>>(a));
    LCPP_CHECK_LAUNCH();
    return LCPP_OK;
}

template <class T, class O, Product P>
int product_launch(const ProductArgs &a, hipStream_t s)
{
    constexpr size_t e = std::is_same_v<T, fp8> ? 1 : sizeof(T);
    auto whole = [&](const void *p, uint64_t stride, uint64_t expert) {
        return reinterpret_cast<uintptr_t>(p) % kChunk == 0 && stride * e % kChunk == 0 && expert * e % kChunk == 0 &&
               stride * e < (1u << 22);
    };
    bool aligned = whole(a.r, a.r_stride, 0) && whole(a.l, a.l_stride, P == Product::kGradMatrix ? 0 : a.l_expert);
    if (P != Product::kGradMatrix) aligned = aligned && a.c * e % kChunk == 0;
    if (P != Product::kForward) aligned = aligned && a.n * e % kChunk == 0;
    if (P == Product::kGradMatrix) aligned = aligned && a.m * e % kChunk == 0;
    if (!aligned) return product_launch_of<T, O, P, 128, 128, 2, 2, false>(a, s);
    if constexpr (P != Product::kGradMatrix) {
        const uint64_t each = a.rows / a.experts;
        if (each < 48) return product_launch_of<T, O, P, 32, 128, 1, 4, true>(a, s);
        if (each < 192) return product_launch_of<T, O, P, 128, 128, 2, 2, true>(a, s);
    }
    return product_launch_of<T, O, P, 256, 256, 4, 2, true>(a, s);
}

}  // namespace
}  // namespace lcpp

using namespace lcpp;

namespace {
int product_sizes(uint64_t rows, uint64_t experts, uint64_t outputs, uint64_t inputs)
{
    if (rows > 0x7FFFFFFFull || experts > 0xFFFFFull || outputs > kMaxCols || inputs > kMaxCols) return LCPP_ERR_INVALID_ARG;
    return LCPP_OK;
}
}  // namespace

extern "C" int lcpp_expert_product(lcpp_dtype t, const void *in, uint64_t in_stride, const void *weight,
                                   uint64_t weight_stride, uint64_t weight_expert_stride, const int32_t *offsets,
                                   lcpp_dtype out_t, void *out, uint64_t out_stride, const float *in_scales,
                                   uint64_t in_scale_row_stride, uint64_t in_scale_group_stride,
                                   const float *weight_scales, uint64_t rows, uint64_t experts, uint64_t outputs,
                                   uint64_t inputs, void *stream)
{
    const bool quant = t == LCPP_FLOAT8_E4M3;
    const size_t e = quant ? 1 : float_size(t), oe = float_size(out_t);
    if (!e || !oe || (!quant && out_t != t)) return LCPP_ERR_UNSUPPORTED_DTYPE;
    if (product_sizes(rows, experts, outputs, inputs)) return LCPP_ERR_INVALID_ARG;
    if (rows == 0 || experts == 0 || outputs == 0) return LCPP_OK;
    if (!elem_ok(offsets, 4) || !elem_ok(out, oe) || !rows_apart(out_stride, rows, outputs)) return LCPP_ERR_INVALID_ARG;
    if (inputs && (!elem_ok(in, e) || !elem_ok(weight, e))) return LCPP_ERR_INVALID_ARG;
    if (quant && inputs && (!elem_ok(in_scales, 4) || !elem_ok(weight_scales, 4))) return LCPP_ERR_INVALID_ARG;
    if (!quant && (in_scales || weight_scales)) return LCPP_ERR_INVALID_ARG;
    if (same_place(out, in) || same_place(out, weight)) return LCPP_ERR_INVALID_ARG;
    ProductArgs a = {};
    a.r = in, a.l = weight, a.o = out;
    a.r_stride = in_stride, a.l_stride = weight_stride, a.l_expert = weight_expert_stride, a.o_stride = out_stride;
    a.offsets = offsets, a.rows = rows, a.experts = (uint32_t)experts;
    a.n = (uint32_t)outputs, a.c = (uint32_t)inputs;
    a.r_scales = in_scales, a.l_scales = weight_scales;
    a.r_scale_row = in_scale_row_stride, a.r_scale_col = in_scale_group_stride;
    a.l_scale_row = (uint32_t)ceil_div(inputs, 128);
    a.l_scale_expert = (uint64_t)a.l_scale_row * ceil_div(outputs, 128);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (quant)
        return float_dispatch(out_t, [&](auto x) -> int { return product_launch<fp8, decltype(x), Product::kForward>(a, s); });
    return float_dispatch(t, [&](auto x) -> int { return product_launch<decltype(x), decltype(x), Product::kForward>(a, s); });
}

extern "C" int lcpp_expert_product_backward(lcpp_dtype t, const void *grad_out, uint64_t grad_out_stride, const void *in,
                                            uint64_t in_stride, const void *weight, uint64_t weight_stride,
                                            uint64_t weight_expert_stride, const int32_t *offsets, void *grad_in,
                                            uint64_t grad_in_stride, lcpp_dtype grad_weight_t, void *grad_weight,
                                            uint64_t grad_weight_stride, uint64_t grad_weight_expert_stride, uint64_t rows,
                                            uint64_t experts, uint64_t outputs, uint64_t inputs, void *stream)
{
    const size_t e = float_size(t), we = float_size(grad_weight_t);
    if (!e || (grad_weight && (!we || (grad_weight_t != t && grad_weight_t != LCPP_FLOAT32)))) return LCPP_ERR_UNSUPPORTED_DTYPE;
    if (product_sizes(rows, experts, outputs, inputs)) return LCPP_ERR_INVALID_ARG;
    if (experts == 0 || inputs == 0) return LCPP_OK;
    if (!elem_ok(offsets, 4)) return LCPP_ERR_INVALID_ARG;
    if (rows && outputs && !elem_ok(grad_out, e)) return LCPP_ERR_INVALID_ARG;
    if (grad_in && rows && (!elem_ok(grad_in, e) || !rows_apart(grad_in_stride, rows, inputs) || (outputs && !elem_ok(weight, e))))
        return LCPP_ERR_INVALID_ARG;
    if (grad_weight && outputs) {
        if (!elem_ok(grad_weight, we) || (rows && !elem_ok(in, e)) || !rows_apart(grad_weight_stride, outputs, inputs)) return LCPP_ERR_INVALID_ARG;
        // (matrices one behind the other, or side by side within the rows of one another)
        const uint64_t span = (outputs - 1) * grad_weight_stride + inputs;
        if (experts > 1 && grad_weight_expert_stride < span) return LCPP_ERR_INVALID_ARG;
    }
    if (same_place(grad_in, grad_weight) || same_place(grad_in, grad_out) || same_place(grad_in, weight) ||
        same_place(grad_weight, in) || same_place(grad_weight, grad_out))
        return LCPP_ERR_INVALID_ARG;
    // (the rows' gradient is made first, and the matrices' reads the rows)
    if (grad_weight && same_place(grad_in, in)) return LCPP_ERR_INVALID_ARG;
    hipStream_t s = static_cast<hipStream_t>(stream);
    ProductArgs a = {};
    a.offsets = offsets, a.rows = rows, a.experts = (uint32_t)experts;
    a.n = (uint32_t)inputs;
    a.r = grad_out, a.r_stride = grad_out_stride;
    if (grad_in && rows) {
        a.l = weight, a.l_stride = weight_stride, a.l_expert = weight_expert_stride;
        a.o = grad_in, a.o_stride = grad_in_stride;
        a.c = (uint32_t)outputs;
        const int status = float_dispatch(t, [&](auto x) -> int { return product_launch<decltype(x), decltype(x), Product::kGradRows>(a, s); });
        if (status) return status;
    }
    if (grad_weight && outputs) {
        a.l = in, a.l_stride = in_stride, a.l_expert = 0;
        a.o = grad_weight, a.o_stride = grad_weight_stride, a.o_expert = grad_weight_expert_stride;
        a.m = (uint32_t)outputs, a.c = 0;
        return float_dispatch(t, [&](auto x) -> int {
            using T = decltype(x);
            if constexpr (!std::is_same_v<T, float>)
                if (grad_weight_t == LCPP_FLOAT32) return product_launch<T, float, Product::kGradMatrix>(a, s);
            return product_launch<T, T, Product::kGradMatrix>(a, s);
        });
    }
    return LCPP_OK;
}
