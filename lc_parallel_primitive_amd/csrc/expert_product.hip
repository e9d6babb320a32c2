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
// Bound by the matrix cores, whose clock falls under their load, and for few rows by reading
// the matrices.  bfloat16: 8192 x 8192 x 8192 at 1290 to 1360 TFLOP/s; 32768 rows of 16
// experts of 2816 x 2048 of 2048 rows each in 351 us forward, 348 and 375 the gradients, of uneven
// ones 1094 to 1138 all three (1.0 PFLOP/s: a tile's end every 32 stages, and rows that no expert
// has); 384 rows of 128 experts of 2048 x 1024 in 73 to 79 us (447 MB, 5.7 to 6.1 TB/s).  float32:
// 122 to 143 TFLOP/s.  Eight waves of 128 x 64 outputs with stages of 128 bytes twice against four
// waves of 128 x 128 with stages of 64 bytes four times 666 to 1209 TFLOP/s, of 128 bytes twice
// 872 to 1217.
//
// 8-bit operands have a scale for each row's 128 inputs and for 128 outputs x 128 inputs of
// a matrix: a stage is 128 inputs deep, its product is made from 0 and then added to the
// sums in 32 bits, times both scales.  (Inside it the matrix cores cut the products, which
// they add in eights, 13 bits below the largest of each eight: up to 7 products are off by
// 2^-13 of the largest, where the operands' own roundings are 2^-4 of each.)  16384 rows of
// 32 experts of 4096 x 2048: 202 to 220 us, 1.25 to 1.36 PFLOP/s; 8192 x 8192 x 8192 2.0 to 2.1.
// The sums' scaling, 16 vector instructions for two matrix instructions, is of the product
// before the one that is being made.
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
    // (m0 is put back: the compiler, which has no way to be told that it changes, may keep an index there)
    uint32_t m0;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0)
                 : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(rsrc)
                 : "memory");
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
// Every wave's loads to LDS but the last LATER ones have arrived, and every wave has read what
// it needed before.
template <int LATER = 0>
__device__ __forceinline__ void stage_barrier()
{
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LATER) : "memory");
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// ---------------------------------------------------------------- an operand's stage
// X elements (rows or columns of the operand) x BYTES of c.  ACROSS: c runs from row to row,
// X columns in each; else X rows with c along them.
template <class T, uint32_t X, uint32_t BYTES, uint32_t THREADS, bool ACROSS>
struct Stage {
    static constexpr uint32_t kElems = kChunk / sizeof(T);         // of a chunk
    static constexpr uint32_t kDepth = BYTES / sizeof(T);          // of c
    static constexpr uint32_t kRowChunks = ACROSS ? X / kElems : BYTES / kChunk;
    static constexpr uint32_t kBytes = X * BYTES;
    static constexpr uint32_t kLoads = kBytes / kChunk / THREADS;  // of a thread
    static_assert(kBytes % (kChunk * THREADS) == 0, "whole loads");
    // Chunk c of a row is kept in place c ^ swizzle(row).  Along: the 16 rows that a read touches at
    // once fill the 256 bytes of all banks, rows of 64 bytes by fours and rows of 128 by twos.  Across:
    // the four rows of a transposing read have 64 bytes each, the two of a 32-bit read, four apart, 128.
    static __device__ __forceinline__ uint32_t swizzle(uint32_t row)
    {
        static_assert(BYTES == 64 || BYTES == 128, "rows of 4 or 8 chunks");
        if constexpr (ACROSS && sizeof(T) == 4) return (row >> 2 & 1) << 3;
        return ACROSS ? (row & 3) << 2 : BYTES == 128 ? (row >> 1) & 7 : (row >> 2) & 3;
    }

    const T *base;     // of the tile
    uint64_t stride;   // of rows, in elements
    uint32_t valid;    // of X
    uint32_t depth;    // of c in all
    // of the thread's chunk 0; the others are kRowStep rows apart and have the same chunk, the rows' swizzles repeating
    // after as many
    static constexpr uint32_t kRowStep = THREADS / kRowChunks;
    static_assert(THREADS % kRowChunks == 0 && kRowStep % (!ACROSS ? 16 : sizeof(T) == 4 ? 8 : 4) == 0, "the same swizzle");
    uint32_t row, chunk;
    uint32_t off[kLoads];

    __device__ __forceinline__ void set(const T *p, uint64_t s, uint32_t x, uint32_t c)
    {
        base = p, stride = s, valid = x, depth = c;
        row = threadIdx.x / kRowChunks;
        chunk = (threadIdx.x % kRowChunks) ^ swizzle(row);
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            const uint32_t r = row + i * kRowStep;
            if constexpr (ACROSS) {
                off[i] = chunk * kElems < valid ? (uint32_t)(r * stride * sizeof(T)) + chunk * kChunk : kOutside;
            } else {
                // (rows past the last one are the last one again, and are not stored)
                off[i] = (uint32_t)((r < valid ? r : valid - 1) * stride * sizeof(T)) + chunk * kChunk;
            }
        }
    }
    // Load i of the stage from c = from on, all of whose chunks are aligned and whole; 0 past the end.
    __device__ __forceinline__ u32x4 source(uint32_t from) const { return stage_rsrc(base + (ACROSS ? from * stride : from)); }
    __device__ __forceinline__ void issue_one(uint32_t i, u32x4 rsrc, uint32_t from, uint32_t lds) const
    {
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
        uint32_t v = off[i];
        if (from + (ACROSS ? row + i * kRowStep : chunk * kElems) >= depth) v = kOutside;
        load_to_lds(rsrc, v, lds + (i * THREADS + wave * kWave) * kChunk);
    }
    __device__ __forceinline__ void issue(uint32_t from, uint32_t lds) const
    {
        const u32x4 rsrc = source(from);
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) issue_one(i, rsrc, from, lds);
    }
    // The same by way of registers, for any stride, size and alignment.
    struct Held {
        u32x4 v[kLoads];
    };
    __device__ __forceinline__ void fetch(uint32_t from, Held &h) const
    {
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            const uint32_t line = row + i * kRowStep, c = from + (ACROSS ? line : chunk * kElems);
            const uint32_t r = ACROSS ? 0 : line < valid ? line : valid - 1;
            const uint32_t inside = ACROSS ? valid : depth, at = ACROSS ? chunk * kElems : c;
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
        return *reinterpret_cast<const u32x4 *>(lds + r * BYTES + ((chunk ^ swizzle(r)) * kChunk));
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
// The tiles of an expert lie one behind the other, kBand rows of tiles at a time, m fastest: the
// 32 that the CUs of an XCD have at once are 8 x 4 and share operands in its L2.
constexpr uint32_t kBand = 8;
__device__ __forceinline__ void tile_place(uint32_t in, uint32_t mt, uint32_t nt, uint32_t &m, uint32_t &n)
{
    const uint32_t band = in / (kBand * nt), from = band * kBand, high = mt - from < kBand ? mt - from : kBand;
    in -= from * nt;
    n = in / high;
    m = from + in - n * high;
}

constexpr uint32_t kProductExperts = 1024;  // at most
constexpr uint32_t kXcds = 8;
struct Tile {
    uint32_t expert, m, n;  // numbers of the tile's first row and column, in tiles
    uint32_t first, count;  // the expert's rows
    bool there;
};
// The experts with their rows, and the number of tiles before each, in LDS.  A workgroup takes
// one tile after the other, without asking the others.  Forward and grad rows, whose tiles take
// the same time: the XCDs, which get the workgroups in turn, have an eighth of all tiles each.
// Grad matrix, whose tiles take as long as their expert has rows: experts with many rows come
// first, and chunks of tiles, one for each workgroup of an XCD, go to the XCD that has least to do
// so far, which every workgroup works out for itself (32768 rows, 16 experts of 2816 x 2048, the
// largest with a quarter of the rows: 985 us with an eighth each in the experts' order, 484
// with chunks dealt to and fro).  Past kChunks they are dealt to and fro.
template <Product P, int TM, int TN, int THREADS>
struct Tiles {
    uint32_t start[kProductExperts + 1];
    uint32_t first[kProductExperts], count[kProductExperts];
    uint16_t order[kProductExperts];
    static constexpr uint32_t kChunks = P == Product::kGradMatrix ? 512 : 1;
    uint16_t mine[kChunks];  // the chunks of this workgroup's XCD
    uint32_t mine_count;
    uint32_t wave_sum[THREADS / kWave];
    uint32_t all;

    __device__ __forceinline__ void make(const ProductArgs &a)
    {
        const uint32_t tid = threadIdx.x, nt = (a.n + TN - 1) / TN;
        for (uint32_t e = tid; e < a.experts; e += THREADS) {
            int64_t b = a.offsets[e], z = a.offsets[e + 1];
            b = b < 0 ? 0 : b;
            z = z > (int64_t)a.rows ? (int64_t)a.rows : z;
            first[e] = (uint32_t)b;
            count[e] = z > b ? (uint32_t)(z - b) : 0;
            order[e] = (uint16_t)e;
        }
        __syncthreads();
        if constexpr (P == Product::kGradMatrix) {
            for (uint32_t e = tid; e < a.experts; e += THREADS) {
                const uint32_t mine = count[e];
                uint32_t rank = 0;
                for (uint32_t j = 0; j < a.experts; ++j) rank += count[j] > mine || (count[j] == mine && j < e);
                order[rank] = (uint16_t)e;
            }
            __syncthreads();
        }
        uint32_t before = 0;
        for (uint32_t base = 0; base < a.experts; base += THREADS) {
            const uint32_t i = base + tid;
            uint32_t tiles = 0;
            if (i < a.experts) tiles = nt * (P == Product::kGradMatrix ? (a.m + TM - 1) / TM : (count[order[i]] + TM - 1) / TM);
            const uint32_t sum = wave_inclusive_scan(tiles, SumOp());
            if (lane_id() == kWave - 1) wave_sum[tid / kWave] = sum;
            __syncthreads();
            uint32_t s = before + sum - tiles;
            for (uint32_t w = 0; w < THREADS / kWave; ++w) {
                if (w < tid / kWave) s += wave_sum[w];
                before += wave_sum[w];
            }
            if (i < a.experts) start[i] = s;
            __syncthreads();
        }
        if (tid == 0) start[a.experts] = all = before;
        __syncthreads();
        if constexpr (P == Product::kGradMatrix) {
            const uint32_t side = gridDim.x / kXcds, chunks = (before + side - 1) / side;
            if (chunks <= kChunks && tid < kWave) {
                // a lane for each XCD holds what it has to do; a stage and a tile's end take about 64 rows' time each
                const uint32_t lane = lane_id();
                uint32_t load = lane < kXcds ? 0 : 0xFFFFFFFFu, e = 0, n = 0;
                for (uint32_t c = 0; c < chunks; ++c) {
                    while (start[e + 1] <= c * side) ++e;
                    const uint32_t key = lane < kXcds ? load << 3 | lane : 0xFFFFFFFFu;
                    const uint32_t xcd = wave_reduce_dpp(key, MinOp()) & 7;
                    if (lane == xcd) load += (count[order[e]] + 63) / 64 + 6;
                    if (xcd == blockIdx.x % kXcds) mine[n++] = (uint16_t)c;
                }
                mine_count = n;
            }
            __syncthreads();
        }
    }
    // The workgroup's tile number `turn`, which may not be there.
    __device__ __forceinline__ Tile get(const ProductArgs &a, uint32_t turn) const
    {
        Tile t = {};
        const uint32_t xcd = blockIdx.x % kXcds, slot = blockIdx.x / kXcds, side = gridDim.x / kXcds;
        const uint32_t total = __builtin_amdgcn_readfirstlane(all);
        uint32_t id;
        if constexpr (P == Product::kGradMatrix) {
            const bool listed = (total + side - 1) / side <= kChunks;
            uint32_t chunk = turn * kXcds + (turn & 1 ? kXcds - 1 - xcd : xcd);
            if (listed) {
                if (turn >= __builtin_amdgcn_readfirstlane(mine_count)) return t;
                chunk = __builtin_amdgcn_readfirstlane(mine[turn]);
            }
            id = chunk * side + slot;
        } else {
            const uint32_t per = (total + kXcds - 1) / kXcds, in = turn * side + slot;
            id = in < per ? xcd * per + in : total;
        }
        if (id >= total) return t;
        uint32_t lo = 0, hi = a.experts;  // start[lo] <= id < start[hi]
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (__builtin_amdgcn_readfirstlane(start[mid]) <= id) lo = mid;
            else hi = mid;
        }
        t.expert = __builtin_amdgcn_readfirstlane(order[lo]);
        t.first = __builtin_amdgcn_readfirstlane(first[t.expert]);
        t.count = __builtin_amdgcn_readfirstlane(count[t.expert]);
        const uint32_t nt = (a.n + TN - 1) / TN, mt = ((P == Product::kGradMatrix ? a.m : t.count) + TM - 1) / TM;
        const uint32_t in = id - __builtin_amdgcn_readfirstlane(start[lo]);
        if (in >= mt * nt) return t;  // (offsets that do not rise, and so many rows that their sum wrapped)
        tile_place(in, mt, nt, t.m, t.n);
        t.there = true;
        return t;
    }
};

template <class O>
__device__ __forceinline__ void store_four(O *row, uint32_t col, uint32_t cols, const float (&x)[4])
{
    if (col + 4 <= cols) store_pack<4>(row + col, x);
    else
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (col + i < cols) row[col + i] = (O)x[i];
}

// The operands of a tile, from its first row and column on.
template <Product P, class E>
__device__ __forceinline__ void tile_operands(const ProductArgs &a, const Tile &t, uint32_t m0, uint32_t n0, const E *&lp, const E *&rp,
                                              uint32_t &rows, uint32_t &depth)
{
    rows = P == Product::kGradMatrix ? a.m : t.count;  // of the output
    depth = P == Product::kGradMatrix ? t.count : a.c;
    lp = static_cast<const E *>(a.l), rp = static_cast<const E *>(a.r);
    if constexpr (P == Product::kForward) lp += t.expert * a.l_expert + n0 * a.l_stride;
    else if constexpr (P == Product::kGradRows) lp += t.expert * a.l_expert + n0;
    else lp += (uint64_t)t.first * a.l_stride + n0;
    if constexpr (P == Product::kGradMatrix) rp += (uint64_t)t.first * a.r_stride + m0;
    else rp += (uint64_t)(t.first + m0) * a.r_stride;
}

// f(0) .. f(N - 1), as integral constants.
template <int N, int I = 0, class F>
__device__ __forceinline__ void each_of(F f)
{
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        each_of<N, I + 1>(f);
    }
}

// Results of 2-byte types.  A lane has column m = lane % 32 of an instruction's result and the rows
// 8 q + 4 (lane / 32) .. + 4 of n; exchanges between the halves and the quarters of the wave make
// that eight neighbouring n of one m, four lanes of which fill 64 bytes of a row of the
// output: chunk (lane / 16) with its bits exchanged, of row lane % 16 and 16 + lane % 16.
// (With four n a lane, in 16-byte pieces, the requests to the L2 took 10 us for 256 tiles of
// 256 x 256.)
template <class O>
constexpr bool kPacked = sizeof(O) == 2;
template <class O>
__device__ __forceinline__ void pack_rows(const f32x16 &acc, u32x4 (&rows)[2])
{
    uint32_t p[4][2];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        typedef O v4 __attribute__((ext_vector_type(4)));
        v4 v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = (O)acc[4 * q + k];
        const uint2 w = __builtin_bit_cast(uint2, v);
        p[q][0] = w.x, p[q][1] = w.y;
    }
    uint32_t half[2][4];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            const auto w = __builtin_amdgcn_permlane32_swap(p[2 * c][d], p[2 * c + 1][d], false, false);
            half[c][d] = w[0], half[c][2 + d] = w[1];
        }
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const auto w = __builtin_amdgcn_permlane16_swap(half[0][d], half[1][d], false, false);
        rows[0][d] = w[0], rows[1][d] = w[1];
    }
}
__device__ __forceinline__ uint32_t packed_chunk()
{
    const uint32_t g = lane_id() / 16;
    return g >> 1 | (g & 1) << 1;
}
// 16 bytes to a row, counted by what waits for the loads around them.  (The values have been
// converted, so no matrix instruction's result is stored directly.)
template <int OFFSET>
__device__ __forceinline__ void store_counted(void *p, u32x4 v)
{
    asm volatile("global_store_dwordx4 %0, %1, off offset:%2\n\ts_nop 0" ::"v"(p), "v"(v), "n"(OFFSET) : "memory");
}
template <class O, int FM, int FN>
__device__ __forceinline__ void store_whole_tile(O *out, uint64_t stride, const f32x16 (&acc)[FN][FM])
{
    O *row = out + lane_id() % 16 * stride + packed_chunk() * 8;
#pragma unroll
    for (int j = 0; j < FM; ++j, row += 32 * stride) {
        each_of<FN>([&](auto i) {
            u32x4 v[2];
            pack_rows<O>(acc[decltype(i)::value][j], v);
            store_counted<decltype(i)::value * 64>(row, v[0]);
            store_counted<decltype(i)::value * 64>(row + 16 * stride, v[1]);
        });
    }
}

// A lane has column m of the instructions' results and rows 8 q + 4 (lane / 32) .. + 4 of n.
template <Product P, class O, int FM, int FN>
__device__ __forceinline__ void store_tile(const ProductArgs &a, const Tile &t, const f32x16 (&acc)[FN][FM], uint32_t m0, uint32_t n0,
                                           uint32_t rows)
{
    O *out = static_cast<O *>(a.o);
    if constexpr (P == Product::kGradMatrix) out += t.expert * a.o_expert;
    else out += (uint64_t)t.first * a.o_stride;
    const uint32_t lane = lane_id();
    if constexpr (kPacked<O>) {
#pragma unroll
        for (int j = 0; j < FM; ++j)
#pragma unroll
            for (int i = 0; i < FN; ++i) {
                u32x4 v[2];
                pack_rows<O>(acc[i][j], v);
                const uint32_t n = n0 + i * 32 + packed_chunk() * 8;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t m = m0 + j * 32 + h * 16 + lane % 16;
                    if (m >= rows || n >= a.n) continue;
                    Octet<O> x;
                    __builtin_memcpy(&x.v, &v[h], sizeof(x.v));
                    O *at = out + m * a.o_stride + n;
                    if (n + kOctet <= a.n) *reinterpret_cast<typename Octet<O>::vec_u *>(at) = x.v;
                    else
#pragma unroll
                        for (uint32_t k = 0; k < kOctet; ++k)
                            if (n + k < a.n) at[k] = x.v[k];
                }
            }
        return;
    }
#pragma unroll
    for (int j = 0; j < FM; ++j) {
        const uint32_t m = m0 + j * 32 + lane % 32;
        if (m >= rows) continue;
        O *row = out + m * a.o_stride;
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint32_t n = n0 + i * 32 + q * 8 + lane / 32 * 4;
                const float v[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                if (n < a.n) store_four(row, n, a.n, v);
            }
    }
}

// The loads of a workgroup's stages, one behind the other over all its tiles.
template <class T, Product P, int TM, int TN, class Left, class Right, class List>
struct Loads {
    Left left;
    Right right;
    uint32_t turn = 0, from = 0, depth = 0;
    bool more = true;
    // The next stage, of the next tile that has any; past the last one loads give 0.
    __device__ __forceinline__ void next(const ProductArgs &a, const List &tiles)
    {
        from += Left::kDepth;
        while (from >= depth && more) {
            const Tile t = tiles.get(a, turn++);
            more = t.there;
            if (!more) break;
            uint32_t rows;
            const T *lp, *rp;
            const uint32_t m0 = t.m * TM, n0 = t.n * TN;
            tile_operands<P>(a, t, m0, n0, lp, rp, rows, depth);
            from = 0;
            if (depth == 0) continue;
            left.set(lp, a.l_stride, a.n - n0, depth);
            right.set(rp, a.r_stride, rows - m0, depth);
        }
    }
    __device__ __forceinline__ void issue(int r, uint32_t lds) const
    {
        if (r < (int)Left::kLoads) left.issue_one(r, left.source(from), from, lds);
        else right.issue_one(r - Left::kLoads, right.source(from), from, lds + Left::kBytes);
    }
};

// A workgroup of WM x WN waves makes tiles of TM x TN outputs, one after the other, from operands
// whose chunks are whole and aligned.  The stages of all its tiles are one stream: loads for a
// tile begin while the one before is multiplied.  Fragments are read one step ahead into the
// other of two sets of registers, loads and reads are issued between the matrix instructions, and
// a stage's barrier comes before its last step: by then every wave has that step's fragments, so
// the stage's place is free for the loads of the stage BUFS later, and the next stage, whose first
// fragments are read now, has arrived.
template <class T, class O, Product P, int TM, int TN, int WM, int WN, int BYTES, int BUFS>
__global__ __launch_bounds__(WM *WN *kWave) void product_kernel(ProductArgs a)
{
    constexpr uint32_t THREADS = WM * WN * kWave;
    constexpr int FM = TM / WM / 32, FN = TN / WN / 32, STEPS = BYTES / 32, kProducts = FM * FN;
    constexpr bool kLeftAcross = P != Product::kForward, kRightAcross = P == Product::kGradMatrix;
    using Left = Stage<T, TN, BYTES, THREADS, kLeftAcross>;
    using Right = Stage<T, TM, BYTES, THREADS, kRightAcross>;
    constexpr uint32_t kBytes = Left::kBytes + Right::kBytes;
    constexpr int kLoads = Left::kLoads + Right::kLoads, kStores = kPacked<O> ? FM * FN * 2 : 0;
    static_assert(kStores + (BUFS - 2) * kLoads < 64, "the counter of memory operations");
    static_assert(BUFS >= 2 && STEPS % 2 == 0, "a stage ahead, and both sets of registers in turn");
    __shared__ __attribute__((aligned(256))) char lds[BUFS * kBytes];
    using List = Tiles<P, TM, TN, (int)THREADS>;
    __shared__ List tiles;

    tiles.make(a);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t wm = wave % WM * (TM / WM), wn = wave / WM * (TN / WN);
    const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)lds);

    // Load r of a stage belongs to its step `portion`, counted from the step that frees its place: spread over
    // a stage, or at once where no other stage is on its way.
    auto portion = [](int r) { return BUFS > 2 ? r * STEPS / kLoads : 0; };
    Loads<T, P, TM, TN, Left, Right, List> loads;
    uint32_t turn = 0;
    Tile t = tiles.get(a, turn++);
    if (!t.there) return;
    loads.next(a, tiles);
    u32x4 w[2][FN], x[2][FM];
    uint32_t at = 0, load_at = (BUFS - 1) * kBytes;  // of the stage that is multiplied, and loaded, in LDS
    if (loads.more) {
#pragma unroll
        for (int s = 0; s < BUFS; ++s) {
            if (s) loads.next(a, tiles);
#pragma unroll
            for (int r = 0; r < kLoads; ++r)
                if (s + 1 < BUFS || portion(r) == 0) loads.issue(r, lds0 + s * kBytes);
        }
        stage_barrier<(BUFS - 2) * kLoads>();
#pragma unroll
        for (int j = 0; j < FM; ++j) x[0][j] = Right::fragment(lds + Left::kBytes, wm + j * 32, 0);
#pragma unroll
        for (int i = 0; i < FN; ++i) w[0][i] = Left::fragment(lds, wn + i * 32, 0);
    }
    bool stores = false;  // this wave's last kStores memory operations are those of a whole tile
    for (;;) {
        const uint32_t rows = P == Product::kGradMatrix ? a.m : t.count, depth = P == Product::kGradMatrix ? t.count : a.c;
        f32x16 acc[FN][FM];
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int j = 0; j < FM; ++j) acc[i][j] = f32x16{};
        for (uint32_t s = 0; s < depth; s += Left::kDepth) {
            const uint32_t next = at + kBytes == BUFS * kBytes ? 0 : at + kBytes;
#pragma unroll
            for (int k = 0; k < STEPS; ++k) {
                const bool last = k + 1 == STEPS;
                if (last) {
                    // (a tile's stores were issued after the loads of its successor's first stages)
                    if (stores) stage_barrier<(BUFS - 2) * kLoads + kStores>();
                    else stage_barrier<(BUFS - 2) * kLoads>();
                    stores = false;
                    loads.next(a, tiles);
                    load_at = at;
                }
                const char *ll = lds + (last ? next : at), *lr = ll + Left::kBytes;
                const int set = k & 1, other = set ^ 1, step = (k + 1) % STEPS;
#pragma unroll
                for (int q = 0; q < kProducts; ++q) {
                    // what is issued before product q: reads in the first half of the step, loads in the last step
#pragma unroll
                    for (int r = 0; r < FM + FN; ++r) {
                        if (r * kProducts / (2 * (FM + FN)) != q) continue;
                        if (r < FM) x[other][r] = Right::fragment(lr, wm + r * 32, step);
                        else w[other][r - FM] = Left::fragment(ll, wn + (r - FM) * 32, step);
                    }
#pragma unroll
                    for (int r = 0; r < kLoads; ++r) {
                        if (portion(r) != step) continue;
                        if ((BUFS > 2 ? r * STEPS % kLoads * kProducts / kLoads : r * kProducts / kLoads) != q) continue;
                        loads.issue(r, lds0 + load_at);
                    }
                    acc[q / FM][q % FM] = multiply(w[set][q / FM], x[set][q % FM], acc[q / FM][q % FM], T());
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            at = next;
        }
        const uint32_t m0 = t.m * TM + wm, n0 = t.n * TN + wn;
        bool whole = false;
        if constexpr (kPacked<O> && BUFS == 2) {
            whole = m0 + TM / WM <= rows && n0 + TN / WN <= a.n;
            if (whole) {
                O *out = static_cast<O *>(a.o);
                if constexpr (P == Product::kGradMatrix) out += t.expert * a.o_expert;
                else out += (uint64_t)t.first * a.o_stride;
                store_whole_tile(out + m0 * a.o_stride + n0, a.o_stride, acc);
            }
        }
        if (!whole) store_tile<P, O>(a, t, acc, m0, n0, rows);
        stores = whole;
        t = tiles.get(a, turn++);
        if (!t.there) break;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the zeros past the end)
}

// Any stride, size and alignment by way of registers, and 8-bit operands: two stages of 128 bytes
// of c.  (16 experts of 1024 rows, 2048 x 1024, rows padded by one element against none: bfloat16 forward
// 106 against 66 us, its gradients 149 and 114 against 62 and 72, float32 575 against 502, 8 bits 249 against 46.)
template <class T, class O, Product P, int TM, int TN, int WM, int WN, bool ALIGNED>
__global__ __launch_bounds__(WM *WN *kWave) void product_simple_kernel(ProductArgs a)
{
    constexpr uint32_t THREADS = WM * WN * kWave, BYTES = 128;
    constexpr int FM = TM / WM / 32, FN = TN / WN / 32;
    constexpr bool kQuant = std::is_same_v<T, fp8>;
    using E = std::conditional_t<kQuant, uint8_t, T>;
    constexpr bool kLeftAcross = P != Product::kForward, kRightAcross = P == Product::kGradMatrix;
    using Left = Stage<E, TN, BYTES, THREADS, kLeftAcross>;
    using Right = Stage<E, TM, BYTES, THREADS, kRightAcross>;
    constexpr uint32_t kBytes = Left::kBytes + Right::kBytes;
    __shared__ __attribute__((aligned(256))) char lds[2 * kBytes];
    __shared__ Tiles<P, TM, TN, (int)THREADS> tiles;

    tiles.make(a);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id();
    const uint32_t wm = wave % WM * (TM / WM), wn = wave / WM * (TN / WN);
    const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)lds);
    Left left;
    Right right;
    typename Left::Held held_l;
    typename Right::Held held_r;
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
    // scales: of the lane's rows of m and of the wave's block of n
    float scale_m[FM], scale_n = 0.0f;
    auto scales = [&](const Tile &t, uint32_t s) {
        if constexpr (kQuant) {
#pragma unroll
            for (int j = 0; j < FM; ++j) {
                const uint32_t m = t.m * TM + wm + j * 32 + lane % 32;
                scale_m[j] = a.r_scales[(t.first + (m < t.count ? m : t.count - 1)) * a.r_scale_row + s * a.r_scale_col];
            }
            const uint32_t at = t.n * TN + wn, n = at < a.n ? at : a.n - 1;
            scale_n = a.l_scales[t.expert * a.l_scale_expert + (uint64_t)(n / 128) * a.l_scale_row + s];
        }
    };
    uint32_t turn = 0, rows = 0, stages = 0;
    // the tile's first stage, on its way while the tile before is stored
    auto enter = [&](const Tile &t) {
        uint32_t depth;
        const E *lp, *rp;
        const uint32_t m0 = t.m * TM, n0 = t.n * TN;
        tile_operands<P>(a, t, m0, n0, lp, rp, rows, depth);
        left.set(lp, a.l_stride, a.n - n0, depth);
        right.set(rp, a.r_stride, rows - m0, depth);
        stages = (depth + Left::kDepth - 1) / Left::kDepth;
        if (stages) {
            begin(0);
            scales(t, 0);
        }
    };
    Tile t = tiles.get(a, turn++);
    if (!t.there) return;
    enter(t);
    for (;;) {
        f32x16 acc[FN][FM];
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int j = 0; j < FM; ++j) acc[i][j] = f32x16{};
        if (stages) finish(0);
        for (uint32_t s = 0; s < stages; ++s) {
            stage_barrier();
            float now_m[FM], now_n = scale_n;
#pragma unroll
            for (int j = 0; j < FM; ++j) now_m[j] = scale_m[j];
            if (s + 1 < stages) {
                begin(s + 1);
                scales(t, s + 1);
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
                // (a product is added to the sums while the matrix cores make the next one)
                u32x8 w[2];
                f32x16 part[2];
#pragma unroll
                for (int q = 0; q <= FM * FN; ++q) {
                    const int i = q / FM, j = q % FM;
                    if (q < FM * FN) {
                        if (q == 0)
#pragma unroll
                            for (int k = 0; k < 2; ++k) w[k] = wide(ll, wn, k);
                        part[q & 1] = f32x16{};
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            part[q & 1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[k], x[j][k], part[q & 1], 0, 0, 0, 0x7F7F7F7F, 0, 0x7F7F7F7F);
                        if (j == FM - 1 && i + 1 < FN)
#pragma unroll
                            for (int k = 0; k < 2; ++k) w[k] = wide(ll, wn + (i + 1) * 32, k);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    if (q > 0) {
                        const int before = q - 1;
                        const float f = now_m[before % FM] * now_n;
#pragma unroll
                        for (int r = 0; r < 16; ++r) acc[before / FM][before % FM][r] += part[before & 1][r] * f;
                    }
                    __builtin_amdgcn_sched_barrier(0);
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
        __syncthreads();  // (the next tile's stages take this one's place)
        const Tile done = t;
        const uint32_t done_rows = rows;
        t = tiles.get(a, turn++);
        if (t.there) enter(t);
        store_tile<P, O>(a, done, acc, done.m * TM + wm, done.n * TN + wn, done_rows);
        if (!t.there) return;
    }
}

template <Product P, int TM, int TN, auto kernel>
int product_launch_of(const ProductArgs &a, int threads, hipStream_t s)
{
    static DeviceCache cache;
    // no more tiles of rows than one for each TM of them and one for each expert
    const uint64_t mt = P == Product::kGradMatrix ? a.experts * ceil_div(a.m, TM) : a.rows / TM + std::min<uint64_t>(a.experts, a.rows);
    const uint64_t tiles = mt * ceil_div(a.n, TN);
    if (tiles > 0x3FFFFFFFull) return LCPP_ERR_SIZE_LIMIT;
    // what the device holds at once, an equal number on every XCD
    const uint64_t most = (uint64_t)device_cus() * device_cached(cache, [&] {
                              int n = 0;
                              const hipError_t e = hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0);
                              return e == hipSuccess && n > 0 ? n : 1;
                          });
    const uint32_t grid = (uint32_t)(ceil_div(std::min(tiles, most), kXcds) * kXcds);
    const char *name = P == Product::kForward ? "expert_product" : P == Product::kGradRows ? "expert_product_rows" : "expert_product_matrix";
    LCPP_LAUNCH(name, s, kernel<<<grid, threads, 0, s>>>(a));
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
    if (!aligned) return product_launch_of<P, 128, 128, product_simple_kernel<T, O, P, 128, 128, 2, 2, false>>(a, 256, s);
    // Tiles by what the device's rounds of them take, in rounds of 256 x 256: some of the experts' last tiles are
    // empty, and the four products of 128 x 128, two workgroups of which share a CU, take 1.25 times as long as one
    // of 256 x 256.  (us forward, 256 -> 128: 16 experts of 256 rows, 2048 x 2048 bfloat16 48 -> 42, 2048 x 1024
    // float32 247 -> 141, 64 of 128 rows, 1408 x 2048 bfloat16 144 -> 109, 16 of 2048 rows, 2816 x 2048 362 -> 459.)
    const double cus = device_cus(), spare = 0.25 * (double)std::min<uint64_t>(a.experts, a.rows);
    auto rounds = [&](uint64_t tile, double at_once) {
        const double mt = P == Product::kGradMatrix ? (double)(a.experts * ceil_div(a.m, tile)) : (double)a.rows / (double)tile + spare;
        return std::max(1.0, mt * (double)ceil_div(a.n, tile) / at_once);
    };
    const bool large = rounds(256, cus) <= rounds(128, 2 * cus) * 0.625;
    // Rows of 32 where an expert has no more on average: one such tile holds them, and reads the matrices as fast as can be; a
    // second tile reads them once more.  (us forward, 128 x 128 -> 32 x 128: 128 experts of 2048 x 1024 with 3, 32, 40 and 64 rows
    // each bfloat16 99 -> 91, 107 -> 98, 111 -> 133, 118 -> 138, e4m3 49 -> 41, 58 -> 49, 60 -> 79, 68 -> 91; 64 of 1408 x 2048
    // bfloat16 97 -> 80, 101 -> 85, 102 -> 94, 105 -> 99; 16 of 4096 x 2048 43 -> 40, 44 -> 41, 44 -> 51, 45 -> 54; uneven
    // ones with 24 and 40 rows on average 105 -> 108 and 123 -> 131, 98 -> 82 and 101 -> 87, 68 -> 54 and 46 -> 57.)
    const bool few = P != Product::kGradMatrix && a.rows / a.experts <= 32;
    if constexpr (std::is_same_v<T, fp8>) {
        if (few) return product_launch_of<P, 32, 128, product_simple_kernel<T, O, P, 32, 128, 1, 4, true>>(a, 256, s);
        if (!large) return product_launch_of<P, 128, 128, product_simple_kernel<T, O, P, 128, 128, 2, 2, true>>(a, 256, s);
        return product_launch_of<P, 256, 256, product_simple_kernel<T, O, P, 256, 256, 4, 2, true>>(a, 512, s);
    } else {
        if constexpr (P != Product::kGradMatrix)
            if (few) return product_launch_of<P, 32, 128, product_kernel<T, O, P, 32, 128, 1, 4, 128, 4>>(a, 256, s);
        if (!large) return product_launch_of<P, 128, 128, product_kernel<T, O, P, 128, 128, 2, 2, 128, 2>>(a, 256, s);
        return product_launch_of<P, 256, 256, product_kernel<T, O, P, 256, 256, 4, 2, 128, 2>>(a, 512, s);
    }
}

}  // namespace
}  // namespace lcpp

using namespace lcpp;

namespace {
int product_sizes(uint64_t rows, uint64_t experts, uint64_t outputs, uint64_t inputs)
{
    if (rows > 0x7FFFFFFFull || experts > kProductExperts || outputs > kMaxCols || inputs > kMaxCols) return LCPP_ERR_INVALID_ARG;
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
        // matrices one behind the other, or side by side within the rows of one another
        const bool behind = grad_weight_expert_stride >= (outputs - 1) * grad_weight_stride + inputs;
        const bool beside = grad_weight_expert_stride >= inputs && grad_weight_stride >= (experts - 1) * grad_weight_expert_stride + inputs;
        if (experts > 1 && !behind && !beside) return LCPP_ERR_INVALID_ARG;
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
