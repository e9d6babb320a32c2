// tensor.hpp — elements of 2 and 4 bytes, rows of any stride and alignment, and
// the random bits of dropout, shared by the layer norm, dropout and recurrence
// kernels.
//
// Activations are float32, bfloat16 or float16; everything is computed in 32
// bits and rounded once, to nearest even, when it is stored.
#pragma once

#include "common.hpp"

namespace lcpp {

using bf16 = __bf16;
using f16 = _Float16;

// N consecutive elements as they lie in memory.  Rows may begin at any element:
// the vector types below ask for the alignment of one element only, and global
// memory instructions take such addresses in one access on this part.
template <class T, int N>
struct Pack {
    typedef T vec __attribute__((ext_vector_type(N)));
    typedef vec vec_u __attribute__((aligned(sizeof(T))));
    vec v;
    __device__ __forceinline__ float operator[](int i) const { return (float)v[i]; }
};

template <int N, class T>
__device__ __forceinline__ Pack<T, N> load_pack(const T *p)
{
    Pack<T, N> r;
    r.v = *reinterpret_cast<const typename Pack<T, N>::vec_u *>(p);
    return r;
}
// The same for data that is read once (streaming policy).
template <int N, class T>
__device__ __forceinline__ Pack<T, N> load_pack_nt(const T *p)
{
    Pack<T, N> r;
    r.v = __builtin_nontemporal_load(reinterpret_cast<const typename Pack<T, N>::vec_u *>(p));
    return r;
}
// The first `valid` of N elements, 0 in the others' place.
template <int N, class T>
__device__ __forceinline__ Pack<T, N> load_pack_part(const T *p, int valid)
{
    Pack<T, N> r;
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = i < valid ? p[i] : (T)0.0f;
    return r;
}
template <int N, class T>
__device__ __forceinline__ void store_pack(T *p, const float (&x)[N])
{
    typename Pack<T, N>::vec v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (T)x[i];
    *reinterpret_cast<typename Pack<T, N>::vec_u *>(p) = v;
}
// The same for results that are larger than the caches or read much later.
template <int N, class T>
__device__ __forceinline__ void store_pack_nt(T *p, const float (&x)[N])
{
    typename Pack<T, N>::vec v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (T)x[i];
    __builtin_nontemporal_store(v, reinterpret_cast<typename Pack<T, N>::vec_u *>(p));
}
template <int N, class T>
__device__ __forceinline__ void store_pack_part(T *p, const float (&x)[N], int valid)
{
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < valid) p[i] = (T)x[i];
}

// Eight columns of a row are what one lane loads at once (16 or 32 bytes) and
// what one block of random bits covers.
constexpr int kOctet = 8;
template <class T>
using Octet = Pack<T, kOctet>;

template <class T>
__device__ __forceinline__ Octet<T> load_octet(const T *row, uint32_t col, uint32_t cols)
{
    return col + kOctet <= cols ? load_pack<kOctet>(row + col) : load_pack_part<kOctet>(row + col, (int)cols - (int)col);
}
template <class T>
__device__ __forceinline__ void store_octet(T *row, uint32_t col, uint32_t cols, const float (&x)[kOctet])
{
    if (col + kOctet <= cols) store_pack<kOctet>(row + col, x);
    else store_pack_part<kOctet>(row + col, x, (int)cols - (int)col);
}

// ---------------------------------------------------------------- dropout
// Philox 4x32 with 7 rounds (Salmon, Moraes, Dror, Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC 2011, which reports that 7 rounds pass
// BigCrush): a block cipher of a counter, so any element's bits can be computed
// anywhere, in the backward pass again, and no mask is stored.  The counter is
// (column / 8, row, offset, offset >> 32) and the key the 64-bit seed; the 128
// bits are 16 for each of eight columns.  An element is kept where its 16 bits
// are at least `cut` = round(65536 p), so p is met to 2^-17, and the kept ones
// are multiplied by 65536 / (65536 - cut), which keeps the mean exactly.
// 16 bits an element instead of 32 halve the multiplications: a round is two
// 32 x 32 -> 64 bit products at a quarter of the ALUs' rate.
struct DropArgs {
    uint32_t cut;            // 0: everything is kept, 65536: nothing
    float scale;
    uint64_t seed, offset;
    const uint64_t *offset_dev;  // added to offset (may be null): a counter that a captured graph advances
};

__device__ __forceinline__ uint64_t drop_offset(const DropArgs &d)
{
    return d.offset + (d.offset_dev ? *d.offset_dev : 0);
}

__device__ __forceinline__ u32x4 philox7(uint32_t c0, uint32_t c1, uint64_t offset, uint64_t seed)
{
    uint32_t c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 7; ++r) {
        const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
        const uint32_t n0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0, n2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)p1;
        c3 = (uint32_t)p0;
        c0 = n0;
        c2 = n2;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    u32x4 v;
    v.x = c0;
    v.y = c1;
    v.z = c2;
    v.w = c3;
    return v;
}

// x[i] scaled or dropped (a select: what is dropped may be infinite or NaN).
__device__ __forceinline__ void drop_octet(float (&x)[kOctet], uint32_t row, uint32_t octet, uint64_t offset,
                                           const DropArgs &d)
{
    const u32x4 bits = philox7(octet, row, offset, d.seed);
#pragma unroll
    for (int i = 0; i < kOctet; ++i) {
        const uint32_t w = bits[i / 2];
        const uint32_t r = i & 1 ? w >> 16 : w & 0xFFFFu;
        x[i] = r >= d.cut ? x[i] * d.scale : 0.0f;
    }
}

// Host: the kernel's arguments for a probability; false where p is not in [0, 1] or the counter is misaligned.
inline bool drop_args(double p, uint64_t seed, uint64_t offset, const uint64_t *offset_dev, DropArgs *d)
{
    if (!(p >= 0.0 && p <= 1.0) || reinterpret_cast<uintptr_t>(offset_dev) % 8) return false;
    d->cut = (uint32_t)(p * 65536.0 + 0.5);
    d->scale = d->cut < 65536u ? (float)(65536.0 / (65536.0 - (double)d->cut)) : 0.0f;
    d->seed = seed;
    d->offset = offset;
    d->offset_dev = offset_dev;
    return true;
}

// ---------------------------------------------------------------- host checks
// Columns and rows that the 32-bit column, row and random-counter arithmetic of
// the row kernels covers.
constexpr uint64_t kMaxCols = 1u << 30;
constexpr uint64_t kMaxRows = 0xFFFFFFFFull;

inline size_t float_size(lcpp_dtype t)
{
    switch (t) {
    case LCPP_FLOAT32: return 4;
    case LCPP_BFLOAT16:
    case LCPP_FLOAT16: return 2;
    default: return 0;
    }
}
// Calls f with a value of the element type; LCPP_ERR_UNSUPPORTED_DTYPE for others.
template <class F>
int float_dispatch(lcpp_dtype t, F f)
{
    switch (t) {
    case LCPP_FLOAT32: return f(float());
    case LCPP_BFLOAT16: return f(bf16());
    case LCPP_FLOAT16: return f(f16());
    default: return LCPP_ERR_UNSUPPORTED_DTYPE;
    }
}
// A pointer that is not null and aligned to one element.
inline bool elem_ok(const void *p, size_t size) { return p && reinterpret_cast<uintptr_t>(p) % size == 0; }
// Two outputs in one place: one of them would be lost.
inline bool same_place(const void *p, const void *q) { return p && p == q; }
// Rows that do not overlap, as every output's have to be.
inline bool rows_apart(uint64_t stride, uint64_t rows, uint64_t cols) { return rows <= 1 || stride >= cols; }

}  // namespace lcpp
