// row_group.hpp — rows in the registers of a group of threads: what the kernels of
// the layer norm and the RMS norm share.
#pragma once

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

constexpr int kLongThreads = 1024;
constexpr int kLongWaves = kLongThreads / kWave;

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

}  // namespace
}  // namespace lcpp
