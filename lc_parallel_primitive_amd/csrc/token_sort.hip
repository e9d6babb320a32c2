// token_sort.hip — the (token, choice) pairs of a router in the order of their experts.
//
// A stable counting sort by a key of at most ten bits: pair p = token * choices + choice
// of expert e goes to row offsets[e] + (the pairs of e before p).  Pairs whose expert is
// not in 0 .. experts - 1 go nowhere (position -1).
//
// A wave ranks 64 neighbouring pairs at once: a ballot for each bit of the key gives every
// lane the lanes of its expert, their number below it is its rank and a counter in LDS,
// one for each wave and expert, carries on to the wave's next 64.  The waves of a
// workgroup take neighbouring parts of a chunk and their counters are summed in order, so
// there are no atomics whose order could matter.  Up to one workgroup's worth of pairs is
// one launch; more are two: the tiles' counts, then every workgroup sums the counts of
// the tiles before its own (and of all, for the experts' offsets) and ranks its tile.
//
// Bound by latency: 48 x 8 pairs of 128 experts take 4.0 us, a launch and six barriers;
// 32768 x 8 of 256 take 2.6 + 10.2 (3 MB): the tiles' counts, a chunk's experts, its
// ranks and its places one after the other.  (Tiles at most and 64s of a wave in a chunk, both
// launches: 128 and 2 12.0 us, 64 and 4 15.4, 32 and 4 19, 32 and 2 21, 64 and 2 16.)
#include <algorithm>

#include "common.hpp"

namespace lcpp {
namespace {

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr uint32_t kSortExperts = 1024;  // at most
constexpr uint32_t kSortTiles = 128;     // at most
constexpr int kSortItems = 2;            // 64s of a wave in a chunk
constexpr uint32_t kSums = 32;           // tiles that a thread sums at once
constexpr uint32_t kSortChunk = kSortThreads * kSortItems;
// Pairs that one workgroup sorts alone.
constexpr uint64_t kSortAlone = 2 * kSortChunk;

struct SortArgs {
    const int32_t *ids;
    int32_t *positions, *offsets, *sources;
    uint32_t *counts;  // [tile][expert]
    uint32_t *status;
    uint32_t n, experts, bits, tiles, tile;  // tile: pairs of one, a multiple of kSortChunk
};

__device__ __forceinline__ uint32_t pair_expert(const SortArgs &a, uint64_t p)
{
    // (experts: none)
    const uint32_t e = p < a.n ? (uint32_t)a.ids[p] : 0xFFFFFFFFu;
    return e < a.experts ? e : a.experts;
}

__global__ __launch_bounds__(kSortThreads) void token_count_kernel(SortArgs a)
{
    __shared__ uint32_t count[kSortExperts + 1];
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.status = 0;
    for (uint32_t e = threadIdx.x; e <= a.experts; e += kSortThreads) count[e] = 0;
    __syncthreads();
    const uint64_t first = (uint64_t)blockIdx.x * a.tile, last = first + a.tile < a.n ? first + a.tile : a.n;
    for (uint64_t p = first + threadIdx.x; p < last; p += kSortThreads)
        __hip_atomic_fetch_add(&count[pair_expert(a, p)], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < a.experts; e += kSortThreads) a.counts[(uint64_t)blockIdx.x * a.experts + e] = count[e];
}

// The lanes of the wave whose expert is this lane's.
__device__ __forceinline__ uint64_t same_expert(uint32_t e, uint32_t experts, uint32_t bits)
{
    uint64_t peers = ballot(e < experts);
    for (uint32_t b = 0; b < bits; ++b) {
        const bool one = (e >> b) & 1u;
        const uint64_t ones = ballot(one);
        peers &= one ? ones : ~ones;
    }
    return peers;
}

// TILES: the counts of all tiles are there; else this workgroup counts its own pairs first,
// which are all.
template <bool TILES>
__global__ __launch_bounds__(kSortThreads) void token_rank_kernel(SortArgs a)
{
    __shared__ uint32_t next[kSortExperts];  // the row of the expert's next pair
    __shared__ uint32_t all[kSortExperts];   // pairs of the expert in all tiles
    __shared__ uint32_t wave_sum[kSortWaves];
    __shared__ uint32_t count[kSortWaves][kSortExperts];
    const uint32_t tid = threadIdx.x, wave = tid / kWave, lane = lane_id();
    if (!TILES && a.status && tid == 0) *a.status = 0;
    for (uint32_t e = tid; e < kSortExperts; e += kSortThreads) next[e] = all[e] = 0;
    __syncthreads();
    if constexpr (TILES) {
        // several threads for each expert where there are few: each sums every parts-th tile
        const uint32_t parts = std::min(kSortThreads / a.experts, a.tiles);
        const uint32_t e = tid % a.experts, part = tid / a.experts;
        if (part < parts) {
            uint32_t before = 0, sum = 0;
            const uint32_t *counts = a.counts + e;
            for (uint32_t from = part; from < a.tiles; from += kSums * parts) {
                // (so many loads at once: one after the other they took 0.1 us a tile)
                uint32_t c[kSums] = {};
#pragma unroll
                for (uint32_t i = 0; i < kSums; ++i) {
                    if (from - part + i / 8 * 8 * parts >= a.tiles) continue;  // (none of these eight)
                    const uint32_t t = from + i * parts;
                    c[i] = counts[(t < a.tiles ? t : part) * a.experts];
                }
#pragma unroll
                for (uint32_t i = 0; i < kSums; ++i) {
                    const uint32_t t = from + i * parts;
                    sum += t < a.tiles ? c[i] : 0;
                    before += t < blockIdx.x ? c[i] : 0;
                }
            }
            __hip_atomic_fetch_add(&next[e], before, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            __hip_atomic_fetch_add(&all[e], sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
    } else {
        for (uint64_t p = tid; p < a.n; p += kSortThreads) {
            const uint32_t e = pair_expert(a, p);
            if (e < a.experts) __hip_atomic_fetch_add(&all[e], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
    }
    __syncthreads();
    // the experts' offsets: an expert for each thread
    const uint32_t mine = tid < kSortExperts ? all[tid] : 0;
    const uint32_t sum = wave_inclusive_scan(mine, SumOp());
    if (lane == kWave - 1) wave_sum[wave] = sum;
    __syncthreads();
    uint32_t offset = sum - mine;
    for (uint32_t w = 0; w < wave; ++w) offset += wave_sum[w];
    if (tid < a.experts) {
        next[tid] += offset;
        if (blockIdx.x == 0) {
            a.offsets[tid] = (int32_t)offset;
            if (tid == a.experts - 1) a.offsets[a.experts] = (int32_t)(offset + mine);
        }
    }
    const uint64_t first = (uint64_t)blockIdx.x * a.tile, last = first + a.tile < a.n ? first + a.tile : a.n;
    for (uint64_t base = first; base < last; base += kSortChunk) {
        for (uint32_t i = tid; i < kSortWaves * a.experts; i += kSortThreads) count[i / a.experts][i % a.experts] = 0;
        __syncthreads();
        const uint64_t from = base + wave * (kWave * kSortItems) + lane;
        uint32_t expert[kSortItems], rank[kSortItems];
#pragma unroll
        for (int i = 0; i < kSortItems; ++i) expert[i] = pair_expert(a, from + i * kWave);
#pragma unroll
        for (int i = 0; i < kSortItems; ++i) {
            const uint64_t peers = same_expert(expert[i], a.experts, a.bits);
            rank[i] = 0;
            if (expert[i] < a.experts) {
                const uint32_t below = mask_rank(peers);
                rank[i] = count[wave][expert[i]] + below;
            }
            wave_lds_sync();
            // (the last of them has the number of all)
            if (expert[i] < a.experts && (peers >> lane) == 1) count[wave][expert[i]] = rank[i] + 1;
            wave_lds_sync();
        }
        __syncthreads();
        if (tid < a.experts) {
            uint32_t row = next[tid];
#pragma unroll
            for (int w = 0; w < kSortWaves; ++w) {
                const uint32_t c = count[w][tid];
                count[w][tid] = row;
                row += c;
            }
            next[tid] = row;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kSortItems; ++i) {
            const uint64_t p = from + i * kWave;
            if (p >= last) continue;
            const uint32_t row = expert[i] < a.experts ? count[wave][expert[i]] + rank[i] : 0xFFFFFFFFu;
            a.positions[p] = (int32_t)row;
            if (a.sources && expert[i] < a.experts) a.sources[row] = (int32_t)p;
        }
        __syncthreads();
    }
}

uint32_t sort_tile(uint64_t n)
{
    return (uint32_t)(ceil_div(ceil_div(n, kSortTiles), kSortChunk) * kSortChunk);
}
// 0 where one workgroup sorts alone.
uint32_t sort_tiles(uint64_t n) { return n <= kSortAlone ? 0 : (uint32_t)ceil_div(n, sort_tile(n)); }
size_t sort_temp(uint64_t n, uint64_t experts)
{
    const uint32_t tiles = sort_tiles(n);
    return tiles ? kStatusBytes + align_up((uint64_t)tiles * experts * 4, 256) : 0;
}
bool index_ok(const int32_t *p) { return p && reinterpret_cast<uintptr_t>(p) % 4 == 0; }
bool sort_sizes(uint64_t tokens, uint64_t choices, uint64_t experts)
{
    return tokens <= 0x7FFFFFFFull && choices <= 0x7FFFFFFFull && tokens * choices <= 0x7FFFFFFFull && experts <= kSortExperts;
}

}  // namespace
}  // namespace lcpp

using namespace lcpp;

extern "C" int lcpp_token_sort_temp_bytes(uint64_t tokens, uint64_t choices, uint64_t experts, size_t *bytes)
{
    if (!bytes || !sort_sizes(tokens, choices, experts)) return LCPP_ERR_INVALID_ARG;
    *bytes = sort_temp(tokens * choices, experts);
    return LCPP_OK;
}

extern "C" int lcpp_token_sort(void *temp, size_t temp_bytes, const int32_t *experts, uint64_t tokens, uint64_t choices,
                               uint64_t num_experts, int32_t *positions, int32_t *offsets, int32_t *sources, void *stream)
{
    if (!sort_sizes(tokens, choices, num_experts)) return LCPP_ERR_INVALID_ARG;
    if (!index_ok(offsets) || num_experts == 0) return LCPP_ERR_INVALID_ARG;
    const uint64_t n = tokens * choices;
    if (n && (!index_ok(experts) || !index_ok(positions))) return LCPP_ERR_INVALID_ARG;
    if (sources && !index_ok(sources)) return LCPP_ERR_INVALID_ARG;
    if (positions == offsets || (sources && (sources == positions || sources == offsets || sources == experts)) || offsets == experts)
        return LCPP_ERR_INVALID_ARG;
    const size_t need = sort_temp(n, num_experts);
    if (need && !temp) return LCPP_ERR_INVALID_ARG;
    if (temp && reinterpret_cast<uintptr_t>(temp) % 256) return LCPP_ERR_INVALID_ARG;
    if (temp_bytes < need) return LCPP_ERR_TEMP_TOO_SMALL;
    SortArgs a = {};
    a.ids = experts, a.positions = positions, a.offsets = offsets, a.sources = sources;
    a.n = (uint32_t)n, a.experts = (uint32_t)num_experts;
    while ((1u << a.bits) < a.experts) ++a.bits;
    a.status = temp && temp_bytes >= kStatusBytes ? static_cast<uint32_t *>(temp) : nullptr;
    hipStream_t s = static_cast<hipStream_t>(stream);
    a.tiles = sort_tiles(n);
    if (a.tiles) {
        a.counts = reinterpret_cast<uint32_t *>(static_cast<char *>(temp) + kStatusBytes);
        a.tile = sort_tile(n);
        LCPP_LAUNCH("token_count", s, token_count_kernel<<<a.tiles, kSortThreads, 0, s>>>(a));
        LCPP_LAUNCH("token_rank", s, token_rank_kernel<true><<<a.tiles, kSortThreads, 0, s>>>(a));
    } else {
        a.tile = (uint32_t)kSortAlone;
        LCPP_LAUNCH("token_sort", s, token_rank_kernel<false><<<1, kSortThreads, 0, s>>>(a));
    }
    LCPP_CHECK_LAUNCH();
    return LCPP_OK;
}
