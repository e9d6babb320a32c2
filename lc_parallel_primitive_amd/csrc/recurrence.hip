// recurrence.hip — the gated linear recurrence h_t = a_t h_{t-1} + b_t over long
// sequences, per channel, its gradient, and its step for single tokens.
//
//   gate "decay":    a = g,          b = x
//   gate "log":      a = exp(g),     b = x
//   gate "sigmoid":  a = sigmoid(g), b = (1 - a) x = sigmoid(-g) x
//
// A step is the affine map h -> a h + b, and maps compose: rows r..s together
// are h -> A h + H with A the product of their a and H what they make of h = 0.
// So time is cut into tiles of kTileRows rows, a workgroup for each tile and 64
// lanes' channels: every wave takes kRows rows and folds them to (A, H), the waves
// meet in LDS, tiles by decoupled look-back, and with h before its first row in
// hand every wave runs through its rows, which wait in registers: the inputs
// are read once.
//
// Backward, with dh_t the whole gradient of h_t and e_t = a_t dh_t what of it
// reaches h_{t-1}:
//   dh_t = dy_t + e_{t+1},   e_t = a_t e_{t+1} + a_t dy_t
// which is a recurrence of the same form from the last row to the first, with the
// same products A; e past the last row is the gradient of the final state, and e
// of the first row is the gradient of the initial state.  The gate's gradient
// needs h_{t-1}: the forward pass keeps the state before each tile (one row in
// kTileRows, in 32 bits) and the backward tile runs through its rows again, which
// is exact to 32 bits and reads no output.
//   "decay":    dg = dh h_{t-1},                   dx = dh
//   "log":      dg = dh h_{t-1} a,                 dx = dh
//   "sigmoid":  dg = dh (h_{t-1} - x) a (1 - a),   dx = dh (1 - a)
//
// Bound by memory where there are chains enough.  bfloat16, us by kernel traces and
// TB/s of the bytes read and written once: 8 x 4096 x 2048 forward 81 (5.0), backward
// 138 (4.9); 1 x 65536 x 2048 forward 163 between events (4.95), 176 in a trace; a copy of
// as many bytes runs at 5.2.  Sequences of different lengths end with few tiles at
// work: 24 of them, 16391 rows x 1536 in all, 35 + 59 (4.3 both).  A single chain is bound
// by the look-back, 0.06 us a tile: 1 x 40000 x 64 forward 27, backward 29.5 between events.
// kRows and kWaves: a tile has to lie in registers at four waves a SIMD.  An earlier
// form's backward pass of 8 x 4096 x 2048 took 181 and 178 us with 18 and 20 rows a wave,
// 159 with 16; 8 rows a wave, sixteen waves, four channels a lane and tiles of 64 rows
// were slower too.
#include <algorithm>

#include "lookback.hpp"
#include "tensor.hpp"

namespace lcpp {
namespace {

constexpr int kRows = 16;  // rows of a wave
constexpr int kWaves = 8;  // waves of a full tile
constexpr int kTileRows = kRows * kWaves;

struct RowsIn {
    const void *p;
    uint64_t row, seq;  // strides in elements (seq 0 with begin and end)
};
struct RowsOut {
    void *p;
    uint64_t row, seq;
};
// One tile of a sequence that lies somewhere in the tensors' rows.
struct alignas(32) PackedTile {
    uint32_t seq, walk;  // walk: tiles of the sequence before this one in the walk
    uint32_t row, len;   // of the sequence
    uint32_t base;       // tiles of the sequences before it
};
constexpr uint32_t kNoSequence = 0xFFFFFFFFu;
struct RecArgs {
    RowsIn gate, in, grad_out;
    RowsOut out, grad_gate, grad_in;
    const float *initial, *grad_final;     // [sequence][channel]
    float *final_state, *grad_initial;     // [sequence][channel]
    float *checkpoints;                    // [tile of all sequences][channel]
    const uint32_t *begin, *end;           // null: sequence s begins at its stride, with max_length rows
    uint64_t rows;                         // with begin and end: rows of the tensors
    uint32_t sequences, tiles, groups, channels, max_length;
    uint32_t run, turns;                   // chains of a run (0: no runs); workgroups of a tile of time
    const PackedTile *list;                // with begin and end, sequences of several tiles: `all` tiles
    uint32_t all;
    uint64_t *words;                       // [sequence][tile of the walk][group][lane's channels]
    WaitCtl ctl;
    uint32_t *status;  // of temp storage that the call does not need, cleared by the kernel (may be null)
};

// ---------------------------------------------------------------- gates
struct GateDecay {
    static constexpr bool kShare = false;  // b is x itself
    __device__ static __forceinline__ void eval(float g, float &a, float &share) { a = g, share = 1.0f; }
    __device__ static __forceinline__ float grad(float dh, float before, float, float, float) { return dh * before; }
};
// (the native exponential: g log2(e) is rounded once, which is |g| roundings of the
// result; where that is much the result is small)
struct GateLog {
    static constexpr bool kShare = false;
    __device__ static __forceinline__ void eval(float g, float &a, float &share) { a = __expf(g), share = 1.0f; }
    __device__ static __forceinline__ float grad(float dh, float before, float, float a, float) { return dh * before * a; }
};
struct GateSigmoid {
    static constexpr bool kShare = true;
    // 1 - a is computed as sigmoid(-g): as a difference it would lose what a has
    // near 1.  exp(-|g|) cannot overflow.
    __device__ static __forceinline__ void eval(float g, float &a, float &share)
    {
        const float e = __expf(-fabsf(g)), r = __builtin_amdgcn_rcpf(1.0f + e), er = e * r;
        a = g >= 0.0f ? r : er;
        share = g >= 0.0f ? er : r;
    }
    __device__ static __forceinline__ float grad(float dh, float before, float x, float a, float share)
    {
        return dh * (before - x) * (a * share);
    }
};

// ---------------------------------------------------------------- tiles
// Where a workgroup's lanes work.  A lane has C channels; the last lane of an odd
// number of channels is moved back by one so that its channels lie inside the row,
// and computes and stores one of its neighbour's too, from the same loads: the
// same value.  Only where that neighbour is in another workgroup (`single`: the
// wave's one channel) is the other channel not stored, since an output over an
// input may already have been written there.  Every access is in bounds as long
// as there are C channels.
struct Place {
    uint32_t seq, tile, len, channel, group;
    uint32_t walk;    // tiles of the sequence before this one in the walk
    uint32_t base;    // tiles of the sequences before it, which its checkpoints come after
    uint32_t word_base;  // the same for the look-back words
    uint32_t number;  // of the tile among all, for the test hook
    bool active;   // the lane has a channel
    bool single;   // the first lane has one channel, the others none
    uint64_t row;  // of the tensors' rows that the sequence begins at (with offsets)
};
// The rows of sequence s, inside the tensors' rows and no more than max_length.
__device__ __forceinline__ void sequence_rows(const uint32_t *begin, const uint32_t *end, uint64_t rows, uint32_t max_length,
                                              uint32_t s, uint64_t &first, uint32_t &len)
{
    first = begin[s];
    const uint64_t last = end[s] < rows ? end[s] : rows;
    const uint64_t n = last > first ? last - first : 0;
    len = n < max_length ? (uint32_t)n : max_length;
}
constexpr uint32_t kXcds = 8;
// Workgroups are numbered tile by tile, so a tile waits only on workgroups
// dispatched before its own; `reverse` counts tiles from the sequence's end.
//
// Within a tile of time the chains (a sequence's groups of channels, one behind
// the other) are cut into runs, and each of the eight XCDs, which get the
// workgroups in turn, works on whole runs: where rows do not begin at a line of
// memory, neighbouring groups share lines, and their parts meet in one L2.  The
// runs go to another XCD at every tile.  Measured (us, forward + backward): 8 x
// 4096 x 2049 bfloat16 125 + 194 with runs of one chain, 98 + 164 with an eighth of
// all (1 x 65536 x 2048, whose rows begin at lines, 157 + 265 and 163 + 273); the latter
// 196 + 292 with the runs on one XCD at all tiles.  Sequences of different lengths have
// runs of 4, or the last one at work would leave XCDs idle (24 packed, 16391 rows: runs of 1,
// 4 and 16 of 1536 channels 36.5 + 57, 37 + 60, 38 + 60, of 1537 channels 53 + 74, 49 + 69, 47 + 69).
// Numbers past the last chain are left at once.
//
// Sequences of different lengths (offsets) have their tiles in a list, which the
// clearing launch makes from the offsets: there are no more than rows / 128 + sequences,
// however long the longest is.  The list is in the same order, the first tiles of
// (up to kListSequences) sequences, then the second tiles of those that have one, and
// so on.  Runs of four chains lie on one XCD there too, dealt out within windows of 8
// runs: a tile of a window may wait on one that is dispatched up to 31 workgroups
// after it, of which each XCD has four at most and room for many more.  Measured against
// the tiles of sequences x the longest, most of them empty (forward + backward): 24 x
// 16391 rows x 1536 bfloat16 40 + 60 -> 36 + 57, 256 x 65536 x 1024 120 + 166 -> 85 + 139, 256 x
// 262144 x 2048 with one of 32768 2255 + 2672 -> 655 + 1092.
template <int C>
__device__ __forceinline__ bool find_place(const RecArgs &a, bool reverse, Place &p)
{
    uint32_t tiles;
    if (a.list) {
        uint32_t item = blockIdx.x;
        if (a.run) {
            const uint32_t window = item / (kXcds * a.run), r = item - window * (kXcds * a.run), y = r / kXcds;
            item = (window * kXcds + (r + window + window / kXcds + window / (kXcds * kXcds)) % kXcds) * a.run + y;
        }
        p.number = item;
        const uint32_t at = item / a.groups;
        p.group = item - at * a.groups;
        if (at >= a.all) return false;
        const PackedTile t = a.list[at];
        if (t.seq == kNoSequence) return false;
        p.seq = t.seq, p.walk = t.walk, p.row = t.row, p.len = t.len;
        p.base = t.base;
        p.word_base = t.base - t.seq;  // (the last tile of a sequence has no words)
        tiles = (p.len + kTileRows - 1) / kTileRows;
    } else {
        const uint32_t k = blockIdx.x / a.turns, turn = blockIdx.x - k * a.turns;
        uint32_t chain = turn;
        if (a.run) {
            const uint32_t y = turn / kXcds;
            chain = (y / a.run * kXcds + (turn + k) % kXcds) * a.run + y % a.run;
        }
        p.seq = chain / a.groups;
        p.group = chain - p.seq * a.groups;
        if (p.seq >= a.sequences) return false;
        p.number = (k * a.sequences + p.seq) * a.groups + p.group;
        p.row = 0;
        p.len = a.max_length;
        if (a.begin) sequence_rows(a.begin, a.end, a.rows, a.max_length, p.seq, p.row, p.len);
        tiles = (p.len + kTileRows - 1) / kTileRows;
        p.walk = k;
        p.base = p.word_base = p.seq * a.tiles;
    }
    p.tile = reverse && tiles ? tiles - 1 - p.walk : p.walk;
    const uint32_t c = p.group * (kWave * C) + lane_id() * C;
    p.active = c < a.channels;
    p.channel = c + C <= a.channels ? c : a.channels - C;
    p.single = C > 1 && p.group > 0 && a.channels - p.group * (kWave * C) == 1;
    return true;
}
// (the wave's number as a scalar, so that row addresses are scalars too and a
// lane holds nothing but its channel's offset)
__device__ __forceinline__ uint32_t wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x / kWave); }
template <class T>
__device__ __forceinline__ const T *row_in(const RowsIn &t, const Place &p, uint64_t row)
{
    return static_cast<const T *>(t.p) + ((p.row + row) * t.row + p.seq * t.seq);
}

// A lane's address in a row: a scalar and a 32-bit offset.
template <class T>
__device__ __forceinline__ T *lane_at(T *row, uint32_t channel)
{
    using Byte = std::conditional_t<std::is_const_v<T>, const char, char>;
    return reinterpret_cast<T *>(reinterpret_cast<Byte *>(row) + (uint32_t)(channel * sizeof(T)));
}
template <class T>
__device__ __forceinline__ T *row_out(const RowsOut &t, const Place &p, uint64_t row)
{
    return static_cast<T *>(t.p) + ((p.row + row) * t.row + p.seq * t.seq);
}

// The packed look-back word of a channel: the map (A, H) of a tile (PARTIAL), or
// the state after it (INCLUSIVE), in one 64-bit store.  The upper half is A's
// bits inverted, so cleared memory is a NaN with all bits set, which no tile
// publishes (a NaN A is stored as 0x7FC00000); another such NaN marks a state.
constexpr uint32_t kWordState = 1;
__device__ __forceinline__ uint64_t word_map(float A, float H)
{
    const uint32_t bits = A == A ? __builtin_bit_cast(uint32_t, A) : 0x7FC00000u;
    return (uint64_t)~bits << 32 | __builtin_bit_cast(uint32_t, H);
}
__device__ __forceinline__ uint64_t word_state(float h)
{
    return (uint64_t)kWordState << 32 | __builtin_bit_cast(uint32_t, h);
}

template <int C>
struct Chan {
    float v[C];
};

// The state after a tile, or after a step: one rounding, the same wherever it is taken.
__device__ __forceinline__ float advance(float A, float h, float H) { return __builtin_fmaf(A, h, H); }

// The state before this tile: the walk goes back over the tiles' maps to the nearest
// state, and then forward again from it, one map after the other.  So the state is
// what each tile in turn makes of the one before it, whichever words the walk meets:
// the same bits at every call.  (Maps composed on the way back would be rounded in
// an order that depends on timing.)  The nearest map stays in registers and those
// after it in LDS; where kBack of them come before a state the walk waits there for
// it.  One wave calls it; `words` are those of this tile's channels, `step` is the
// distance to the tile before it, `before` the number of tiles there.
// The first poll reads one tile's words: as all chains advance together, the tile
// before has its state when its map is there, and a first window of 2, 4 or 8 tiles
// reads words that are not needed (an earlier form at 1 x 65536 x 2048: 195 us with one,
// 216, 240 and 270).  A walk that goes on reads kWindow at once (forward + backward, one at once ->
// four: 1 x 100000 x 512 float32 121 + 184 -> 113 + 184, 1 x 65536 x 2048 165 + 280 -> 163 +
// 273), and 32 KB of maps are 64 or 32 of them (1 x 40000 x 64 with 32 maps 30 + 32, with
// 64 27 + 29.5).  Maps composed on the way back, in no fixed order, took 112 + 183, 160 +
// 276 and 20 + 22 for these three.  More registers than these cost the backward pass of
// two channels a workgroup per CU.
template <int C>
constexpr uint32_t kBack = 64 / C;
constexpr uint32_t kWindow = 4;
template <int C>
struct Words {
    uint64_t v[C];
};
template <int C>
__device__ __forceinline__ void apply_words(const Words<C> &w, Chan<C> &h)
{
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t up = (uint32_t)(w.v[c] >> 32);
        const float H = __builtin_bit_cast(float, (uint32_t)w.v[c]);
        h.v[c] = up == kWordState ? H : advance(__builtin_bit_cast(float, ~up), h.v[c], H);
    }
}
// Whether a word can be taken: a state, or a map where the walk may go on; a channel
// that has met its state takes any.
template <int C>
__device__ __forceinline__ bool words_ready(const Words<C> &w, const bool (&done)[C], bool maps)
{
    bool ready = true;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t up = (uint32_t)(w.v[c] >> 32);
        ready = ready && (done[c] || up == kWordState || (up != 0 && maps));
    }
    return ballot(!ready) == 0;
}
template <int C>
__device__ __forceinline__ bool words_end(const Words<C> &w, bool (&done)[C])
{
    bool all = true;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        done[c] = done[c] || (uint32_t)(w.v[c] >> 32) == kWordState;
        all = all && done[c];
    }
    return ballot(!all) == 0;
}
template <int C>
__device__ __forceinline__ void load_words(const uint64_t *words, Words<C> &w)
{
#pragma unroll
    for (int c = 0; c < C; ++c) w.v[c] = ld_relaxed(words + c);
}
template <int C>
__device__ __forceinline__ Chan<C> look_back(const uint64_t *words, uint64_t step, uint32_t before,
                                             Words<C> (*maps)[kWave], const WaitCtl &ctl)
{
    const uint32_t lane = lane_id();
    Chan<C> h;
    bool done[C];
#pragma unroll
    for (int c = 0; c < C; ++c) h.v[c] = 0.0f, done[c] = false;
    uint32_t spins = 0;
    auto again = [&] {
        if (++spins >= ctl.spin_limit) {
            if (lane == 0) report_timeout(ctl);
            return false;
        }
        // (a tile's stores take longer than this; 1 x 65536 x 2048 takes the same with polls
        // at every 64 cycles, which only add to the traffic)
        __builtin_amdgcn_s_sleep(8);
        return true;
    };
    Words<C> near;
    words -= step;
    for (;;) {
        load_words(words, near);
        if (words_ready(near, done, true)) break;
        if (!again()) return h;
    }
    Words<C> far = near;
    bool end = words_end(near, done);
    const bool alone = end;
    uint32_t met = 0;  // maps in LDS, the nearest first
    while (!end) {
        // (the first tile has a state, so there is a tile before a walk that is not at its end)
        const uint32_t left = before - 1 - met, n = left < kWindow ? left : kWindow;
        Words<C> w[kWindow];
#pragma unroll
        for (uint32_t i = 0; i < kWindow; ++i) load_words(words - (i < n ? i + 1 : n) * step, w[i]);
        uint32_t took = 0;
        bool go = true;
#pragma unroll
        for (uint32_t i = 0; i < kWindow; ++i) {
            if (!go || i >= n) continue;
            go = words_ready(w[i], done, met < kBack<C>);
            if (!go) continue;
            far = w[i];
            end = words_end(w[i], done);
            go = !end;
            if (end) continue;
            maps[met++][lane] = w[i];
            ++took;
        }
        words -= took * step;
        if (!end && !took && !again()) return h;
    }
    // (a channel that was done nearer ends with that state)
    apply_words(far, h);
    while (met) {
        constexpr uint32_t kAtOnce = 4;
        const uint32_t n = met < kAtOnce ? met : kAtOnce;
        Words<C> m[kAtOnce];
#pragma unroll
        for (uint32_t i = 0; i < kAtOnce; ++i) m[i] = maps[met - 1 - (i < n ? i : n - 1)][lane];
#pragma unroll
        for (uint32_t i = 0; i < kAtOnce; ++i)
            if (i < n) apply_words(m[i], h);
        met -= n;
    }
    if (!alone) apply_words(near, h);
    return h;
}

// One wave publishes its tile's map, and then the state after it.
template <int C>
__device__ __forceinline__ void publish_map(uint64_t *words, const Chan<C> &A, const Chan<C> &H)
{
#pragma unroll
    for (int c = 0; c < C; ++c) st_relaxed(words + c, word_map(A.v[c], H.v[c]));
}
template <int C>
__device__ __forceinline__ void publish_state(uint64_t *words, const Chan<C> &A, const Chan<C> &H, const Chan<C> &h)
{
#pragma unroll
    for (int c = 0; c < C; ++c) st_relaxed(words + c, word_state(advance(A.v[c], h.v[c], H.v[c])));
}

// Rows that begin at a line of memory (STREAM) are read and written with the
// streaming policy: 8 x 4096 x 2048 bfloat16 82 + 136 us, without it 88 + 147; 4 x
// 512 x 1024 10.4 + 15.0 and 10.6 + 15.6.  Where neighbouring groups share lines
// these are better kept in the L2: of 2050 channels 113 + 197 us with the policy,
// 95 + 158 without it.
template <bool STREAM, int N, class T>
__device__ __forceinline__ Pack<T, N> load_rows_of(const T *p)
{
    if constexpr (STREAM) return load_pack_nt<N>(p);
    else return load_pack<N>(p);
}
template <bool STREAM, int N, class T>
__device__ __forceinline__ void store_rows_of(T *p, const float (&x)[N])
{
    if constexpr (STREAM) store_pack_nt<N>(p, x);
    else store_pack<N>(p, x);
}
// A lane's channels of a row or of a state, at the row's first channel.
template <bool STREAM, bool SINGLE, int C, class T>
__device__ __forceinline__ void store_own(T *row, const Place &p, const float (&x)[C])
{
    if constexpr (SINGLE) *lane_at(row, p.channel + C - 1) = (T)x[C - 1];
    else store_rows_of<STREAM, C>(lane_at(row, p.channel), x);
}
template <int C>
__device__ __forceinline__ void store_state(float *row, const Place &p, const Chan<C> &x)
{
    if (p.single) store_own<false, true>(row, p, x.v);
    else store_own<false, false>(row, p, x.v);
}
// f with whether the wave has a single channel as a constant: the loops over rows
// are made for either (a branch in them costs 5 % at 8 x 4096 x 2048).  Streamed
// rows have no odd channel.
template <bool STREAM, int C, class F>
__device__ __forceinline__ void with_single(const Place &p, F f)
{
    if constexpr (C > 1 && !STREAM) {
        if (p.single) {
            f(std::true_type{});
            return;
        }
    }
    f(std::false_type{});
}

template <class T, class G, int C, int W, bool STREAM>
__global__ __launch_bounds__(W *kWave) __attribute__((amdgpu_waves_per_eu(4))) void rec_forward_kernel(RecArgs a)
{
    __shared__ Chan<C> s_A[W][kWave], s_H[W][kWave], s_carry[kWave];
    constexpr bool kWalks = W == kWaves;  // (sequences of one tile have fewer waves)
    __shared__ Words<C> s_back[kWalks ? kBack<C> : 1][kWave];
    if (a.status && blockIdx.x == 0 && threadIdx.x == 0) *a.status = 0;
    Place p;
    if (!find_place<C>(a, false, p)) return;
    const uint32_t wave = wave_id(), lane = lane_id();
    const uint64_t state_row = (uint64_t)p.seq * a.channels, state_at = state_row + p.channel;
    const uint32_t first = p.tile * kTileRows + wave * kRows;
    const uint32_t last = p.len ? p.len - 1 : 0;
    const bool more = ((uint64_t)p.tile + 1) * kTileRows < p.len;  // a tile follows
    const uint64_t tile_words = (uint64_t)a.groups * kWave * C;
    uint64_t *words = a.words + ((uint64_t)p.word_base + p.walk) * tile_words + (uint64_t)p.group * kWave * C + lane * C;

    Chan<C> ga[kRows], gb[kRows], A, H;
    {
        Pack<T, C> gr[kRows], xr[kRows];
        if (p.len) {
            const T *g = row_in<T>(a.gate, p, first < last ? first : last), *x = row_in<T>(a.in, p, first < last ? first : last);
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                gr[r] = load_rows_of<STREAM, C>(lane_at(g, p.channel));
                xr[r] = load_rows_of<STREAM, C>(lane_at(x, p.channel));
                const bool next = first + r < last;  // (rows past the end read the last one and are not used)
                g += next ? a.gate.row : 0;
                x += next ? a.in.row : 0;
            }
        }
#pragma unroll
        for (int c = 0; c < C; ++c) A.v[c] = 1.0f, H.v[c] = 0.0f;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const bool in = first + r < p.len;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float al, share;
                G::eval(gr[r][c], al, share);
                ga[r].v[c] = in ? al : 1.0f;
                gb[r].v[c] = in ? (G::kShare ? share * xr[r][c] : xr[r][c]) : 0.0f;
                H.v[c] = ga[r].v[c] * H.v[c] + gb[r].v[c];
                A.v[c] *= ga[r].v[c];
            }
        }
    }
    s_A[wave][lane] = A;
    s_H[wave][lane] = H;
    __syncthreads();
    if (wave == 0) {
        const bool publish = more && p.number != a.ctl.withhold;
        if (publish) {
#pragma unroll
            for (int w = 1; w < W; ++w)
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    H.v[c] = s_A[w][lane].v[c] * H.v[c] + s_H[w][lane].v[c];
                    A.v[c] *= s_A[w][lane].v[c];
                }
            if (p.walk > 0) publish_map<C>(words, A, H);
        }
        Chan<C> h;
        if (!kWalks || p.walk == 0) {
#pragma unroll
            for (int c = 0; c < C; ++c) h.v[c] = a.initial ? a.initial[state_at + c] : 0.0f;
        } else {
            h = look_back<C>(words, tile_words, p.walk, s_back, a.ctl);
        }
        s_carry[lane] = h;
        if (publish) publish_state<C>(words, A, H, h);
        if (p.active) {
            if (a.checkpoints && p.len)
                store_state(a.checkpoints + ((uint64_t)p.base + p.tile) * a.channels, p, h);
            if (a.final_state && !p.len) store_state(a.final_state + state_row, p, h);
        }
    }
    __syncthreads();
    Chan<C> h = s_carry[lane];
    for (uint32_t w = 0; w < wave; ++w)
#pragma unroll
        for (int c = 0; c < C; ++c) h.v[c] = s_A[w][lane].v[c] * h.v[c] + s_H[w][lane].v[c];
    with_single<STREAM, C>(p, [&](auto single) {
        T *y = row_out<T>(a.out, p, first);
#pragma unroll
        for (int r = 0; r < kRows; ++r, y += a.out.row) {
#pragma unroll
            for (int c = 0; c < C; ++c) h.v[c] = ga[r].v[c] * h.v[c] + gb[r].v[c];
            if (first + r < p.len && p.active) store_own<STREAM, decltype(single)::value>(y, p, h.v);
        }
    });
    // (rows past the end left h as it was)
    if (a.final_state && p.active && p.len && first <= last && last - first < kRows)
        store_state(a.final_state + state_row, p, h);
}

// Makes the compiler forget where a value came from: what is computed from it
// before and after is computed twice instead of held in registers.
template <class T, int N>
__device__ __forceinline__ void forget(Pack<T, N> &x)
{
    if constexpr (sizeof(T) * N == 2) {
        uint16_t b = __builtin_bit_cast(uint16_t, x.v);
        asm volatile("" : "+v"(b));
        x.v = __builtin_bit_cast(decltype(x.v), b);
    } else if constexpr (sizeof(T) * N == 4) {
        uint32_t b = __builtin_bit_cast(uint32_t, x.v);
        asm volatile("" : "+v"(b));
        x.v = __builtin_bit_cast(decltype(x.v), b);
    } else {
        static_assert(sizeof(T) * N == 8, "2, 4 or 8 bytes");
        uint64_t b = __builtin_bit_cast(uint64_t, x.v);
        asm volatile("" : "+v"(b));
        x.v = __builtin_bit_cast(decltype(x.v), b);
    }
}

// The same tiles from the last to the first.  h before the tile is the forward
// pass's checkpoint, so only e is looked back for.
template <class T, class G, int C, int W, bool STREAM>
__global__ __launch_bounds__(W *kWave) void rec_backward_kernel(RecArgs a)
{
    __shared__ Chan<C> s_A[W][kWave], s_H[W][kWave], s_E[W][kWave], s_carry[kWave];
    constexpr bool kWalks = W == kWaves;  // (sequences of one tile have fewer waves)
    __shared__ Words<C> s_back[kWalks ? kBack<C> : 1][kWave];
    if (a.status && blockIdx.x == 0 && threadIdx.x == 0) *a.status = 0;
    Place p;
    if (!find_place<C>(a, true, p)) return;
    const uint32_t wave = wave_id(), lane = lane_id();
    const uint64_t state_row = (uint64_t)p.seq * a.channels, state_at = state_row + p.channel;
    if (p.len == 0) {  // nothing lies between the final and the initial state
        if (wave == 0 && a.grad_initial && p.active) {
            Chan<C> v;
#pragma unroll
            for (int c = 0; c < C; ++c) v.v[c] = a.grad_final ? a.grad_final[state_at + c] : 0.0f;
            store_state(a.grad_initial + state_row, p, v);
        }
        return;
    }
    const uint32_t first = p.tile * kTileRows + wave * kRows;
    const uint32_t last = p.len - 1;
    const uint64_t tile_words = (uint64_t)a.groups * kWave * C;
    uint64_t *words = a.words + ((uint64_t)p.word_base + p.walk) * tile_words + (uint64_t)p.group * kWave * C + lane * C;

    Pack<T, C> gr[kRows], xr[kRows], dyr[kRows];
    {
        const uint32_t t = first < last ? first : last;
        const T *g = row_in<T>(a.gate, p, t), *x = row_in<T>(a.in, p, t), *dy = row_in<T>(a.grad_out, p, t);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            gr[r] = load_rows_of<STREAM, C>(lane_at(g, p.channel));
            xr[r] = load_rows_of<STREAM, C>(lane_at(x, p.channel));
            dyr[r] = load_rows_of<STREAM, C>(lane_at(dy, p.channel));
            const bool next = first + r < last;  // (rows past the end read the last one and are not used)
            g += next ? a.gate.row : 0;
            x += next ? a.in.row : 0;
            dy += next ? a.grad_out.row : 0;
        }
    }
    // the wave's rows as one map, forward (A, H) and backward (A, E)
    Chan<C> A, H, E;
#pragma unroll
    for (int c = 0; c < C; ++c) A.v[c] = 1.0f, H.v[c] = 0.0f, E.v[c] = 0.0f;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        if (first + r < p.len) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float al, share;
                G::eval(gr[r][c], al, share);
                H.v[c] = al * H.v[c] + (G::kShare ? share * xr[r][c] : xr[r][c]);
                A.v[c] *= al;
                // e before the rows: the last row's share comes first, times all a up to it
                E.v[c] += A.v[c] * dyr[r][c];
            }
        }
    }
    s_A[wave][lane] = A;
    s_H[wave][lane] = H;
    s_E[wave][lane] = E;
    __syncthreads();
    if (wave == 0) {
        const bool publish = p.tile > 0 && p.number != a.ctl.withhold;
        if (publish) {
            A = s_A[W - 1][lane], E = s_E[W - 1][lane];
#pragma unroll
            for (int w = W - 2; w >= 0; --w)
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    E.v[c] = s_A[w][lane].v[c] * E.v[c] + s_E[w][lane].v[c];
                    A.v[c] *= s_A[w][lane].v[c];
                }
            if (p.walk > 0) publish_map<C>(words, A, E);
        }
        Chan<C> e;
        if (!kWalks || p.walk == 0) {
#pragma unroll
            for (int c = 0; c < C; ++c) e.v[c] = a.grad_final ? a.grad_final[state_at + c] : 0.0f;
        } else {
            e = look_back<C>(words, tile_words, p.walk, s_back, a.ctl);
        }
        s_carry[lane] = e;
        if (publish) publish_state<C>(words, A, E, e);
    }
    Chan<C> h, before[kRows];
    {
        const float *saved = a.checkpoints + ((uint64_t)p.base + p.tile) * a.channels + p.channel;
#pragma unroll
        for (int c = 0; c < C; ++c) h.v[c] = saved[c];
    }
    __syncthreads();
    Chan<C> e = s_carry[lane];
    for (uint32_t w = W - 1; w > wave; --w)
#pragma unroll
        for (int c = 0; c < C; ++c) e.v[c] = s_A[w][lane].v[c] * e.v[c] + s_E[w][lane].v[c];
    for (uint32_t w = 0; w < wave; ++w)
#pragma unroll
        for (int c = 0; c < C; ++c) h.v[c] = s_A[w][lane].v[c] * h.v[c] + s_H[w][lane].v[c];
    // (the gates are evaluated three times: kept, they would take half of the register file's waves)
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        before[r] = h;
        forget(gr[r]);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float al, share;
            G::eval(gr[r][c], al, share);
            h.v[c] = al * h.v[c] + (G::kShare ? share * xr[r][c] : xr[r][c]);
        }
    }
    with_single<STREAM, C>(p, [&](auto single) {
        T *pg = row_out<T>(a.grad_gate, p, first + kRows - 1), *px = row_out<T>(a.grad_in, p, first + kRows - 1);
#pragma unroll
        for (int r = kRows - 1; r >= 0; --r, pg -= a.grad_gate.row, px -= a.grad_in.row) {
            forget(gr[r]);
            if (first + r < p.len) {
                float dg[C], dx[C];
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    float al, share;
                    G::eval(gr[r][c], al, share);
                    const float dh = dyr[r][c] + e.v[c];
                    dg[c] = G::grad(dh, before[r].v[c], xr[r][c], al, share);
                    dx[c] = G::kShare ? dh * share : dh;
                    e.v[c] = al * dh;
                }
                if (p.active) {
                    store_own<STREAM, decltype(single)::value>(pg, p, dg);
                    store_own<STREAM, decltype(single)::value>(px, p, dx);
                }
            }
        }
    });
    if (p.tile == 0 && wave == 0 && a.grad_initial && p.active) store_state(a.grad_initial + state_row, p, e);
}

// One token for each of some sequences: h = a h + b on the states of a pool, at
// slots that the caller names (or one behind the other).  A slot outside the
// pool (a batch's padding) leaves every state alone and gives 0.
struct StepArgs {
    const void *gate, *in;
    void *out;
    uint64_t gate_stride, in_stride, out_stride;
    const float *state_in;
    float *state_out;
    const int32_t *slots;
    uint64_t num_slots;
    uint64_t items;  // octets of all sequences
    uint32_t channels, row_octets;
};
constexpr int kStepThreads = 256;
template <class T, class G>
__global__ __launch_bounds__(kStepThreads) void rec_step_kernel(StepArgs a)
{
    const uint64_t stride = (uint64_t)gridDim.x * kStepThreads;
    for (uint64_t item = (uint64_t)blockIdx.x * kStepThreads + threadIdx.x; item < a.items; item += stride) {
        const uint64_t seq = item / a.row_octets;
        const uint32_t col = (uint32_t)(item - seq * a.row_octets) * kOctet;
        const int64_t slot = a.slots ? (int64_t)a.slots[seq] : (int64_t)seq;
        float y[kOctet] = {};
        if (slot >= 0 && (uint64_t)slot < a.num_slots) {
            const Octet<T> g = load_octet(static_cast<const T *>(a.gate) + seq * a.gate_stride, col, a.channels);
            const Octet<T> x = load_octet(static_cast<const T *>(a.in) + seq * a.in_stride, col, a.channels);
            const Octet<float> h = load_octet(a.state_in + (uint64_t)slot * a.channels, col, a.channels);
#pragma unroll
            for (int i = 0; i < kOctet; ++i) {
                float al, share;
                G::eval(g[i], al, share);
                y[i] = al * h[i] + (G::kShare ? share * x[i] : x[i]);
            }
            store_octet(a.state_out + (uint64_t)slot * a.channels, col, a.channels, y);
        }
        store_octet(static_cast<T *>(a.out) + seq * a.out_stride, col, a.channels, y);
    }
}

// ---------------------------------------------------------------- the list of packed tiles
// A workgroup sorts kListSequences sequences by their tiles, c_0 >= c_1 >= ..: level k
// of the walk (their tile k) has as many entries as sequences have more than k tiles, so
// between c_{m+1} and c_m the levels have m + 1 each and an entry's level and sequence
// follow from its position by one search and one division.  Levels of sequences that
// come later in the tensors follow behind.  The sums over all sequences before these are
// made anew by every workgroup.  The other workgroups of the launch clear the status
// word and the look-back words.  Between events, which add some 4 us: for 24
// sequences of 16391 rows x 1536 in all 7.0 us, for 256 of 262144 x 2048, the longest of
// 32768, 14.6 (clearing the words of 256 sequences of that one's tiles took 220).
constexpr int kListSequences = 256;
struct ListArgs {
    const uint32_t *begin, *end;
    uint64_t rows;
    uint32_t max_length, sequences, all, builders, slices;
    PackedTile *list;
    uint64_t *status, *words;
    uint64_t count;  // words
};
__global__ __launch_bounds__(kListSequences) void rec_list_kernel(ListArgs a)
{
    constexpr uint32_t N = kListSequences;
    __shared__ uint32_t s_tiles[N + 1], s_sorted[N + 1], s_from[N], s_row[N], s_len[N];
    __shared__ uint64_t s_base[N + 1], s_start[N], s_wave[N / kWave], s_after[N + 1];
    const uint32_t t = threadIdx.x, wave = t / kWave;
    if (blockIdx.x >= a.builders) {
        const uint64_t at = (uint64_t)(blockIdx.x - a.builders) * N + t, stride = (uint64_t)(gridDim.x - a.builders) * N;
        if (at < kStatusBytes / 8) a.status[at] = 0;
        for (uint64_t i = at; i < a.count; i += stride) a.words[i] = 0;
        return;
    }
    const uint32_t block = blockIdx.x / a.slices, slice = blockIdx.x - block * a.slices, first = block * N;
    const uint32_t n = a.sequences - first < N ? a.sequences - first : N;
    auto tiles_of = [&](uint32_t seq, uint64_t &row, uint32_t &len) {
        sequence_rows(a.begin, a.end, a.rows, a.max_length, seq, row, len);
        return len ? (len + kTileRows - 1) / kTileRows : 1u;  // (an empty one's tile passes the state on)
    };
    uint64_t sum = 0;
    for (uint32_t i = t; i < first; i += N) {
        uint64_t row;
        uint32_t len;
        sum += tiles_of(i, row, len);
    }
    uint64_t row = 0;
    uint32_t len = 0;
    const uint32_t own = t < n ? tiles_of(first + t, row, len) : 0;
    s_tiles[t] = own, s_row[t] = (uint32_t)row, s_len[t] = len;
    // the sum over all sequences before these, and the sums over these up to each
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) sum += shfl_xor(sum, m);
    uint64_t scan = own;
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) {
        const uint64_t up = shfl_up(scan, m);
        scan += lane_id() >= (uint32_t)m ? up : 0;
    }
    if (lane_id() == kWave - 1) s_wave[wave] = sum, s_after[wave] = scan;
    __syncthreads();
    uint64_t before = 0, base = 0;
    for (uint32_t w = 0; w < N / kWave; ++w) {
        base += s_wave[w];
        before += w < wave ? s_after[w] : 0;
    }
    s_base[t] = base + before + scan - own;
    // place in the order of falling numbers of tiles
    uint32_t place = 0;
#pragma unroll 16
    for (uint32_t j = 0; j < n; ++j) place += s_tiles[j] > own || (s_tiles[j] == own && j < t) ? 1 : 0;
    __syncthreads();
    if (t < n) s_sorted[place] = own, s_from[place] = t;
    else s_sorted[t] = 0, s_from[t] = 0;
    if (t == 0) s_sorted[N] = 0;
    __syncthreads();
    // s_after[m]: the sum of sorted numbers from m on
    uint64_t rest = s_sorted[N - 1 - t];
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) {
        const uint64_t up = shfl_up(rest, m);
        rest += lane_id() >= (uint32_t)m ? up : 0;
    }
    if (lane_id() == kWave - 1) s_wave[wave] = rest;
    __syncthreads();
    for (uint32_t w = 0; w < wave; ++w) rest += s_wave[w];
    s_after[N - 1 - t] = rest;
    if (t == 0) s_after[N] = 0;
    __syncthreads();
    // where the levels with t + 1 entries begin
    s_start[t] = (uint64_t)(t + 1) * s_sorted[t + 1] + s_after[t + 1];
    __syncthreads();
    const uint64_t mine = s_after[0];
    const uint32_t words_end = a.all - a.sequences;
    for (uint64_t r = (uint64_t)slice * N + t; r < mine && base + r < a.all; r += (uint64_t)a.slices * N) {
        uint32_t lo = 0, hi = n - 1;  // the smallest m whose levels begin at r or before
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (s_start[mid] <= r) hi = mid;
            else lo = mid + 1;
        }
        const uint32_t at = (uint32_t)(r - s_start[lo]), level = at / (lo + 1), from = s_from[at - level * (lo + 1)];
        PackedTile e = {};
        e.seq = first + from, e.walk = s_sorted[lo + 1] + level, e.row = s_row[from], e.len = s_len[from];
        // Disjoint sequences have no more tiles than `all`.  Tiles past that are left
        // out, the later ones of a sequence with them, so that none waits for a tile
        // that there is not and none writes past the words.
        const uint64_t slot = s_base[from] + e.walk;
        const bool fits = slot < a.all && (e.walk + 1 == s_tiles[from] || slot - e.seq < words_end) &&
                          (e.walk == 0 || slot - 1 - e.seq < words_end);
        e.base = (uint32_t)s_base[from];
        if (!fits) e.seq = kNoSequence;
        a.list[base + r] = e;
    }
    if (first + N >= a.sequences) {
        for (uint64_t i = base + mine + (uint64_t)slice * N + t; i < a.all; i += (uint64_t)a.slices * N) a.list[i].seq = kNoSequence;
    }
}

// ---------------------------------------------------------------- launches
template <class F>
int gate_dispatch(lcpp_gate g, F f)
{
    switch (g) {
    case LCPP_GATE_DECAY: return f(GateDecay());
    case LCPP_GATE_LOG: return f(GateLog());
    case LCPP_GATE_SIGMOID: return f(GateSigmoid());
    default: return LCPP_ERR_INVALID_ARG;
    }
}

// Channels of a lane: two, so that a wave's row is 256 or 512 bytes; one where
// 64 lanes cover the channels.
uint32_t rec_lane_channels(uint64_t channels, size_t size) { return channels <= kWave || size == 4 ? 1 : 2; }
struct RecShape {
    uint64_t max_length, tiles, groups, run, turns;
    uint64_t all, grid, words;  // tiles of all sequences, workgroups, look-back words
    bool list;                  // packed, of several tiles
};
// `packed`: with offsets, of `rows` rows.
bool rec_shape(uint64_t sequences, uint64_t max_length, uint64_t channels, size_t size, bool packed, uint64_t rows, RecShape *r)
{
    if (sequences > 0xFFFFFFFFull || max_length > 0x7FFFFFFFull || channels > kMaxCols) return false;
    const uint64_t lanes = kWave * rec_lane_channels(channels, size);
    r->max_length = packed ? std::min(max_length, rows) : max_length;
    r->groups = ceil_div(channels, lanes);
    r->tiles = std::max<uint64_t>(ceil_div(r->max_length, kTileRows), 1);
    r->list = packed && r->tiles > 1;
    // workgroups are numbered in 32 bits, and a launch has less than 2^32 threads
    const uint64_t most = 0xFFFFFFFFull / (kWaves * kWave);
    if (r->groups && sequences > most / r->groups) return false;
    const uint64_t chains = sequences * r->groups;
    r->run = chains < kXcds ? 0 : ceil_div(chains, kXcds);
    if (packed) r->run = std::min<uint64_t>(r->run, 4);
    r->all = sequences * r->tiles;
    if (r->list) {
        r->all = std::min(r->all, rows / kTileRows + sequences);
        if (r->groups && r->all > most / r->groups) return false;
        r->turns = 0;
        r->grid = r->run ? align_up(r->all * r->groups, kXcds * r->run) : r->all * r->groups;
        r->words = (r->all - sequences) * r->groups * lanes;
        return r->grid <= most;
    }
    r->turns = r->run ? align_up(ceil_div(chains, r->run), kXcds) * r->run : chains;
    if (r->turns && r->tiles > most / r->turns) return false;
    r->grid = r->tiles * r->turns;
    r->words = r->tiles > 1 ? r->all * r->groups * lanes : 0;
    return true;
}
uint64_t rec_list_bytes(const RecShape &r) { return r.list ? align_up(r.all * sizeof(PackedTile), 256) : 0; }
uint64_t rec_temp_bytes(const RecShape &r)
{
    return r.tiles > 1 ? kStatusBytes + rec_list_bytes(r) + align_up(r.words * sizeof(uint64_t), 256) : 0;
}
// The larger of the types' sizes, of those whose call can be launched (2-byte types have
// half the workgroups), or false.
bool rec_most_bytes(uint64_t sequences, uint64_t max_length, uint64_t channels, bool packed, uint64_t rows, uint64_t *most)
{
    bool any = false;
    for (size_t size : {2, 4}) {
        RecShape r;
        if (!rec_shape(sequences, max_length, channels, size, packed, rows, &r)) continue;
        any = true;
        *most = std::max(*most, rec_temp_bytes(r));
    }
    return any;
}

template <class T, class G, int C, int W, bool STREAM>
int rec_launch_waves(bool forward, const RecArgs &a, uint32_t grid, hipStream_t s)
{
    if (forward) LCPP_LAUNCH("recurrence_forward", s, rec_forward_kernel<T, G, C, W, STREAM><<<grid, W * kWave, 0, s>>>(a));
    else LCPP_LAUNCH("recurrence_backward", s, rec_backward_kernel<T, G, C, W, STREAM><<<grid, W * kWave, 0, s>>>(a));
    LCPP_CHECK_LAUNCH();
    return LCPP_OK;
}
// Sequences of one tile take no more waves than have rows.
template <class T, class G, int C>
int rec_launch(bool forward, const RecArgs &a, uint32_t grid, hipStream_t s)
{
    if (a.max_length <= kRows) return rec_launch_waves<T, G, C, 1, false>(forward, a, grid, s);
    if (a.max_length <= 4 * kRows) return rec_launch_waves<T, G, C, 4, false>(forward, a, grid, s);
    constexpr uint64_t kLine = 128;
    auto lined = [](const void *p, uint64_t row, uint64_t seq) {
        return (reinterpret_cast<uintptr_t>(p) | row * sizeof(T) | seq * sizeof(T)) % kLine == 0;
    };
    auto in = [&](const RowsIn &t) { return lined(t.p, t.row, t.seq); };
    auto out = [&](const RowsOut &t) { return lined(t.p, t.row, t.seq); };
    // (sequences with offsets begin at whole rows; the tensors that a pass does not have are null)
    if (a.channels % C == 0 && in(a.gate) && in(a.in) && in(a.grad_out) && out(a.out) && out(a.grad_gate) && out(a.grad_in))
        return rec_launch_waves<T, G, C, kWaves, true>(forward, a, grid, s);
    return rec_launch_waves<T, G, C, kWaves, false>(forward, a, grid, s);
}

int rec_run(bool forward, lcpp_dtype t, lcpp_gate g, void *temp, size_t temp_bytes, RecArgs &a, uint64_t sequences,
            uint64_t max_length, uint64_t channels, uint64_t rows, hipStream_t s)
{
    const size_t e = float_size(t);
    if (!e) return LCPP_ERR_UNSUPPORTED_DTYPE;
    if (g != LCPP_GATE_DECAY && g != LCPP_GATE_LOG && g != LCPP_GATE_SIGMOID) return LCPP_ERR_INVALID_ARG;
    RecShape r;
    if (!rec_shape(sequences, max_length, channels, e, a.begin != nullptr, rows, &r) || (!a.begin) != (!a.end)) return LCPP_ERR_INVALID_ARG;
    if (sequences == 0 || channels == 0) return LCPP_OK;
    if (a.begin && (!elem_ok(a.begin, 4) || !elem_ok(a.end, 4))) return LCPP_ERR_INVALID_ARG;
    auto optional = [](const void *p) { return !p || elem_ok(p, 4); };
    if (!optional(a.initial) || !optional(a.final_state) || !optional(a.grad_final) || !optional(a.grad_initial) ||
        !optional(a.checkpoints))
        return LCPP_ERR_INVALID_ARG;
    const bool some = max_length != 0 && (!a.begin || rows != 0);  // (else only the states are copied)
    const uint64_t total = a.begin ? rows : max_length;
    auto out_ok = [&](const RowsOut &o) {
        return elem_ok(o.p, e) && rows_apart(o.row, total, channels) &&
               (a.begin || rows_apart(o.seq, sequences, channels));
    };
    if (some) {
        if (!elem_ok(a.gate.p, e) || !elem_ok(a.in.p, e)) return LCPP_ERR_INVALID_ARG;
        if (forward ? !out_ok(a.out) : !(elem_ok(a.grad_out.p, e) && out_ok(a.grad_gate) && out_ok(a.grad_in) && a.checkpoints))
            return LCPP_ERR_INVALID_ARG;
        if (!forward && same_place(a.grad_gate.p, a.grad_in.p)) return LCPP_ERR_INVALID_ARG;
    }
    const uint64_t need = rec_temp_bytes(r);
    if (need) {
        if (temp_bytes < need) return LCPP_ERR_TEMP_TOO_SMALL;
        if (!temp || (reinterpret_cast<uintptr_t>(temp) & 255)) return LCPP_ERR_INVALID_ARG;
    }
    a.run = (uint32_t)r.run, a.turns = (uint32_t)r.turns, a.all = (uint32_t)r.all;
    a.sequences = (uint32_t)sequences, a.tiles = (uint32_t)r.tiles, a.groups = (uint32_t)r.groups;
    a.channels = (uint32_t)channels, a.max_length = some ? (uint32_t)r.max_length : 0, a.rows = rows;
    if (a.begin) a.gate.seq = a.in.seq = a.grad_out.seq = a.out.seq = a.grad_gate.seq = a.grad_in.seq = 0;
    char *head = static_cast<char *>(temp);
    a.ctl = wait_ctl(need ? static_cast<uint32_t *>(temp) : nullptr);  // (one tile a sequence: nothing waits)
    if (!need && temp && temp_bytes >= kStatusBytes && !(reinterpret_cast<uintptr_t>(temp) & 255))
        a.status = static_cast<uint32_t *>(temp);
    if (need) a.words = reinterpret_cast<uint64_t *>(head + kStatusBytes + rec_list_bytes(r));
    if (r.list) {
        ListArgs l = {a.begin, a.end, rows, a.max_length, a.sequences, a.all, 0, 0, nullptr, nullptr, a.words, r.words};
        l.list = reinterpret_cast<PackedTile *>(head + kStatusBytes), l.status = reinterpret_cast<uint64_t *>(head);
        a.list = l.list;
        const uint64_t blocks = ceil_div(sequences, kListSequences);
        l.slices = (uint32_t)std::min<uint64_t>(ceil_div(r.all, blocks * kListSequences), 16);
        l.builders = (uint32_t)blocks * l.slices;
        const uint32_t grid = l.builders + (uint32_t)std::min<uint64_t>(ceil_div(r.words, kListSequences) + 1, 1024);
        LCPP_LAUNCH("recurrence_init", s, rec_list_kernel<<<grid, kListSequences, 0, s>>>(l));
        LCPP_CHECK_LAUNCH();
    } else if (need) {
        const int rc = lb_init(static_cast<uint64_t *>(temp), kStatusBytes / 8 + r.words, s, "recurrence_init");
        if (rc != LCPP_OK) return rc;
    }
    const uint32_t grid = (uint32_t)r.grid;
    return float_dispatch(t, [&](auto x) -> int {
        using T = decltype(x);
        return gate_dispatch(g, [&](auto gate) -> int {
            using G = decltype(gate);
            if constexpr (sizeof(T) == 2) {
                if (rec_lane_channels(channels, sizeof(T)) == 2) return rec_launch<T, G, 2>(forward, a, grid, s);
            }
            return rec_launch<T, G, 1>(forward, a, grid, s);
        });
    });
}

}  // namespace
}  // namespace lcpp

using namespace lcpp;

extern "C" int lcpp_recurrence_temp_bytes(uint64_t sequences, uint64_t max_length, uint64_t channels, size_t *bytes)
{
    if (!bytes) return LCPP_ERR_INVALID_ARG;
    uint64_t most = 0;
    const bool fixed = rec_most_bytes(sequences, max_length, channels, false, 0, &most);
    const bool packed = rec_most_bytes(sequences, max_length, channels, true, ~0ull, &most);
    if (!fixed && !packed) return LCPP_ERR_INVALID_ARG;
    *bytes = most;
    return LCPP_OK;
}

extern "C" int lcpp_recurrence_packed_temp_bytes(uint64_t sequences, uint64_t max_length, uint64_t channels, uint64_t rows,
                                                 size_t *bytes)
{
    uint64_t most = 0;
    if (!bytes || !rec_most_bytes(sequences, max_length, channels, true, rows, &most)) return LCPP_ERR_INVALID_ARG;
    *bytes = most;
    return LCPP_OK;
}

extern "C" int lcpp_recurrence_checkpoint_rows(uint64_t max_length, uint64_t *rows)
{
    if (!rows || max_length > 0x7FFFFFFFull) return LCPP_ERR_INVALID_ARG;
    *rows = std::max<uint64_t>(ceil_div(max_length, kTileRows), 1);
    return LCPP_OK;
}

extern "C" int lcpp_recurrence_packed_checkpoint_rows(uint64_t sequences, uint64_t max_length, uint64_t rows, uint64_t *out)
{
    RecShape r;
    if (!out || !rec_shape(sequences, max_length, 1, 2, true, rows, &r)) return LCPP_ERR_INVALID_ARG;
    *out = r.all;
    return LCPP_OK;
}

extern "C" int lcpp_recurrence_forward(lcpp_dtype t, lcpp_gate g, void *temp, size_t temp_bytes, const void *gate,
                                       uint64_t gate_row, uint64_t gate_seq, const void *in, uint64_t in_row,
                                       uint64_t in_seq, void *out, uint64_t out_row, uint64_t out_seq,
                                       const float *initial, float *final_state, float *checkpoints, uint64_t sequences,
                                       uint64_t max_length, uint64_t channels, const uint32_t *begin,
                                       const uint32_t *end, uint64_t rows, void *stream)
{
    RecArgs a = {};
    a.gate = {gate, gate_row, gate_seq}, a.in = {in, in_row, in_seq}, a.out = {out, out_row, out_seq};
    a.initial = initial, a.final_state = final_state, a.checkpoints = checkpoints, a.begin = begin, a.end = end;
    return rec_run(true, t, g, temp, temp_bytes, a, sequences, max_length, channels, rows,
                   static_cast<hipStream_t>(stream));
}

extern "C" int lcpp_recurrence_backward(lcpp_dtype t, lcpp_gate g, void *temp, size_t temp_bytes, const void *gate,
                                        uint64_t gate_row, uint64_t gate_seq, const void *in, uint64_t in_row,
                                        uint64_t in_seq, const float *checkpoints, const void *grad_out,
                                        uint64_t grad_out_row, uint64_t grad_out_seq, void *grad_gate,
                                        uint64_t grad_gate_row, uint64_t grad_gate_seq, void *grad_in,
                                        uint64_t grad_in_row, uint64_t grad_in_seq, const float *grad_final,
                                        float *grad_initial, uint64_t sequences, uint64_t max_length, uint64_t channels,
                                        const uint32_t *begin, const uint32_t *end, uint64_t rows, void *stream)
{
    RecArgs a = {};
    a.gate = {gate, gate_row, gate_seq}, a.in = {in, in_row, in_seq}, a.grad_out = {grad_out, grad_out_row, grad_out_seq};
    a.grad_gate = {grad_gate, grad_gate_row, grad_gate_seq}, a.grad_in = {grad_in, grad_in_row, grad_in_seq};
    a.checkpoints = const_cast<float *>(checkpoints), a.grad_final = grad_final, a.grad_initial = grad_initial;
    a.begin = begin, a.end = end;
    return rec_run(false, t, g, temp, temp_bytes, a, sequences, max_length, channels, rows,
                   static_cast<hipStream_t>(stream));
}

extern "C" int lcpp_recurrence_step(lcpp_dtype t, lcpp_gate g, const void *gate, uint64_t gate_stride, const void *in,
                                    uint64_t in_stride, const float *state_in, float *state_out, const int32_t *slots,
                                    uint64_t num_slots, void *out, uint64_t out_stride, uint64_t sequences,
                                    uint64_t channels, void *stream)
{
    const size_t e = float_size(t);
    if (!e) return LCPP_ERR_UNSUPPORTED_DTYPE;
    if (g != LCPP_GATE_DECAY && g != LCPP_GATE_LOG && g != LCPP_GATE_SIGMOID) return LCPP_ERR_INVALID_ARG;
    if (sequences > kMaxRows || channels > kMaxCols || num_slots > kMaxRows) return LCPP_ERR_INVALID_ARG;
    if (sequences == 0 || channels == 0) return LCPP_OK;
    if (!elem_ok(gate, e) || !elem_ok(in, e) || !elem_ok(out, e) || !rows_apart(out_stride, sequences, channels))
        return LCPP_ERR_INVALID_ARG;
    if (!elem_ok(state_in, 4) || !elem_ok(state_out, 4) || (slots && !elem_ok(slots, 4)) || (!slots && num_slots < sequences))
        return LCPP_ERR_INVALID_ARG;
    StepArgs a = {gate, in, out, gate_stride, in_stride, out_stride, state_in, state_out, slots, num_slots, 0, 0, 0};
    a.channels = (uint32_t)channels;
    a.row_octets = (uint32_t)ceil_div(channels, kOctet);
    a.items = sequences * a.row_octets;
    const uint32_t grid = (uint32_t)std::min<uint64_t>(ceil_div(a.items, kStepThreads), 1u << 20);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return float_dispatch(t, [&](auto x) -> int {
        using T = decltype(x);
        return gate_dispatch(g, [&](auto kind) -> int {
            using G = decltype(kind);
            LCPP_LAUNCH("recurrence_step", s, rec_step_kernel<T, G><<<grid, kStepThreads, 0, s>>>(a));
            LCPP_CHECK_LAUNCH();
            return LCPP_OK;
        });
    });
}
