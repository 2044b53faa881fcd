// Embedding lookup with scaling, and the gradient of the table:
//   out_n = scale weight[id_n],   gw_v = scale sum over the n with id_n = v, in their order, of g_n
// The gradient of more than a few positions orders them by their tokens (equal ones by position, so that a row's terms come in one order
// whatever runs first), then adds every run of equal tokens: no atomics on floats, the same bits at every call.
//
// Bound by the writes: a whole gradient of 50304 rows is one fill of the card's memory (206 MB of 2048 bfloat16 columns: 31 us by 16
// bytes a thread, 6.7 TB/s; stores that pass the caches by are faster where nobody reads the gradient next, 59 -> 53 us for 8192 tokens, and slower with who
// does: with its norm 79 -> 95). Measured, us of the kernels: 8192 tokens into 50304 x 2048 bfloat16 12 + 45 (240
// MB: 4.2 TB/s), 512 into 50304 x 1024 float32 33 to 40 in one (5.2 to 6.2), 3001 of 1001 float32 channels into a gradient that is there 6 + 12;
// the lookup of one token 1.6, a launch; of 8192 tokens of 2048 14 bfloat16 (67 MB: 4.9 TB/s), 24.5 float32 (134 MB: 5.5).
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "launch.hpp"

namespace hffn {
namespace {

__device__ __forceinline__ int64_t id_at(const EmbeddingIds& ids, uint32_t i) {
    const int64_t at = static_cast<int64_t>(i) * ids.stride;
    const int64_t id = ids.wide ? static_cast<const int64_t*>(ids.p)[at] : static_cast<const int32_t*>(ids.p)[at];
    return id < 0 ? id + ids.end : id;
}

// The token of position i, ~0 where it has no row (outside the vocabulary, or the padding).
__device__ __forceinline__ uint32_t token_at(const EmbeddingGradient& a, uint32_t i) {
    const int64_t id = id_at(a.ids, i);
    return id >= 0 && id < a.vocab && id != a.padding ? static_cast<uint32_t>(id) : ~0u;
}

// A lane's share of one slice (64 E columns) of a row of d entries: 16 bytes of it, or, where rows start anywhere or end inside
// 16 bytes (not WHOLE), E entries 64 columns apart.
template <typename T, bool WHOLE>
struct Lane {
    static constexpr int E = 16 / sizeof(T);
    static constexpr uint32_t SLICE = kWave * E;
    typedef typename std::conditional<WHOLE, uint4, T>::type Raw;
    static constexpr int R = WHOLE ? 1 : E;
    struct Share { Raw raw[R]; };
    uint32_t first, d;
    __device__ __forceinline__ Lane(uint32_t slice, uint32_t lane, uint32_t d) : first(slice * SLICE + lane * (WHOLE ? E : 1)), d(d) {}
    __device__ __forceinline__ void load(const T* row, Share& to) const {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (first + r * kWave < d) to.raw[r] = *reinterpret_cast<const Raw*>(row + first + r * kWave);
            else if constexpr (WHOLE) to.raw[r] = make_uint4(0, 0, 0, 0);
            else to.raw[r] = 0;
        }
    }
    __device__ __forceinline__ static void widened(const Share& from, float (&to)[E]) {
        if constexpr (!WHOLE) {
#pragma unroll
            for (int e = 0; e < E; ++e) to[e] = widen(from.raw[e]);
        } else {
            const uint32_t words[4] = {from.raw[0].x, from.raw[0].y, from.raw[0].z, from.raw[0].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (sizeof(T) == 4) {
                    to[k] = __uint_as_float(words[k]);
                } else {
                    to[2 * k] = __uint_as_float(words[k] << 16);
                    to[2 * k + 1] = __uint_as_float(words[k] & 0xffff0000u);
                }
            }
        }
    }
    __device__ __forceinline__ void store(T* row, const float (&from)[E]) const {
        if constexpr (WHOLE) {
            if (first >= d) return;
            if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(row + first) = make_float4(from[0], from[1], from[2], from[3]);
            else
                *reinterpret_cast<uint4*>(row + first) =
                    make_uint4(bf16_pair(from[0], from[1]), bf16_pair(from[2], from[3]), bf16_pair(from[4], from[5]), bf16_pair(from[6], from[7]));
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (first + e * kWave >= d) continue;
                if constexpr (sizeof(T) == 4) row[first + e * kWave] = from[e];
                else row[first + e * kWave] = bf16_bits(from[e]);
            }
        }
    }
};

// A wave takes one slice of ROWS rows: ids first, then every row's request, then the stores. The id is read by every slice of its row, from the
// caches.
constexpr uint32_t kLookupThreads = 256;
template <typename T, bool WHOLE, int ROWS>
__global__ __launch_bounds__(kLookupThreads) void lookup_kernel(EmbeddingForward a, uint32_t slices) {
    using L = Lane<T, WHOLE>;
    const uint32_t job = uniform(blockIdx.x * (kLookupThreads / kWave) + threadIdx.x / kWave), first = job / slices * ROWS;
    if (first >= a.n) return;
    const L lane(job % slices, threadIdx.x % kWave, a.d);
    int64_t id[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) id[k] = first + k < a.n ? id_at(a.ids, first + k) : -1;
    typename L::Share share[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k)
        if (id[k] >= 0 && id[k] < a.vocab) lane.load(static_cast<const T*>(a.weight) + id[k] * a.d, share[k]);
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
        if (first + k >= a.n) break;
        float v[L::E];
        if (id[k] >= 0 && id[k] < a.vocab) {
            L::widened(share[k], v);
#pragma unroll
            for (int e = 0; e < L::E; ++e) v[e] *= a.scale;
        } else {
#pragma unroll
            for (int e = 0; e < L::E; ++e) v[e] = __builtin_nanf("");
            if (a.outside != nullptr) *a.outside = 1;
        }
        lane.store(static_cast<T*>(a.out) + static_cast<uint64_t>(first + k) * a.d, v);
    }
}

// ------------------------------------------------------------------------------------------------------- the order

// A position's place in its chunk's order by token (equal tokens in the order of the positions): the number of positions before it, counted
// one by one, 2 N^2 / 64 instructions over the whole card, 4 us of it for 8192 tokens (the launch 11), where a sort by digits in one
// block is a chain of passes (25 us). A block takes 32 positions, two lanes each (for the even and the odd 64s of the chunk's keys, which lie in
// LDS), its waves a part of the chunk each. Tokens without a row (outside the vocabulary, the padding) take the key `vocab` and come
// last. where[token] is the place of one of its positions; elsewhere it holds anything.
constexpr uint32_t kRankThreads = 1024, kRankWaves = kRankThreads / kWave, kChunk = 16384, kOwn = kWave / 2;
__global__ __launch_bounds__(kRankThreads) void rank_kernel(EmbeddingIds ids, uint32_t n, uint32_t vocab, int64_t padding, uint32_t* __restrict__ sorted,
                                                            uint32_t* __restrict__ places, uint32_t* __restrict__ where, uint32_t* __restrict__ counters,
                                                            uint32_t counter_count) {
    extern __shared__ __attribute__((aligned(16))) uint32_t keys[];  // the chunk's, up to a multiple of 64 of them
    __shared__ uint32_t counts[kRankWaves][kWave];
    for (uint32_t i = blockIdx.x * kRankThreads + threadIdx.x; i < counter_count; i += gridDim.x * kRankThreads) counters[i] = 0;
    const uint32_t lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave), per = kChunk / kOwn, chunk = blockIdx.x / per, block = blockIdx.x % per;
    const uint32_t base = chunk * kChunk, count = n - base < kChunk ? n - base : kChunk, groups = (count + kWave - 1) / kWave;
    for (uint32_t i = threadIdx.x; i < groups * kWave; i += kRankThreads) {
        uint32_t key = ~0u;
        if (i < count) {
            const int64_t id = id_at(ids, base + i);
            key = id >= 0 && id < vocab && id != padding ? static_cast<uint32_t>(id) : vocab;
        }
        keys[i] = key;
    }
    __syncthreads();
    const uint32_t mine = block * kOwn + lane % kOwn, key = keys[mine], own = mine / kWave;
    uint32_t before = 0;
    for (uint32_t g = 2 * wave + lane / kOwn; g < groups; g += 2 * kRankWaves) {
        const uint4* const from = reinterpret_cast<const uint4*>(keys + g * kWave);
        const uint32_t bound = g < own ? key + 1 : key;  // equal tokens of earlier positions come before
#pragma unroll 4
        for (uint32_t j = 0; j < kWave / 4; ++j) {
            const uint4 v = from[j];
            before += (v.x < bound) + (v.y < bound) + (v.z < bound) + (v.w < bound);
        }
    }
    if (wave == 0 && lane < kOwn) {  // the equal ones before it in its own 64
        const uint4* const from = reinterpret_cast<const uint4*>(keys + own * kWave);
        const uint32_t end = mine - own * kWave;
#pragma unroll 4
        for (uint32_t j = 0; j < kWave / 4; ++j) {
            const uint4 v = from[j];
            before += (v.x == key && 4 * j < end) + (v.y == key && 4 * j + 1 < end) + (v.z == key && 4 * j + 2 < end) + (v.w == key && 4 * j + 3 < end);
        }
    }
    counts[wave][lane] = before;
    __syncthreads();
    if (wave != 0 || lane >= kOwn || mine >= count) return;
    uint32_t to = base;
#pragma unroll
    for (uint32_t w = 0; w < kRankWaves; ++w) to += counts[w][lane] + counts[w][lane + kOwn];
    sorted[to] = key;
    places[to] = base + mine;
    if (where != nullptr && key < vocab) where[key] = to;
}

// Sorted chunks to one order: an entry's place is its own in its chunk and, in every other, the number of entries before it:
// those of smaller keys, and of equal ones in the chunks that come before its own.
constexpr uint32_t kMergeThreads = 256;
__global__ __launch_bounds__(kMergeThreads) void merge_kernel(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ places, uint32_t n, uint32_t chunk,
                                                              uint32_t* __restrict__ sorted, uint32_t* __restrict__ order, uint32_t* __restrict__ where,
                                                              uint32_t vocab) {
    const uint32_t i = blockIdx.x * kMergeThreads + threadIdx.x;
    if (i >= n) return;
    const uint32_t key = keys[i], own = i / chunk;
    uint32_t to = i - own * chunk;
    for (uint32_t c = 0, first = 0; first < n; ++c, first += chunk) {
        if (c == own) continue;
        const uint32_t before = c < own ? key + 1 : key;  // entries below this come first
        uint32_t low = first, high = first + chunk < n ? first + chunk : n;
        while (low < high) {
            const uint32_t middle = (low + high) / 2;
            if (keys[middle] < before) low = middle + 1;
            else high = middle;
        }
        to += low - first;
    }
    sorted[to] = key;
    order[to] = places[i];
    if (where != nullptr && key < vocab) where[key] = to;
}

// ------------------------------------------------------------------------------------------------------- sums

// A wave takes the runs that begin in `window` (4 at most) sorted positions, one slice of the columns: it walks their rows one after
// the other, U requested at a time, and writes a sum where the next token begins. A run of more than 64 positions is cut into pieces
// of 64 from its head on, each the whole block's whose positions it begins in (16 waves with 4 rows each, added in order); the
// block that ends a run's last piece adds them up, in order too. The rows' order and these cuts depend on the run alone. Behind the
// blocks that add come those that fill the other rows with zeros: what the long runs wait for passes beside that. (All rows
// filled beside the order instead: 60 us for 51 with 8192 positions, 42 for 40 with 4096.)
constexpr uint32_t kSumThreads = 1024, kSumWaves = kSumThreads / kWave, kRun = 64, kShare = kRun / kSumWaves;
constexpr uint32_t kWindow = 4;
static_assert(kWindow * kSumWaves <= kRun, "at most one long run begins in a block, and at most one piece of an earlier one");

// The first position in [low, high) whose key is not below `bound` (high: none); 64 probes at a time.
__device__ __forceinline__ uint32_t first_from(const uint32_t* __restrict__ sorted, uint32_t low, uint32_t high, uint32_t bound, uint32_t lane) {
    while (low < high) {
        const uint32_t stride = (high - low + kWave - 1) / kWave, at = low + lane * stride + stride - 1;
        const uint32_t less = static_cast<uint32_t>(__popcll(__ballot(at < high && sorted[at] < bound)));
        low += less * stride;
        high = low + stride - 1 < high ? low + stride - 1 : high;
    }
    return low;
}

// Zeros in the rows without a position, 64 KB by a block, in pieces of 16 bytes; one that belongs to several rows goes entry by entry where
// one of them has a position. Rows within the block's entries are told by a product with 2^32 / d, rounded up: below 2^16 entries
// and 2^15 a row it is exact.
template <typename T>
struct Fill {
    static constexpr uint32_t U = 4, E = 16 / sizeof(T), kEntries = U * kSumThreads * E;
    uint64_t begin;
    uint32_t first_row, inside, rest, inverse, d;
    T* gw;
    bool aligned;
    __device__ __forceinline__ Fill(const EmbeddingGradient& a, uint32_t block) : begin(static_cast<uint64_t>(block) * kEntries), d(a.d) {
        const uint64_t entries = static_cast<uint64_t>(a.vocab) * d;
        first_row = static_cast<uint32_t>(begin / d);
        inside = static_cast<uint32_t>(begin - static_cast<uint64_t>(first_row) * d);
        rest = entries - begin < kEntries ? static_cast<uint32_t>(entries - begin) : kEntries;
        inverse = d == 1 ? 0 : 0xffffffffu / d + 1;
        gw = static_cast<T*>(a.gw) + begin;
        aligned = reinterpret_cast<uintptr_t>(a.gw) % 16 == 0;
    }
    __device__ __forceinline__ uint32_t row_of(uint32_t entry) const { return first_row + (d == 1 ? entry : __umulhi(inside + entry, inverse)); }
    __device__ __forceinline__ static uint32_t entry(uint32_t u) { return (u * kSumThreads + threadIdx.x) * E; }
    __device__ __forceinline__ void rows(uint32_t u, uint32_t& row, uint32_t& next) const {  // of piece u's ends
        row = row_of(entry(u) < rest ? entry(u) : rest - 1);
        next = row_of(entry(u) + E - 1 < rest ? entry(u) + E - 1 : rest - 1);
    }
    __device__ __forceinline__ bool whole(uint32_t u) const { return aligned && entry(u) + E <= rest; }
    __device__ __forceinline__ void zero(uint32_t u) const { *reinterpret_cast<uint4*>(gw + entry(u)) = make_uint4(0, 0, 0, 0); }
    template <typename HAS>
    __device__ __forceinline__ void zero_without(uint32_t u, HAS&& has) const {
        for (uint32_t e = 0; e < E && entry(u) + e < rest; ++e)
            if (!has(row_of(entry(u) + e))) gw[entry(u) + e] = 0;
    }
};

// A row has a position if the place that `where` gives, whatever that may be, holds it.
template <typename T>
__device__ __forceinline__ void fill_rows(const EmbeddingGradient& a, const uint32_t* __restrict__ sorted, const uint32_t* __restrict__ where, uint32_t block) {
    typedef Fill<T> F;
    const F fill(a, block);
    const auto has = [&](uint32_t row, uint32_t place) { return place < a.n && sorted[place] == row; };
    uint32_t row[F::U], next[F::U], at[F::U], at_next[F::U];
#pragma unroll
    for (uint32_t u = 0; u < F::U; ++u) {
        fill.rows(u, row[u], next[u]);
        at[u] = where[row[u]];
        at_next[u] = next[u] == row[u] ? at[u] : where[next[u]];
    }
    bool none[F::U];
#pragma unroll
    for (uint32_t u = 0; u < F::U; ++u) none[u] = !has(row[u], at[u]) && (next[u] == row[u] || !has(next[u], at_next[u]));
#pragma unroll
    for (uint32_t u = 0; u < F::U; ++u) {
        if (fill.entry(u) >= fill.rest) break;
        if (none[u] && next[u] <= row[u] + 1 && fill.whole(u)) fill.zero(u);
        else if (none[u] || next[u] != row[u]) fill.zero_without(u, [&](uint32_t of) { return has(of, where[of]); });
    }
}

// The rows in lanes [at, end) of `place` added to acc one after the other; before(j) comes before row j is added.
template <typename T, bool WHOLE, typename BEFORE>
__device__ __forceinline__ void walk(const EmbeddingGradient& a, const Lane<T, WHOLE>& column, uint32_t place, uint32_t at, uint32_t end,
                                     float (&acc)[Lane<T, WHOLE>::E], BEFORE&& before) {
    typedef Lane<T, WHOLE> L;
    constexpr int U = WHOLE ? 4 : 16 / L::E;
    for (uint32_t j = at; j < end; j += U) {
        typename L::Share share[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (j + u < end) {
                const uint32_t row = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(place), j + u));
                column.load(static_cast<const T*>(a.g) + row * a.g_stride, share[u]);
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (j + u < end) {
                before(j + u);
                float v[L::E];
                L::widened(share[u], v);
#pragma unroll
                for (int e = 0; e < L::E; ++e) acc[e] += v[e];
            }
    }
}
// A token's sum to its row; acc is zero afterwards.
template <bool INTO, typename T, bool WHOLE>
__device__ __forceinline__ void finish(const EmbeddingGradient& a, const Lane<T, WHOLE>& column, uint32_t token, float (&acc)[Lane<T, WHOLE>::E]) {
    typedef Lane<T, WHOLE> L;
    T* const row = static_cast<T*>(a.gw) + static_cast<uint64_t>(token) * a.d;
    if constexpr (INTO) {
        typename L::Share old;
        column.load(row, old);
        float v[L::E];
        L::widened(old, v);
#pragma unroll
        for (int e = 0; e < L::E; ++e) acc[e] = fmaf(a.scale, acc[e], v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < L::E; ++e) acc[e] *= a.scale;
    }
    column.store(row, acc);
#pragma unroll
    for (int e = 0; e < L::E; ++e) acc[e] = 0.0f;
}
// Every wave's acc, in order, to wave 0's.
template <int E>
__device__ __forceinline__ void join_waves(float (&lds)[kSumWaves][E][kWave], uint32_t wave, uint32_t lane, float (&acc)[E]) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) lds[wave][e][lane] = acc[e];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        acc[e] = 0.0f;
#pragma unroll 4
        for (uint32_t v = 0; v < kSumWaves; ++v) acc[e] += lds[v][e][lane];
    }
}

template <typename T, bool WHOLE, bool INTO>
__global__ __launch_bounds__(kSumThreads, 8) void sums_kernel(EmbeddingGradient a, const uint32_t* __restrict__ sorted, const uint32_t* __restrict__ places,
                                                              uint32_t window, uint32_t* counters, float* partials, const uint32_t* __restrict__ where, uint32_t slices, uint32_t summers) {
    using L = Lane<T, WHOLE>;
    constexpr int E = L::E;
    __shared__ float lds[kSumWaves][E][kWave];
    __shared__ uint32_t long_first, long_end, last_piece;
    if constexpr (!INTO)
        if (blockIdx.x >= summers) {
            fill_rows<T>(a, sorted, where, blockIdx.x - summers);
            return;
        }
    const uint32_t block_at = blockIdx.x / slices, slice = blockIdx.x % slices;
    const uint32_t lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave), block = window * kSumWaves, from = block_at * block, begin = from + wave * window;
    const L column(slice, lane, a.d);
    const auto nothing = [](uint32_t) {};
    const uint32_t i = begin + lane, key = i < a.n ? sorted[i] : ~0u, before = i > 0 && i <= a.n ? sorted[i - 1] : ~0u, place = i < a.n ? places[i] : 0;
    const uint64_t heads = __ballot(i < a.n && key < a.vocab && (i == 0 || key != before)), mine = heads & ((1ull << window) - 1);
    const auto key_at = [&](uint32_t at) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(key), at)); };
    if (threadIdx.x == 0) long_first = ~0u;
    __syncthreads();
    if (mine != 0) {
        const uint32_t first = __ffsll(static_cast<long long>(mine)) - 1, last = 63 - __clzll(static_cast<long long>(mine)), last_token = key_at(last);
        uint32_t end = last + static_cast<uint32_t>(__popcll(__ballot(i < a.n && key == last_token)));  // of the last run, from begin on
        if (end == kWave && begin + kWave < a.n) end = first_from(sorted, begin + kWave, a.n, last_token + 1, lane) - begin;  // it goes on behind the keys at hand
        const bool whole_block = end - last > kRun;
        if (whole_block && lane == 0) {
            long_first = begin + last;
            long_end = begin + end;
        }
        const uint32_t stop = whole_block ? last : end;
        if (stop > first) {
            float acc[E] = {};
            uint32_t token = key_at(first);
            walk(a, column, place, first, stop < kWave ? stop : kWave, acc, [&](uint32_t j) {
                if (j == first || !(mine >> j & 1)) return;
                finish<INTO>(a, column, token, acc);
                token = key_at(j);
            });
            if (stop > kWave) walk(a, column, lane < stop - kWave ? places[begin + kWave + lane] : 0, 0, stop - kWave, acc, nothing);
            finish<INTO>(a, column, token, acc);
        }
    }
    __syncthreads();
    // The long run that begins here, then the one that the block's first position lies in, if any: a piece of [head, end), from `start` on.
#pragma unroll 1
    for (int turn = 0; turn < 2; ++turn) {
        uint32_t head, end, start;
        if (turn == 0) {
            head = start = uniform(long_first);
            end = uniform(long_end);
            if (head == ~0u) continue;
        } else {
            if (from == 0 || from >= a.n) return;
            const uint32_t here = uniform(sorted[from]);
            if (here >= a.vocab || uniform(sorted[from - 1]) != here) return;
            head = first_from(sorted, 0, from, here, lane);
            end = first_from(sorted, from, a.n, here + 1, lane);
            start = head + (from - head + kRun - 1) / kRun * kRun;
            if (end - head <= kRun || start >= end || start >= from + block) return;
            __syncthreads();
        }
        const uint32_t stop = start + kRun < end ? start + kRun : end, own = start + wave * kShare, count = own < stop ? stop - own : 0;
        const uint32_t pieces = (end - head + kRun - 1) / kRun, token = uniform(sorted[head]);
        const auto slot = [&](uint32_t j) {  // where piece j's sums lie: a block has one of a run that it begins and one of another
            return partials + (2ull * ((head + j * kRun) / block) + (j > 0)) * a.d;
        };
        const auto columns = [&](auto&& f) {  // f(entry, column) of the lane's columns
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const uint32_t c = column.first + (WHOLE ? e : e * kWave);
                if (c < a.d) f(e, c);
            }
        };
        float acc[E] = {};
        walk(a, column, lane < count ? places[own + lane] : 0, 0, count < kShare ? count : kShare, acc, nothing);
        join_waves(lds, wave, lane, acc);
        if (wave == 0) {
            float* const to = slot((start - head) / kRun);
            // past the caches of this die, and there before the count is: a fence would write back all that they hold, the zeros too
            columns([&](int e, uint32_t c) { __hip_atomic_store(to + c, acc[e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); });
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (lane == 0) last_piece = atomicAdd(counters + static_cast<uint64_t>(head / block) * slices + slice, 1u) == pieces - 1;
        }
        __syncthreads();
        if (!uniform(last_piece)) continue;
        const uint32_t share = (pieces + kSumWaves - 1) / kSumWaves;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = 0.0f;
#pragma unroll 1
        for (uint32_t j = wave * share; j < (wave + 1) * share; ++j) {
            if (j >= pieces) break;
            const float* const sums = slot(j);
            columns([&](int e, uint32_t c) { acc[e] += __hip_atomic_load(sums + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); });
        }
        join_waves(lds, wave, lane, acc);
        if (wave == 0) finish<INTO>(a, column, token, acc);
    }
}

// A few positions in one launch, without an order: every block has all of their tokens in LDS. A wave takes one position and one slice; if
// it is its token's first, it adds the rows of that token in their order, and a token of more than 64 positions the whole block, in the
// pieces above: the same bits as from the order. The blocks that fill look their rows up among the tokens. What that saves is the
// launch of the order, behind which fill and sums wait: 512 positions of 1024 float32 into 50304 rows 28.8 us for 34.5 where the caches hold
// the gradient, 39.8 for 42.9 where they do not; added to a gradient 7.6 for 10.5. One token at all positions is a chain of pieces: 27.9 for 33.3 and 10.5 for
// 11.8 (512 of 512 into 50304: 21.9 for 22.1), but 36.8 for 34.7 and 18.2 for 12.6 at 1024 positions, which are therefore ordered.
constexpr uint32_t kFew = 512;
static_assert(kFew <= kSumThreads && kFew / kRun <= kSumWaves && 8 <= kSumWaves, "a thread a position; every piece of a run is a wave's share; a wave for every entry of a lane");
template <typename T, bool WHOLE, bool INTO>
__global__ __launch_bounds__(kSumThreads, INTO ? 4 : 8) void few_kernel(EmbeddingGradient a, uint32_t slices, uint32_t summers) {
    using L = Lane<T, WHOLE>;
    constexpr int E = L::E;
    __shared__ float lds[kSumWaves][E][kWave];
    __shared__ uint32_t tokens[kSumThreads + 1], list[kSumThreads], long_tokens[kSumWaves], counts[kSumWaves];
    const uint32_t key = threadIdx.x < a.n ? token_at(a, threadIdx.x) : ~0u;
    if constexpr (!INTO)
        if (blockIdx.x >= summers) {
            typedef Fill<T> F;
            const F fill(a, blockIdx.x - summers);
            uint32_t* const bits = tokens;  // of the block's rows: whether one has a position
            const uint32_t last_row = fill.row_of(fill.rest - 1);
            for (uint32_t w = threadIdx.x; w <= (last_row - fill.first_row) / 32; w += kSumThreads) bits[w] = 0;
            __syncthreads();
            const bool its = key >= fill.first_row && key <= last_row;
            if (its) atomicOr(bits + (key - fill.first_row) / 32, 1u << (key - fill.first_row) % 32);
            const bool any = __syncthreads_or(its);
            const auto has = [&](uint32_t row) { return (bits[(row - fill.first_row) / 32] >> (row - fill.first_row) % 32 & 1) != 0; };
#pragma unroll
            for (uint32_t u = 0; u < F::U; ++u) {
                if (fill.entry(u) >= fill.rest) break;
                uint32_t row = 0, next = 0;
                if (any) fill.rows(u, row, next);
                const bool none = !any || (next <= row + 1 && !has(row) && !has(next));
                if (none && fill.whole(u)) fill.zero(u);
                else if (!any || !(next == row && has(row))) fill.zero_without(u, has);
            }
            return;
        }
    const uint32_t lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave), mine = blockIdx.x / slices * kSumWaves + wave;
    const L column(blockIdx.x % slices, lane, a.d);
    const auto nothing = [](uint32_t) {};
    const auto before_me = [&](uint64_t mask) { return static_cast<uint32_t>(__popcll(mask & ((1ull << lane) - 1))); };
    tokens[threadIdx.x] = key;
    __syncthreads();
    const uint32_t token = mine < a.n ? uniform(tokens[mine]) : ~0u;
    uint32_t count = 0;  // of its positions, if this is the first
    if (token != ~0u) {
        uint64_t earlier = 0;
        for (uint32_t i = lane; i - lane < mine; i += kWave) earlier |= __ballot(i < mine && tokens[i] == token);
        if (earlier == 0)
            for (uint32_t i = mine / kWave * kWave + lane; i - lane < a.n; i += kWave) {
                const uint64_t its = __ballot(tokens[i] == token);
                const uint32_t to = count + before_me(its);
                if (its >> lane & 1 && to < kRun) list[wave * kRun + to] = i;
                count += static_cast<uint32_t>(__popcll(its));
            }
    }
    if (lane == 0) long_tokens[wave] = count > kRun ? token : ~0u;
    __syncthreads();
    const uint32_t place = list[wave * kRun + lane], long_token = lane < kSumWaves ? long_tokens[lane] : ~0u;
    uint64_t long_waves = __ballot(long_token != ~0u);
    if (count > 0 && count <= kRun) {
        float acc[E] = {};
        walk(a, column, place, 0, count, acc, nothing);
        finish<INTO>(a, column, token, acc);
    }
    for (; long_waves != 0; long_waves &= long_waves - 1) {
        const uint32_t of = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(long_token), __ffsll(static_cast<long long>(long_waves)) - 1));
        const uint64_t its = __ballot(key == of);
        if (lane == 0) counts[wave] = static_cast<uint32_t>(__popcll(its));
        __syncthreads();  // the list was read
        uint32_t first = 0, all = 0;
#pragma unroll
        for (uint32_t w = 0; w < kSumWaves; ++w) {
            if (w < wave) first += counts[w];
            all += counts[w];
        }
        if (key == of) list[first + before_me(its)] = threadIdx.x;
        __syncthreads();
        // Every wave's rows of a piece are requested before the last piece is joined, of which a wave takes one entry of each lane.
        typename L::Share share[kShare];
        const auto request = [&](uint32_t piece) {
            const uint32_t own = piece + wave * kShare;
#pragma unroll
            for (uint32_t r = 0; r < kShare; ++r)
                if (own + r < all) column.load(static_cast<const T*>(a.g) + uniform(list[own + r]) * a.g_stride, share[r]);
        };
        request(0);
        float sum = 0.0f;
        for (uint32_t piece = 0; piece < all; piece += kRun) {
            float acc[E] = {};
#pragma unroll
            for (uint32_t r = 0; r < kShare; ++r) {
                if (piece + wave * kShare + r >= all) break;
                float v[E];
                L::widened(share[r], v);
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] += v[e];
            }
            request(piece + kRun);
            lds_barrier();
#pragma unroll
            for (int e = 0; e < E; ++e) lds[wave][e][lane] = acc[e];
            lds_barrier();
            if (wave < E) {
                float joined = 0.0f;
#pragma unroll
                for (uint32_t v = 0; v < kSumWaves; ++v) joined += lds[v][wave][lane];
                sum += joined;
            }
        }
        lds_barrier();
        if (wave < E) lds[0][wave][lane] = sum;
        lds_barrier();
        if (wave == 0) {
            float acc[E];
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = lds[0][e][lane];
            finish<INTO>(a, column, of, acc);
        }
    }
}

// Positions of a wave: fewer where that leaves CUs without a block.
uint32_t sum_window(int vt, uint32_t n, uint32_t d) {
    const uint32_t slice = kWave * (vt == kBF16 ? 8 : 4), slices = (d + slice - 1) / slice;
    uint32_t window = kWindow;
    while (window > 1 && static_cast<uint64_t>(n) * slices < 512 * window * kSumWaves) window /= 2;
    return window;
}

bool whole_rows(int vt, uint32_t d, std::initializer_list<const void*> rows, uint64_t stride) {
    const uint32_t per = vt == kBF16 ? 8 : 4;
    if (d % per != 0 || stride % per != 0) return false;
    for (const void* p : rows)
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
    return true;
}

template <typename T, bool WHOLE>
hipError_t lookup(const EmbeddingForward& a, hipStream_t stream) {
    constexpr uint32_t slice = Lane<T, WHOLE>::SLICE, waves = kLookupThreads / kWave;
    const uint32_t slices = (a.d + slice - 1) / slice;
    // four rows a wave once that leaves every CU its waves
    if (static_cast<uint64_t>(a.n) * slices >= 16384)
        hipLaunchKernelGGL((lookup_kernel<T, WHOLE, 4>), dim3(((a.n + 3) / 4 * slices + waves - 1) / waves), dim3(kLookupThreads), 0, stream, a, slices);
    else
        hipLaunchKernelGGL((lookup_kernel<T, WHOLE, 1>), dim3((a.n * slices + waves - 1) / waves), dim3(kLookupThreads), 0, stream, a, slices);
    return hipGetLastError();
}

// The workspace's parts: sorted keys and positions by place (twice with more than one chunk), a place of every token, the blocks'
// counters, the pieces' sums.
struct Parts {
    uint64_t one, where, counters, partials, bytes;  // bytes of an array; where the others begin; all
    uint32_t window, blocks, slices;
    Parts(int vt, uint32_t n, uint32_t d, uint32_t vocab) {
        const auto whole = [](uint64_t v) { return (v + 255) / 256 * 256; };
        const uint32_t slice = kWave * (vt == kBF16 ? 8 : 4);
        slices = (d + slice - 1) / slice;
        window = sum_window(vt, n, d);
        blocks = (n + window * kSumWaves - 1) / (window * kSumWaves);
        one = whole(4ull * n);
        where = (n > kChunk ? 4 : 2) * one;
        counters = where + whole(4ull * vocab);
        partials = counters + whole(4ull * blocks * slices);
        bytes = partials + (n > kRun ? 8ull * blocks * d : 0);
    }
};

template <typename T>
uint64_t fill_blocks(const EmbeddingGradient& a) { return a.into ? 0 : (static_cast<uint64_t>(a.vocab) * a.d + Fill<T>::kEntries - 1) / Fill<T>::kEntries; }

template <typename T, bool WHOLE>
hipError_t few(const EmbeddingGradient& a, hipStream_t stream) {
    constexpr uint32_t slice = Lane<T, WHOLE>::SLICE;
    const uint32_t slices = (a.d + slice - 1) / slice, summers = (a.n + kSumWaves - 1) / kSumWaves * slices;
    const dim3 grid(static_cast<uint32_t>(summers + fill_blocks<T>(a)));
    if (a.into) hipLaunchKernelGGL((few_kernel<T, WHOLE, true>), grid, dim3(kSumThreads), 0, stream, a, slices, summers);
    else hipLaunchKernelGGL((few_kernel<T, WHOLE, false>), grid, dim3(kSumThreads), 0, stream, a, slices, summers);
    return hipGetLastError();
}

template <typename T, bool WHOLE>
hipError_t sums(const EmbeddingGradient& a, const Parts& parts, char* workspace, const uint32_t* sorted, const uint32_t* places, hipStream_t stream) {
    uint32_t* const counters = reinterpret_cast<uint32_t*>(workspace + parts.counters);
    float* const partials = reinterpret_cast<float*>(workspace + parts.partials);
    const uint32_t* const where = reinterpret_cast<const uint32_t*>(workspace + parts.where);
    const uint32_t summers = parts.blocks * parts.slices;
    const dim3 grid(static_cast<uint32_t>(summers + fill_blocks<T>(a)));
    if (a.into) hipLaunchKernelGGL((sums_kernel<T, WHOLE, true>), grid, dim3(kSumThreads), 0, stream, a, sorted, places, parts.window, counters, partials, where, parts.slices, summers);
    else hipLaunchKernelGGL((sums_kernel<T, WHOLE, false>), grid, dim3(kSumThreads), 0, stream, a, sorted, places, parts.window, counters, partials, where, parts.slices, summers);
    return hipGetLastError();
}

}  // namespace

uint64_t embedding_workspace_bytes(int vt, uint32_t n, uint32_t d, uint32_t vocab) { return Parts(vt, n, d, vocab).bytes; }

hipError_t launch_embedding(int vt, const EmbeddingForward& a, hipStream_t stream) {
    const bool whole = whole_rows(vt, a.d, {a.weight, a.out}, a.d);
    if (vt == kBF16) return whole ? lookup<uint16_t, true>(a, stream) : lookup<uint16_t, false>(a, stream);
    return whole ? lookup<float, true>(a, stream) : lookup<float, false>(a, stream);
}

hipError_t launch_embedding_gradient(int vt, const EmbeddingGradient& a, void* workspace, hipStream_t stream) {
    const bool whole = whole_rows(vt, a.d, {a.g, a.gw}, a.g_stride);
    if (a.n <= kFew) {
        if (vt == kBF16) return whole ? few<uint16_t, true>(a, stream) : few<uint16_t, false>(a, stream);
        return whole ? few<float, true>(a, stream) : few<float, false>(a, stream);
    }
    const Parts parts(vt, a.n, a.d, a.vocab);
    char* const base = static_cast<char*>(workspace);
    const auto array = [&](int k) { return reinterpret_cast<uint32_t*>(base + k * parts.one); };
    uint32_t *sorted = array(0), *places = array(1), *const where = a.into ? nullptr : reinterpret_cast<uint32_t*>(base + parts.where);
    const bool chunks = a.n > kChunk;
    const uint32_t held = std::min((a.n + kWave - 1) / kWave * kWave, kChunk) * 4;
    if (held > 32768)
        if (const hipError_t status = hipFuncSetAttribute(reinterpret_cast<const void*>(rank_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kChunk * 4); status != hipSuccess)
            return status;
    hipLaunchKernelGGL(rank_kernel, dim3((a.n + kOwn - 1) / kOwn), dim3(kRankThreads), held, stream, a.ids, a.n, a.vocab, a.padding, sorted, places,
                       chunks ? nullptr : where, reinterpret_cast<uint32_t*>(base + parts.counters), parts.blocks * parts.slices);
    if (const hipError_t status = hipGetLastError(); status != hipSuccess) return status;
    if (chunks) {
        uint32_t *const all = array(2), *const order = array(3);
        hipLaunchKernelGGL(merge_kernel, dim3((a.n + kMergeThreads - 1) / kMergeThreads), dim3(kMergeThreads), 0, stream, sorted, places, a.n, kChunk, all, order, where, a.vocab);
        if (const hipError_t status = hipGetLastError(); status != hipSuccess) return status;
        sorted = all;
        places = order;
    }
    if (vt == kBF16) return whole ? sums<uint16_t, true>(a, parts, base, sorted, places, stream) : sums<uint16_t, false>(a, parts, base, sorted, places, stream);
    return whole ? sums<float, true>(a, parts, base, sorted, places, stream) : sums<float, false>(a, parts, base, sorted, places, stream);
}

}  // namespace hffn
