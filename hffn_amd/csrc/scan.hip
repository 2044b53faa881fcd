// The gated linear recurrence over sequences laid end to end, forward, backward and one token at a time. Per channel, with
// z = sigmoid(gate + bias):
//   h_t = (1 - z_t) h_t-1 + v_t,   v = z x (tied), sqrt(1 - (1 - z)^2) x (normed) or x (free)
//   G_t = gh_t + (1 - z_t+1) G_t+1;   gx = G dv/dx,   ggate = G (dv/dz - h_t-1) z (1 - z)
// Time is cut into tiles of rows, one block each, which stay in its registers. What a tile does to the value that enters it is
// h -> p h + b with p the product of its factors 1 - z: each block publishes its (p, b), folds those before it to what enters
// its own, and walks its rows again from there. Rows are read once and written once, by one launch.
//
// Forward 3 N d entries moved, backward 6 N d (a large copy: 5.2 TB/s). Measured, us a call of the kernels' own time: forward 8 x 2048
// tokens of 1024 channels, tied bfloat16, 36 (101 MB: 2.8 TB/s), 32768 tokens of 512 channels, normed float32, 54 (201 MB: 3.7); backward of
// the former 53 (201 MB: 3.8). What bounds it is neither the memory nor the instructions alone: of the 36 us the bytes are 19.5 and the vector
// instructions, 43 an entry, 18 on every SIMD (float32 56, 24 of the 54; backward 58, 25 of the 53). 1024 blocks are two rounds of the 512 that
// the card holds; a CU has 29 of its 32 waves while it has any block, 30 of the 36 us, and a wave waits 64 % of its cycles (58 and 57): a
// block's chain (a tile's stamps, bfloat16 forward: ticket 2 us, requests and bounds 4.5, gates and the first walk 4, the fold of the
// waves 1.3, the tiles before 2, the groups 1, the last walk 1.4) passes beside that of one other block.
// Blocks that stay, with waves of their own for the folds and the next tile's rows requested ahead, took 62 us where this takes 40:
// the folds are the longest chain, and had fewer waves to hide in.
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "launch.hpp"

namespace hffn {
namespace {

// A factor p = 1 - q of a value that is carried on, as one float that keeps both ends: q itself where that is at most a half,
// -p else, and kCut where a sequence begins and nothing passes, whatever came before it (an infinity or a NaN too). A slow
// channel's p = 1 - 2^-20 as a float alone would be off by 2^-5 of its q, at every token the same way.
constexpr float kCut = -2.0f;
__device__ __forceinline__ bool is_rest(float f) { return __float_as_int(f) < 0; }  // -p (or the cut)
__device__ __forceinline__ float passed(float f, float h) { return fmaf(-f, h, is_rest(f) ? 0.0f : h); }
__device__ __forceinline__ float passed_and(float f, float h, float v) { return fmaf(-f, h, is_rest(f) ? v : h + v); }  // p h + v
__device__ __forceinline__ float factor_rest(float f) { return is_rest(f) ? -f : 1.0f - f; }

// An infinity stays one until its sequence ends or meets a NaN or its opposite, however small the p; the forms above make a NaN of it
// (inf - z inf, 0 inf). Whatever comes out not finite is looked at again: what follows an infinite h is h + v.
__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.402823466e38f; }
__device__ __forceinline__ bool infinite(float v) { return fabsf(v) == INFINITY; }
__device__ __forceinline__ float defined(float f, float h, float v) { return infinite(h) ? h + v : passed_and(f, h, v); }
template <int V>
__device__ __forceinline__ bool all_finite(const float (&h)[V]) {
    bool good = true;
#pragma unroll
    for (int v = 0; v < V; ++v) good &= finite(h[v]);
    return good;
}

// (f, b): h -> p h + b.
struct Step {
    float f, b;
};
template <bool CAREFUL = false>
__device__ __forceinline__ float apply(const Step& s, float h) {
    return s.f == kCut ? s.b : CAREFUL && infinite(h) ? h + s.b : passed(s.f, h) + s.b;
}
template <bool CAREFUL = false>
__device__ __forceinline__ Step then(const Step& first, const Step& second) {
    const float q = fmaf(-first.f, second.f, first.f) + second.f;
    const bool whole = !is_rest(first.f) && !is_rest(second.f) && q <= 0.5f;
    const float p = factor_rest(first.f) * factor_rest(second.f);
    Step s;
    s.f = first.f == kCut || second.f == kCut ? kCut : whole ? q : -p;
    s.b = apply<CAREFUL>(second, first.b);
    return s;
}

// z = sigmoid(a) as a factor: f = z where that is at most a half, else -(1 - z), the smaller of the two in either case and taken from
// the exponential itself. root = sqrt(1 - (1 - z)^2) = sqrt(z (2 - z)), still a float where z is
// none any more (a below -87). Beyond 256 all are at their ends; a NaN stays one. bfloat16 gates are off by 2^-9 by themselves: their
// exponential is the hardware's of a rounded product (off by 2^-24 |a|), float32 gates' loses nothing to that rounding.
template <bool FINE>
struct Gate {
    float f, z, root;
    __device__ __forceinline__ explicit Gate(float minus_a) {
        const float m = __builtin_elementwise_minimum(fabsf(minus_a), 256.0f);
        const float t = FINE ? exp_split(-m) : __builtin_amdgcn_exp2f(m * -1.44269504f), r = __builtin_amdgcn_rcpf(1.0f + t), small = t * r;
        f = copysignf(small, minus_a);
        z = is_rest(f) ? r : small;
        root = __builtin_amdgcn_sqrtf(r + r * (is_rest(f) ? small : r)) * (is_rest(f) ? 1.0f : exp_split(-0.5f * m));
    }
};

// A product that is rounded by itself, so that a row's bits do not depend on what its variant fuses.
__device__ __forceinline__ float product(float a, float b) {
#pragma clang fp contract(off)
    return a * b;
}

// v = input x
template <int KIND, bool FINE>
__device__ __forceinline__ float input(const Gate<FINE>& g) {
    return KIND == kTied ? g.z : KIND == kNormed ? g.root : 1.0f;
}

// Where the sequences begin, and the end of the last, all held to [0, n]; without a table one sequence of all rows.
__device__ __forceinline__ uint32_t bound_at(const ScanBounds& b, uint32_t n, uint32_t s) {
    if (b.p == nullptr) return s == 0 ? 0 : n;
    const int64_t at = b.wide ? static_cast<const int64_t*>(b.p)[s] : static_cast<const int32_t*>(b.p)[s];
    return at < 0 ? 0 : at > n ? n : static_cast<uint32_t>(at);
}

// The first entry in [low, high) above t (high: none); 64 probes at a time, by the whole wave.
__device__ __forceinline__ uint32_t first_above(const ScanBounds& b, uint32_t n, uint32_t low, uint32_t high, uint32_t t, uint32_t lane) {
    while (low < high) {
        const uint32_t stride = (high - low + kWave - 1) / kWave, at = low + lane * stride + stride - 1;
        const uint32_t less = static_cast<uint32_t>(__popcll(__ballot(at < high && bound_at(b, n, at) <= t)));
        low += less * stride;
        high = low + stride - 1 < high ? low + stride - 1 : high;
    }
    return low;
}

// Rows of a wave's share of a tile: what its registers hold beside a second block of 16 waves on the CU. float32 forward: 16 rows 60 us,
// 8 rows, whose waves searched the bounds twice as often, 73 (32768 x 512). bfloat16 rows of two columns a lane could be kept as they came in and their gates computed twice: 16 of
// them spill, 96 us where 8 take 46.
constexpr int forward_rows(bool single) { return single ? 16 : 8; }
constexpr int kBackRows = 8;
constexpr uint32_t kWaves = 16;
constexpr uint32_t kGroup = 16;  // tiles whose steps are folded into one

// The rows [t0, t0 + R) of a wave, as bits: which of them belong to a sequence, begin one, end one. The table is searched 64
// entries at a time: one load for up to 63 sequences.
template <int R>
struct Rows {
    static constexpr uint32_t kAllRows = (1u << R) - 1;
    uint32_t live, begins = 0, ends = 0;
    uint32_t next;    // the first sequence that begins at t0 or later (the count: none does)
    uint32_t behind;  // the first bound behind the last row
    uint32_t before;  // where the sequence before `next` begins (t0: there is none, or one begins at t0)
    uint32_t after;   // the bound `behind`: where the last row's sequence ends (0: there is none)
    // `cached`: of a table of at most 64 entries, entry `lane` (the last beyond the end).
    __device__ __forceinline__ static uint32_t cache(const ScanBounds& b, uint32_t n, uint32_t lane) { return bound_at(b, n, lane < b.count ? lane : b.count); }
    __device__ __forceinline__ Rows(const ScanBounds& b, uint32_t n, uint32_t t0, uint32_t lane, uint32_t cached) {
        const uint32_t stop = t0 + R;
        uint32_t low = 0, high = b.count;  // next is in [low, high]
        while (high - low >= kWave) {
            const uint32_t stride = (high - low + kWave - 1) / kWave, at = low + lane * stride + stride - 1;
            const uint32_t less = static_cast<uint32_t>(__popcll(__ballot(at < high && bound_at(b, n, at) < t0)));
            low += less * stride;
            high = low + stride - 1 < high ? low + stride - 1 : high;
        }
        const bool whole = b.count < kWave;
        uint32_t own = whole ? cached : bound_at(b, n, low + lane < b.count ? low + lane : b.count);
        const uint32_t less = static_cast<uint32_t>(__popcll(__ballot(low + lane < high && own < t0)));
        next = low + less;
        before = less > 0 ? static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(own), less - 1)) : next > 0 ? bound_at(b, n, next - 1) : t0;
        const uint32_t first = whole ? static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(cached), 0)) : bound_at(b, n, 0),
                       last = whole ? static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(cached), kWave - 1)) : bound_at(b, n, b.count);
        live = kAllRows;
        if (first > t0) live = first < stop ? live & kAllRows << (first - t0) : 0;
        if (last < stop) live = last > t0 ? live & kAllRows >> (stop - last) : 0;
        behind = b.count;
        after = 0;
        for (uint32_t base = low; base <= b.count;) {
            const uint32_t s = base + lane;
            if (base != low) own = bound_at(b, n, s < b.count ? s : b.count);
            const uint64_t begin = __ballot(s < b.count && own >= t0 && own < stop), end = __ballot(s > 0 && s <= b.count && own > t0 && own <= stop),
                           later = __ballot(s <= b.count && s >= next && own >= stop);
            for (uint64_t rest = begin; rest != 0;) {
                const uint32_t t = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(own), __ffsll(static_cast<long long>(rest)) - 1));
                begins |= 1u << (t - t0);
                rest &= ~__ballot(own == t);
            }
            for (uint64_t rest = end; rest != 0;) {
                const uint32_t t = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(own), __ffsll(static_cast<long long>(rest)) - 1));
                ends |= 1u << (t - 1 - t0);
                rest &= ~__ballot(own == t);
            }
            if (later == 0) {  // on behind the last one's equals
                base += kWave;
                if (base <= b.count) base = first_above(b, n, base, b.count + 1, static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(own), kWave - 1)), lane);
                continue;
            }
            const uint32_t k = __ffsll(static_cast<long long>(later)) - 1;
            behind = base + k;
            after = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(own), k));
            break;
        }
        begins = uniform(begins & live);
        ends = uniform(ends & live);
        live = uniform(live);
        next = uniform(next);
        behind = uniform(behind);
        before = begins & 1 ? t0 : uniform(before);
        after = uniform(after);
    }
    __device__ __forceinline__ bool plain() const { return live == kAllRows && (begins | ends) == 0; }
};

// Rows of T, V adjacent columns a lane (one load).
template <typename T, int V>
struct Cell {
    typedef typename std::conditional<V == 1, T, typename std::conditional<V * sizeof(T) == 4, uint32_t, float2>::type>::type Raw;
    __device__ __forceinline__ static Raw load(const void* rows, uint64_t stride, uint32_t t, uint32_t column) {
        return *reinterpret_cast<const Raw*>(static_cast<const T*>(rows) + t * stride + column);
    }
    __device__ __forceinline__ static float get(const Raw& raw, int v) {
        if constexpr (V == 1) return widen(raw);
        else if constexpr (sizeof(T) == 4) return v == 0 ? raw.x : raw.y;
        else return __uint_as_float(v == 0 ? raw << 16 : raw & 0xffff0000u);
    }
    __device__ __forceinline__ static void store(void* rows, uint32_t t, uint32_t d, uint32_t column, const float (&in)[V]) {
        T* const p = static_cast<T*>(rows) + static_cast<uint64_t>(t) * d + column;
        if constexpr (V == 1) {
            if constexpr (sizeof(T) == 4) *p = in[0];
            else *p = bf16_bits(in[0]);
        } else if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float2*>(p) = make_float2(in[0], in[1]);
        } else {
            *reinterpret_cast<uint32_t*>(p) = bf16_pair(in[0], in[1]);
        }
    }
};

template <int V>
__device__ __forceinline__ void load_floats(const float* p, float otherwise, float (&to)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) to[v] = p == nullptr ? otherwise : p[v];
}

// What the rows of a wave do to what enters them, summed up row by row (forward: ascending, backward: descending). The product of the
// factors is held as it is and as its complement, of which the step takes the one that is whole.
template <int V>
struct Summary {
    float b[V], p[V], q[V];
    int rest[V];  // its sign: whether a factor was -p
    __device__ __forceinline__ Summary() {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            b[v] = q[v] = 0.0f;
            p[v] = 1.0f;
            rest[v] = 0;
        }
    }
    __device__ __forceinline__ void row(int v, float f) {  // the factors; b is the caller's
        p[v] = passed(f, p[v]);
        q[v] = fmaf(-f, q[v], q[v] + f);
        rest[v] |= __float_as_int(f);
    }
    __device__ __forceinline__ Step step(int v, bool cut) const { return {cut ? kCut : rest[v] >= 0 && q[v] <= 0.5f ? q[v] : -p[v], b[v]}; }
};

// A step as one 64-bit word, which a reader has whole or not at all; all ones while it is not there (no step has that f).
typedef unsigned long long Word;
constexpr Word kNothing = ~0ull;
__device__ __forceinline__ void publish(Word* to, const Step& s) {
    const uint32_t f = s.f != s.f ? 0x7fc00000u : __float_as_uint(s.f);
    __hip_atomic_store(to, static_cast<Word>(f) << 32 | __float_as_uint(s.b), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ Step await(Word* from) {
    Word word = __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    while (word == kNothing) {
        __builtin_amdgcn_s_sleep(1);
        word = __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    return {__uint_as_float(static_cast<uint32_t>(word >> 32)), __uint_as_float(static_cast<uint32_t>(word))};
}

// The workspace: the blocks' ticket, the tiles' and the groups' steps by tile (group) and column, all ones before the launch.
struct Chain {
    uint32_t* ticket;
    Word *tiles, *groups;
    uint32_t count;  // tiles
    __host__ __device__ static uint64_t words(uint32_t tiles, uint32_t d) { return 1 + static_cast<uint64_t>(tiles + (tiles + kGroup - 1) / kGroup) * d; }
    __device__ __forceinline__ Chain(void* workspace, uint32_t tiles, uint32_t d)
        : ticket(static_cast<uint32_t*>(workspace)), tiles(static_cast<Word*>(workspace) + 1), groups(this->tiles + static_cast<uint64_t>(tiles) * d), count(tiles) {}
};

// A block's tile (in the order of the walk) and slice of the columns. With more than one tile blocks take them in the order in which
// they start, so that every tile another one waits for is held by a block that runs and waits for none behind it.
struct Place {
    uint32_t tile, slice;
    __device__ __forceinline__ Place(const Chain& chain, uint32_t slices, uint32_t* lds) {
        uint32_t at = blockIdx.x;
        if (chain.count > 1) {
            if (threadIdx.x == 0) *lds = atomicAdd(chain.ticket, 1u) + 1;  // from all ones
            __syncthreads();
            at = uniform(*lds);
        }
        tile = at / slices;
        slice = at % slices;
    }
};

// From every wave's step to what enters its rows. The first V waves hold a column a lane: they fold the waves' steps and publish the
// tile's; every wave then waits for one tile before this in its group of kGroup, the V waves fold these, the last tile of a group
// publishes the group's, every wave waits for one group before this one (kWaves at a time), and the V waves carry what comes
// of it over the tile's waves. Folds run from the nearest step to the farthest, so that results do not depend on who came
// first, and no farther than `reach`, the tile where the sequence begins that this one's first row belongs to.
// `order(w)`: the w-th wave in the order of the walk.
template <int V>
struct Carry {
    Step steps[kWaves][V][kWave];
    union {
        Step before[kWaves][V][kWave];
        float enters[kWaves][V][kWave];
    };
    uint32_t ticket, reach;
};
template <int V, typename ORDER>
__device__ __forceinline__ void carry(Carry<V>& lds, const Chain& chain, uint32_t tile, uint32_t d, uint32_t column, bool here, uint32_t lane, uint32_t wave,
                                      ORDER order) {
    const bool folds = wave < V;
    const uint32_t mine = column + wave;  // of a folding wave's lane
    lds_barrier();
    Step acc = {0.0f, 0.0f};
    if (chain.count > 1) {
        Step own = acc;
        if (folds) {
            own = lds.steps[order(0)][wave][lane];
#pragma unroll
            for (uint32_t w = 1; w < kWaves; ++w) own = then(own, lds.steps[order(w)][wave][lane]);
            if (!finite(own.b)) {
                own = lds.steps[order(0)][wave][lane];
#pragma unroll 1
                for (uint32_t w = 1; w < kWaves; ++w) own = then<true>(own, lds.steps[order(w)][wave][lane]);
            }
            if (here) publish(chain.tiles + static_cast<uint64_t>(tile) * d + mine, own);
        }
        const uint32_t reach = uniform(lds.reach < tile ? lds.reach : tile), group = tile / kGroup, in_group = tile % kGroup;
        const uint32_t tiles = in_group < tile - reach ? in_group : tile - reach, groups = reach < group * kGroup ? group - reach / kGroup : 0;
        if (wave < tiles && here)
#pragma unroll
            for (int v = 0; v < V; ++v) lds.before[wave][v][lane] = await(chain.tiles + static_cast<uint64_t>(tile - 1 - wave) * d + column + v);
        lds_barrier();
        const auto fold = [&](uint32_t count) {  // of `before` to acc
            const Step behind = acc;
            for (uint32_t k = 0; k < count; ++k) acc = then(lds.before[k][wave][lane], acc);
            if (finite(acc.b)) return;
            acc = behind;
#pragma unroll 1
            for (uint32_t k = 0; k < count; ++k) acc = then<true>(lds.before[k][wave][lane], acc);
        };
        if (folds) {
            fold(tiles);
            if (in_group == kGroup - 1 && here) publish(chain.groups + static_cast<uint64_t>(group) * d + mine, then<true>(acc, own));
        }
        for (uint32_t back = 0; back < groups; back += kWaves) {
            lds_barrier();
            if (wave < groups - back && here)
#pragma unroll
                for (int v = 0; v < V; ++v) lds.before[wave][v][lane] = await(chain.groups + static_cast<uint64_t>(group - 1 - back - wave) * d + column + v);
            lds_barrier();
            if (folds) fold(groups - back < kWaves ? groups - back : kWaves);
        }
        if (V > 1) lds_barrier();  // the other folding waves' steps were read
    }
    if (folds) {
        float h = acc.b;
        bool good = true;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) {
            lds.enters[order(w)][wave][lane] = h;
            good &= finite(h);
            h = apply(lds.steps[order(w)][wave][lane], h);
        }
        if (!good) {
            h = acc.b;
#pragma unroll 1
            for (uint32_t w = 0; w < kWaves; ++w) {
                lds.enters[order(w)][wave][lane] = h;
                h = apply<true>(lds.steps[order(w)][wave][lane], h);
            }
        }
    }
    lds_barrier();
}

// f(true_type) or f(false_type): whether all of a wave's rows lie inside one sequence; that walk has no branches.
template <int R, typename F>
__device__ __forceinline__ auto by_rows(const Rows<R>& rows, F&& f) {
    return rows.plain() ? f(std::true_type()) : f(std::false_type());
}

// The state of the sequence that begins at row t; `s`: the first that begins there or later, moved behind it.
template <int V>
__device__ __forceinline__ void begin_at(const ScanForward& a, uint32_t t, uint32_t& s, uint32_t lane, uint32_t from, float (&h)[V]) {
    if (s + 1 < a.bounds.count && bound_at(a.bounds, a.n, s + 1) <= t) s = first_above(a.bounds, a.n, s + 1, a.bounds.count, t, lane) - 1;
    if (s >= a.bounds.count) s = a.bounds.count - 1;
    load_floats<V>(a.state == nullptr ? nullptr : a.state + static_cast<uint64_t>(s) * a.d + from, 0.0f, h);
    ++s;
}

// The rows of a wave again, from memory, where values are not finite; `fast` repeats what was stored. A function of its own, called by nearly nobody:
// inside the kernels its registers would be theirs (bfloat16 backward 59 -> 80 us, by 11 registers in scratch memory).
template <typename T, int V, int KIND>
__device__ __attribute__((noinline)) void again(const void* arguments, uint32_t t0, uint32_t column, const float* enters) {
    using C = Cell<T, V>;
    constexpr int R = forward_rows(sizeof(T) == 4);
    const ScanForward a = *static_cast<const ScanForward*>(arguments);
    const uint32_t lane = __lane_id(), from = column < a.d ? column : 0;
    t0 = uniform(t0);
    const Rows<R> rows(a.bounds, a.n, t0, lane, Rows<R>::cache(a.bounds, a.n, lane));
    float bias[V], fast[V], h[V];
    load_floats<V>(a.bias == nullptr ? nullptr : a.bias + from, 0.0f, bias);
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = fast[v] = enters[v * kWave + lane];
    uint32_t s = rows.next;
#pragma unroll 1
    for (uint32_t r = 0; r < R; ++r) {
        const uint32_t t = t0 + r;
        if (!(rows.live >> r & 1)) continue;
        if (rows.begins >> r & 1) {
            begin_at<V>(a, t, s, lane, from, h);
#pragma unroll
            for (int v = 0; v < V; ++v) fast[v] = h[v];
        }
        const typename C::Raw gate_t = C::load(a.gate, a.gate_stride, t, from), x_t = C::load(a.x, a.x_stride, t, from);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const Gate<sizeof(T) == 4> g(-C::get(gate_t, v) - bias[v]);
            const float in_t = product(input<KIND>(g), C::get(x_t, v));
            fast[v] = passed_and(g.f, fast[v], in_t);
            h[v] = finite(fast[v]) ? fast[v] : defined(g.f, h[v], in_t);
        }
        if (column >= a.d || all_finite<V>(fast)) continue;
        C::store(a.h, t, a.d, column, h);
        if (!(rows.ends >> r & 1)) continue;
        const uint64_t at = static_cast<uint64_t>(s > 0 ? s - 1 : 0) * a.d + column;
#pragma unroll
        for (int v = 0; v < V; ++v) a.last[at + v] = h[v];
    }
}

template <typename T, int V, int KIND>
__global__ __launch_bounds__(kWaves* kWave, 8) void scan_kernel(ScanForward a, uint32_t slices, uint32_t tiles) {
    using C = Cell<T, V>;
    constexpr bool FINE = sizeof(T) == 4;
    constexpr int R = forward_rows(sizeof(T) == 4);
    constexpr uint32_t kTileRows = kWaves * R;
    __shared__ Carry<V> lds;
    const Chain chain(a.steps, tiles, a.d);
    const uint32_t cached = Rows<R>::cache(a.bounds, a.n, threadIdx.x % kWave);
    const Place place(chain, slices, &lds.ticket);
    const uint32_t lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave), column = (place.slice * kWave + lane) * V;
    const uint32_t t0 = place.tile * kTileRows + wave * R;
    const bool here = column < a.d;
    typename C::Raw x[R], gate[R];
    const uint32_t from = here ? column : 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint32_t t = t0 + r < a.n ? t0 + r : a.n - 1;
        gate[r] = C::load(a.gate, a.gate_stride, t, from);
    }
    float bias[V];
    load_floats<V>(a.bias == nullptr ? nullptr : a.bias + from, 0.0f, bias);
#pragma unroll
    for (int r = 0; r < R; ++r) x[r] = C::load(a.x, a.x_stride, t0 + r < a.n ? t0 + r : a.n - 1, from);
    const Rows<R> rows(a.bounds, a.n, t0, lane, cached);
    if (threadIdx.x == 0) lds.reach = rows.before / kTileRows;
    float f[R][V], in[R][V];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const Gate<FINE> g(-C::get(gate[r], v) - bias[v]);
            f[r][v] = g.f;
            in[r][v] = product(input<KIND>(g), C::get(x[r], v));
        }
    const auto begin = [&](uint32_t t, uint32_t& s, float (&h)[V]) { begin_at<V>(a, t, s, lane, from, h); };
    bool good = by_rows(rows, [&](auto plain) {
        Summary<V> sum;
        uint32_t s = rows.next;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if constexpr (!plain) {
                if (!(rows.live >> r & 1)) continue;
                if (rows.begins >> r & 1) begin(t0 + r, s, sum.b);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) {
                sum.b[v] = passed_and(f[r][v], sum.b[v], in[r][v]);
                sum.row(v, f[r][v]);
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) lds.steps[wave][v][lane] = sum.step(v, rows.begins != 0);
        return all_finite<V>(sum.b);
    });
    if (__builtin_expect(__ballot(!good) != 0, 0)) {  // b is what entered last that is not finite, by its sum
        const int last = 31 - __clz(static_cast<int>(rows.begins));  // the last row where a sequence begins
        float sum[V] = {};
        uint32_t s = rows.next;
        if (last >= 0) begin(t0 + last, s, sum);
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (r >= last && rows.live >> r & 1)
#pragma unroll
                for (int v = 0; v < V; ++v) sum[v] += in[r][v];
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (!finite(sum[v]) && !finite(lds.steps[wave][v][lane].b)) lds.steps[wave][v][lane].b = sum[v];
    }
    carry<V>(lds, chain, place.tile, a.d, column, here, lane, wave, [](uint32_t w) { return w; });
    float h[V];
    good = true;
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = lds.enters[wave][v][lane];
    by_rows(rows, [&](auto plain) {
        uint32_t s = rows.next;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint32_t t = t0 + r;
            if constexpr (!plain) {
                if (t >= a.n) break;
                if (!(rows.live >> r & 1)) {
                    const float none[V] = {};
                    if (here) C::store(a.h, t, a.d, column, none);
                    continue;
                }
                if (rows.begins >> r & 1) {
                    good &= all_finite<V>(h);
                    begin(t, s, h);
                }
            }
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = passed_and(f[r][v], h[v], in[r][v]);
            if (here) C::store(a.h, t, a.d, column, h);
            if constexpr (!plain) {
                if (!(rows.ends >> r & 1) || !here) continue;
                const uint64_t at = static_cast<uint64_t>(s > 0 ? s - 1 : 0) * a.d + column;
#pragma unroll
                for (int v = 0; v < V; ++v) a.last[at + v] = h[v];
            }
        }
    });
    good &= all_finite<V>(h);
    if (__builtin_expect(__ballot(!good) != 0, 0)) again<T, V, KIND>((const void*)__builtin_amdgcn_kernarg_segment_ptr(), t0, column, &lds.enters[wave][0][0]);
}

// Before a scan: the workspace's words to all ones, and what leaves sequences without rows is what entered (zero where nothing was
// given; to null: not wanted). Blocks below `fillers` fill, the others take a sequence each.
constexpr uint32_t kPrepareThreads = 256;
__global__ __launch_bounds__(kPrepareThreads) void prepare_kernel(Word* words, uint64_t count, uint32_t fillers, ScanBounds bounds, uint32_t n, const float* from,
                                                                  float* to, uint32_t d) {
    if (blockIdx.x < fillers) {
        for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * kPrepareThreads + threadIdx.x; i < count; i += static_cast<uint64_t>(fillers) * kPrepareThreads)
            words[i] = kNothing;
        return;
    }
    const uint32_t s = blockIdx.x - fillers;
    if (bound_at(bounds, n, s) < bound_at(bounds, n, s + 1)) return;
    for (uint32_t c = threadIdx.x; c < d; c += kPrepareThreads)
        to[static_cast<uint64_t>(s) * d + c] = from == nullptr ? 0.0f : from[static_cast<uint64_t>(s) * d + c];
}

// The sequence of row t, `s` being at or behind it.
__device__ __forceinline__ uint32_t sequence_of(const ScanBounds& bounds, uint32_t n, uint32_t t, uint32_t& s, uint32_t lane) {
    if (s >= bounds.count) s = bounds.count - 1;
    if (s > 0 && bound_at(bounds, n, s) > t) --s;
    if (s > 0 && bound_at(bounds, n, s) > t) {
        s = first_above(bounds, n, 0, s, t, lane);
        if (s > 0) --s;
    }
    return s;
}
template <int V>
__device__ __forceinline__ void end_at(const ScanBackward& a, uint32_t t, uint32_t& s, uint32_t lane, uint32_t from, float (&g)[V]) {
    const uint64_t at = static_cast<uint64_t>(sequence_of(a.bounds, a.n, t, s, lane)) * a.d + from;
    load_floats<V>(a.g_last == nullptr ? nullptr : a.g_last + at, 0.0f, g);
}

// One row: gx and ggate of G, `whole`; h: the state before it. z and c = 1 - z from the factor; z c (dv/dz x - h) is (x - h) z c (tied), -h z c
// (free) or, with u = 2 - z = 1 + c, (x c root / u - h z) c (normed).
template <int KIND>
__device__ __forceinline__ void row_back(float factor, float root, float x_t, float h, float whole, float& gx, float& ggate) {
    const float c = factor_rest(factor), z = is_rest(factor) ? 1.0f + factor : factor;
    if constexpr (KIND == kTied) {
        gx = whole * z;
        ggate = gx * (x_t - h) * c;
    } else if constexpr (KIND == kFree) {
        gx = whole;
        ggate = whole * -h * z * c;
    } else {
        gx = whole * root;
        ggate = whole * c * fmaf(x_t * c * root, __builtin_amdgcn_rcpf(1.0f + c), -h * z);
    }
}

// As `again`; returns the wave's sums of the bias's gradient.
template <int V>
struct Columns {
    float of[V];
};
template <typename T, int V, int KIND>
__device__ __attribute__((noinline)) Columns<V> back_again(const void* arguments, uint32_t t0, uint32_t column, const float* enters) {
    using C = Cell<T, V>;
    constexpr int R = kBackRows;
    const ScanBackward a = *static_cast<const ScanBackward*>(arguments);
    const uint32_t lane = __lane_id(), from = column < a.d ? column : 0;
    t0 = uniform(t0);
    const Rows<R> rows(a.bounds, a.n, t0, lane, Rows<R>::cache(a.bounds, a.n, lane));
    float bias[V], fast[V], g[V];
    Columns<V> sums = {};
    load_floats<V>(a.bias == nullptr ? nullptr : a.bias + from, 0.0f, bias);
#pragma unroll
    for (int v = 0; v < V; ++v) g[v] = fast[v] = enters[v * kWave + lane];
    uint32_t s = rows.behind;
#pragma unroll 1
    for (int r = R - 1; r >= 0; --r) {
        const uint32_t t = t0 + r;
        if (!(rows.live >> r & 1)) continue;
        if (rows.ends >> r & 1) {
            end_at<V>(a, t, s, lane, from, g);
#pragma unroll
            for (int v = 0; v < V; ++v) fast[v] = g[v];
        }
        const bool begins = rows.begins >> r & 1;
        const typename C::Raw gate_t = C::load(a.gate, a.gate_stride, t, from), gh_t = C::load(a.gh, a.gh_stride, t, from);
        const typename C::Raw x_t = C::load(a.x, a.x_stride, t, from), before_t = C::load(a.h, a.h_stride, t == 0 ? 0 : t - 1, from);
        float h[V], gx[V], ggate[V];
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = C::get(before_t, v);
        if (begins) {
            sequence_of(a.bounds, a.n, t, s, lane);
            load_floats<V>(a.state == nullptr ? nullptr : a.state + static_cast<uint64_t>(s) * a.d + from, 0.0f, h);
        }
        bool stays = true;  // what was stored
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const Gate<sizeof(T) == 4> at(-C::get(gate_t, v) - bias[v]);
            const float whole = g[v] + C::get(gh_t, v);
            row_back<KIND>(at.f, at.root, C::get(x_t, v), h[v], whole, gx[v], ggate[v]);
            sums.of[v] += ggate[v];
            stays &= finite(fast[v]);
            fast[v] = passed(at.f, fast[v] + C::get(gh_t, v));
            stays &= !begins || finite(fast[v]);
            g[v] = finite(fast[v]) ? fast[v] : defined(at.f, whole, 0.0f);
        }
        if (column >= a.d || stays) continue;
        if (begins && a.g_state != nullptr) {
            const uint64_t at = static_cast<uint64_t>(s) * a.d + column;
#pragma unroll
            for (int v = 0; v < V; ++v) a.g_state[at + v] = g[v];
        }
        C::store(a.gx, t, a.d, column, gx);
        C::store(a.g_gate, t, a.d, column, ggate);
    }
    return sums;
}

template <typename T, int V, int KIND>
__global__ __launch_bounds__(kWaves* kWave, 8) void scan_back_kernel(ScanBackward a, uint32_t slices, uint32_t tiles) {
    using C = Cell<T, V>;
    constexpr bool FINE = sizeof(T) == 4;
    constexpr int R = kBackRows;
    constexpr uint32_t kTileRows = kWaves * R;
    __shared__ Carry<V> lds;
    const Chain chain(a.steps, tiles, a.d);
    const uint32_t cached = Rows<R>::cache(a.bounds, a.n, threadIdx.x % kWave);
    const Place place(chain, slices, &lds.ticket);
    const uint32_t lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave), column = (place.slice * kWave + lane) * V, tile = tiles - 1 - place.tile;
    const uint32_t t0 = tile * kTileRows + wave * R;
    const bool here = column < a.d;
    const uint32_t from = here ? column : 0;
    typename C::Raw gate[R], gh[R], x[R], before[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint32_t t = t0 + r < a.n ? t0 + r : a.n - 1;
        gate[r] = C::load(a.gate, a.gate_stride, t, from);
        gh[r] = C::load(a.gh, a.gh_stride, t, from);
    }
    float bias[V];
    load_floats<V>(a.bias == nullptr ? nullptr : a.bias + from, 0.0f, bias);
#pragma unroll
    for (int r = 0; r < R; ++r) {  // wanted by the second walk alone: the first does not wait for them
        const uint32_t t = t0 + r < a.n ? t0 + r : a.n - 1;
        x[r] = C::load(a.x, a.x_stride, t, from);
        before[r] = C::load(a.h, a.h_stride, t == 0 ? 0 : t - 1, from);
    }
    const Rows<R> rows(a.bounds, a.n, t0, lane, cached);
    if (threadIdx.x == (kWaves - 1) * kWave)  // in the order of the walk
        lds.reach = rows.ends >> (R - 1) & 1 || rows.after == 0 ? place.tile : tiles - 1 - (rows.after - 1) / kTileRows;
    // Factors are kept between the walks; the normed kind, which would have to keep roots too, computes both again.
    const auto gate_of = [&](int r, int v) { return Gate<FINE>(-C::get(gate[r], v) - bias[v]); };
    float f[R][V];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int v = 0; v < V; ++v) f[r][v] = gate_of(r, v).f;
    const auto sequence = [&](uint32_t t, uint32_t& s) { return sequence_of(a.bounds, a.n, t, s, lane); };
    const auto end = [&](uint32_t t, uint32_t& s, float (&g)[V]) { end_at<V>(a, t, s, lane, from, g); };
    const bool good = by_rows(rows, [&](auto plain) {
        Summary<V> sum;
        uint32_t s = rows.behind;
#pragma unroll
        for (int r = R - 1; r >= 0; --r) {
            if constexpr (!plain) {
                if (!(rows.live >> r & 1)) continue;
                if (rows.ends >> r & 1) end(t0 + r, s, sum.b);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) {
                sum.b[v] = passed(f[r][v], sum.b[v] + C::get(gh[r], v));
                sum.row(v, f[r][v]);
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) lds.steps[wave][v][lane] = sum.step(v, rows.ends != 0);
        return all_finite<V>(sum.b);
    });
    if (__builtin_expect(__ballot(!good) != 0, 0)) {  // as in the forward
        const int first = __ffs(static_cast<int>(rows.ends)) - 1;  // the first row where a sequence ends
        float sum[V] = {};
        uint32_t s = rows.behind;
        if (first >= 0) end(t0 + first, s, sum);
#pragma unroll
        for (int r = R - 1; r >= 0; --r)
            if ((first < 0 || r <= first) && rows.live >> r & 1)
#pragma unroll
                for (int v = 0; v < V; ++v) sum[v] += C::get(gh[r], v);
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (!finite(sum[v]) && !finite(lds.steps[wave][v][lane].b)) lds.steps[wave][v][lane].b = sum[v];
    }
    carry<V>(lds, chain, place.tile, a.d, column, here, lane, wave, [](uint32_t w) { return kWaves - 1 - w; });
    float g[V], g_bias[V] = {};
#pragma unroll
    for (int v = 0; v < V; ++v) g[v] = lds.enters[wave][v][lane];
    by_rows(rows, [&](auto plain) {
        uint32_t s = rows.behind;
#pragma unroll
        for (int r = R - 1; r >= 0; --r) {
            const uint32_t t = t0 + r;
            float gx[V] = {}, ggate[V] = {}, h[V];
            bool live = true, begins = false;
            if constexpr (!plain) {
                if (t >= a.n) continue;
                live = rows.live >> r & 1;
                begins = live && (rows.begins >> r & 1);
                if (live && (rows.ends >> r & 1)) end(t, s, g);
            }
            if (begins) {
                sequence(t, s);
                load_floats<V>(a.state == nullptr ? nullptr : a.state + static_cast<uint64_t>(s) * a.d + from, 0.0f, h);
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v) h[v] = C::get(before[r], v);
            }
            if (live)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    float factor, root = 1.0f;
                    if constexpr (KIND == kNormed) {
                        if (v == 0) asm volatile("" : "+v"(gate[r]));  // or the compiler keeps the first walk's values, in scratch memory
                        const Gate<FINE> again = gate_of(r, v);
                        factor = again.f;
                        root = again.root;
                    } else {
                        factor = f[r][v];
                    }
                    const float whole = g[v] + C::get(gh[r], v);
                    row_back<KIND>(factor, root, C::get(x[r], v), h[v], whole, gx[v], ggate[v]);
                    g_bias[v] += ggate[v];
                    g[v] = passed(factor, whole);
                }
            if (!here) continue;
            if (begins && a.g_state != nullptr) {
                const uint64_t at = static_cast<uint64_t>(s) * a.d + column;
#pragma unroll
                for (int v = 0; v < V; ++v) a.g_state[at + v] = g[v];
            }
            C::store(a.gx, t, a.d, column, gx);
            C::store(a.g_gate, t, a.d, column, ggate);
        }
    });
    if (__builtin_expect(__ballot(!all_finite<V>(g_bias)) != 0, 0)) {  // as G times anything is where G is not
        const Columns<V> sums = back_again<T, V, KIND>((const void*)__builtin_amdgcn_kernarg_segment_ptr(), t0, column, &lds.enters[wave][0][0]);
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (!finite(g_bias[v])) g_bias[v] = sums.of[v];
    }
    __syncthreads();  // what enters was read
#pragma unroll
    for (int v = 0; v < V; ++v) lds.enters[wave][v][lane] = g_bias[v];
    __syncthreads();
    const uint32_t mine = column + wave;
    if (wave >= V || !here) return;
    float all = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) all += lds.enters[w][wave][lane];
    a.partials[static_cast<uint64_t>(tile) * a.d + mine] = all;
}

// out[i] = the sum over the tiles of partials[tile][i], in a fixed order: 64 columns a block, 16 waves over the tiles (4 to 5 us for 128
// tiles of 1024 columns; atomics would not keep the order).
constexpr uint32_t kBiasWaves = 16;
__global__ __launch_bounds__(kBiasWaves* kWave) void bias_kernel(const float* __restrict__ partials, float* out, uint32_t tiles, uint32_t d) {
    __shared__ float lds[kBiasWaves][kWave];
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, column = blockIdx.x * kWave + lane;
    float sum = 0.0f;
    if (column < d)
#pragma unroll 4
        for (uint32_t tile = wave; tile < tiles; tile += kBiasWaves) sum += partials[static_cast<uint64_t>(tile) * d + column];
    lds[wave][lane] = sum;
    __syncthreads();
    if (wave != 0 || column >= d) return;
    sum = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < kBiasWaves; ++w) sum += lds[w][lane];
    out[column] = sum;
}

// One token of each of n sequences: the state in place, float32. A thread an entry; 16 sequences of 2048 channels take 2.4 us, a launch.
template <typename T, int KIND>
__global__ __launch_bounds__(256) void step_kernel(ScanStep a) {
    const uint32_t column = blockIdx.y * 256 + threadIdx.x, row = blockIdx.x;
    if (column >= a.d) return;
    const float x = widen(static_cast<const T*>(a.x)[row * a.x_stride + column]);
    const Gate<sizeof(T) == 4> g(-widen(static_cast<const T*>(a.gate)[row * a.gate_stride + column]) - (a.bias == nullptr ? 0.0f : a.bias[column]));
    float* const state = a.state + row * a.state_stride + column;
    const float h = defined(g.f, *state, product(input<KIND>(g), x));
    *state = h;
    T* const out = static_cast<T*>(a.h) + static_cast<uint64_t>(row) * a.d + column;
    if constexpr (sizeof(T) == 4) *out = h;
    else *out = bf16_bits(h);
}

uint32_t scan_tiles(uint32_t n, int rows) { return (n + kWaves * rows - 1) / (kWaves * rows); }

// Whether two bfloat16 columns can be read and written as one 32-bit word everywhere. Rows of which that does not hold go one column a
// lane, at half the bytes a request.
bool word_pairs(uint32_t d, std::initializer_list<const void*> rows, std::initializer_list<uint64_t> strides) {
    if (d % 2 != 0) return false;
    for (const void* p : rows)
        if (reinterpret_cast<uintptr_t>(p) % 4 != 0) return false;
    for (uint64_t s : strides)
        if (s % 2 != 0) return false;
    return true;
}

// Before the scan, where there is something to do: more than one tile, or sequences that may be empty.
hipError_t prepare(void* workspace, uint32_t tiles, const ScanBounds& bounds, uint32_t n, const float* from, float* to, uint32_t d, hipStream_t stream) {
    const uint64_t words = tiles > 1 ? Chain::words(tiles, d) : 0;
    const uint32_t fillers = static_cast<uint32_t>(std::min<uint64_t>((words + 4 * kPrepareThreads - 1) / (4 * kPrepareThreads), 1024));
    const uint32_t sequences = bounds.p != nullptr && to != nullptr ? bounds.count : 0;
    if (fillers + sequences == 0) return hipSuccess;
    hipLaunchKernelGGL(prepare_kernel, dim3(fillers + sequences), dim3(kPrepareThreads), 0, stream, static_cast<Word*>(workspace), words, fillers, bounds, n, from, to, d);
    return hipGetLastError();
}

template <typename T, int V, int KIND>
hipError_t forward(const ScanForward& a, hipStream_t stream) {
    const uint32_t slices = (a.d + kWave * V - 1) / (kWave * V), tiles = scan_tiles(a.n, forward_rows(sizeof(T) == 4));
    if (const hipError_t status = prepare(a.steps, tiles, a.bounds, a.n, a.state, a.last, a.d, stream); status != hipSuccess) return status;
    hipLaunchKernelGGL((scan_kernel<T, V, KIND>), dim3(slices * tiles), dim3(kWaves * kWave), 0, stream, a, slices, tiles);
    return hipGetLastError();
}

template <typename T, int V, int KIND>
hipError_t backward(const ScanBackward& call, hipStream_t stream) {
    ScanBackward a = call;
    const uint32_t slices = (a.d + kWave * V - 1) / (kWave * V), tiles = scan_tiles(a.n, kBackRows);
    a.partials = reinterpret_cast<float*>(static_cast<Word*>(a.steps) + Chain::words(tiles, a.d));
    if (const hipError_t status = prepare(a.steps, tiles, a.bounds, a.n, a.g_last, a.g_state, a.d, stream); status != hipSuccess) return status;
    hipLaunchKernelGGL((scan_back_kernel<T, V, KIND>), dim3(slices * tiles), dim3(kWaves * kWave), 0, stream, a, slices, tiles);
    if (const hipError_t status = hipGetLastError(); status != hipSuccess) return status;
    hipLaunchKernelGGL(bias_kernel, dim3((a.d + kWave - 1) / kWave), dim3(kBiasWaves * kWave), 0, stream, a.partials, a.g_bias, tiles, a.d);
    return hipGetLastError();
}

template <typename F>
hipError_t with_kind(int kind, F&& f) {
    if (kind == kTied) return f(std::integral_constant<int, kTied>());
    if (kind == kNormed) return f(std::integral_constant<int, kNormed>());
    return f(std::integral_constant<int, kFree>());
}

}  // namespace

uint64_t scan_workspace_bytes(uint32_t n, uint32_t d, bool gradients) {
    const uint32_t tiles = scan_tiles(n, 8);  // the most tiles of any variant
    return Chain::words(tiles, d) * sizeof(Word) + (gradients ? static_cast<uint64_t>(tiles) * d * sizeof(float) : 0);
}

hipError_t launch_scan(int vt, const ScanForward& a, hipStream_t stream) {
    return with_kind(a.kind, [&](auto kind) {
        if (vt == kF32) return forward<float, 1, kind>(a, stream);
        return word_pairs(a.d, {a.x, a.gate, a.h}, {a.x_stride, a.gate_stride}) ? forward<uint16_t, 2, kind>(a, stream) : forward<uint16_t, 1, kind>(a, stream);
    });
}

hipError_t launch_scan_backward(int vt, const ScanBackward& a, hipStream_t stream) {
    return with_kind(a.kind, [&](auto kind) {
        if (vt == kF32) return backward<float, 1, kind>(a, stream);
        return word_pairs(a.d, {a.x, a.gate, a.h, a.gh, a.gx, a.g_gate}, {a.x_stride, a.gate_stride, a.h_stride, a.gh_stride}) ? backward<uint16_t, 2, kind>(a, stream)
                                                                                                                           : backward<uint16_t, 1, kind>(a, stream);
    });
}

hipError_t launch_scan_step(int vt, const ScanStep& a, hipStream_t stream) {
    const dim3 grid(a.n, (a.d + 255) / 256);
    return with_kind(a.kind, [&](auto kind) {
        if (vt == kF32) hipLaunchKernelGGL((step_kernel<float, kind>), grid, dim3(256), 0, stream, a);
        else hipLaunchKernelGGL((step_kernel<uint16_t, kind>), grid, dim3(256), 0, stream, a);
        return hipGetLastError();
    });
}

}  // namespace hffn
