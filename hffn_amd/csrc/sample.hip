// One token a row from its logits and a given uniform number. With w_j = exp((z_j - max z) / T), entries ordered by z descending
// and index ascending: top-k, top-p and min-p each keep a prefix of that order, so what is kept is every key above a threshold
// and the first few at it. Weights are whole numbers, w 2^bits rounded: their sums are the same in any order, so that the
// histograms may be added to by whatever lane comes first.
//
// A row is one block's, read three or four times (from the caches after the first). Thresholds are looked for among a few of
// the largest entries, kept aside: for top-k those at or above the k-th largest of the threads' own maxima, which are at least k; for
// top-p alone those up to the bin of one weighted histogram over the row in which the target is reached.
//
// Bound by one CU's chain for a row, not by memory: 50304 logits are 50 entries a lane, a pass that weighs them all in float64 takes
// some 10 us, and every histogram is a chain of barriers and atomics in LDS. Measured, us a call: one row of 50304
// float32, top-p 37 where what it keeps fits the list, 45 to 63 else (the draw weighs the row again); 256 rows, bfloat16, all filters
// mixed, 50 to 64 (26 MB: 0.5 TB/s; the slowest row's chain); 17 rows of 32003 float32, no filter, 24. A sort of the row would be some 12 passes over it.
#include "common.hpp"
#include "launch.hpp"

namespace hffn {
namespace {

constexpr uint32_t kThreads = 1024, kWaves = kThreads / kWave;
constexpr uint32_t kBins = 2048;  // of a histogram: 11 bits of a key
constexpr uint32_t kList = 2048;  // entries kept aside at most (4096 and 6144: the same times for one row, 2 us more for 256)
constexpr uint32_t kTable = 256;

typedef unsigned long long Sum;

// Order-preserving bits of a logit: 0 for minus infinity and NaN, which are never drawn; both zeros the same (the key below theirs
// would be the negative one's: no logit has it, and a float made of it is no smaller than zero).
constexpr uint32_t kZeroKey = 0x80000000u;
__device__ __forceinline__ uint32_t order_key(float z) {
    const uint32_t bits = __float_as_uint(z + 0.0f), key = bits ^ (static_cast<uint32_t>(static_cast<int>(bits) >> 31) | 0x80000000u);
    return z > -INFINITY ? key : 0;
}
// bfloat16 keys are the upper halves, the lower ones zero.
template <typename T>
__device__ __forceinline__ uint32_t row_key(float z) { return sizeof(T) == 4 ? order_key(z) : order_key(z) & 0xffff0000u; }
template <typename T>
__device__ __forceinline__ float key_logit(uint32_t key) {
    const uint32_t bits = key ^ (static_cast<uint32_t>(static_cast<int>(~key) >> 31) | 0x80000000u);
    return key == 0 ? -INFINITY : __uint_as_float(sizeof(T) == 4 ? bits : bits & 0xffff0000u);
}

struct Lds {
    double table[kTable];
    Sum bins[kBins];  // zeros between the histograms
    uint32_t keys[kList], indices[kList];
    Sum sums[kWaves], ties[kWaves];
    uint32_t words[kWaves];
    uint32_t count, digit;
    Sum above, at;
};

// Weights of a row's logits: exp(y), y = (z - top) / T, 2^bits, rounded. For y of -20 and above in float64: with s = y / ln 2 in
// 256ths = n + f, 2^floor(n / 256) by the exponent's bits, 2^((n mod 256) / 256) from a table and 2^(f / 256), |f| <= 1 / 2, by its Taylor series
// to the 4th power (remainder 4e-17). Below (weights under 2^-28) float32 is enough: what it is off by, 2^-18 of the weight, is
// 2^-46 of the largest.
struct Weights {
    const double* table;
    double top, rate;  // 256 / (T ln 2)
    float top_single, rate_single;
    int bits;
    bool infinite;  // the largest logit is: it and its equals take all
    __device__ __forceinline__ Weights(const double* table, float largest, float temperature, int bits)
        : table(table), top(largest), rate(kTable * 1.4426950408889634 / static_cast<double>(temperature)), top_single(largest), rate_single(fminf(1.0f / temperature, 3.402823466e38f)), bits(bits), infinite(largest == INFINITY) {}
    // exp(y) 2^up, for y down to -690 (2^(up - 1000) below)
    __device__ __forceinline__ double scaled(float z, int up) const {
        constexpr double L = 0.6931471805599453 / kTable, kWhole = 6755399441055744.0;  // added to a number, 1.5 2^52 leaves it rounded in the low bits
        const double s = fmax((z - top) * rate, -1000.0 * kTable), moved = s + kWhole, f = s - (moved - kWhole);
        const int n = static_cast<int>(__double_as_longlong(moved));
        double p = L * L * L * L / 24.0;
        p = fma(p, f, L * L * L / 6.0);
        p = fma(p, f, L * L / 2.0);
        p = fma(p, f, L);
        p = fma(p, f, 1.0) * table[n & (kTable - 1)];
        return __longlong_as_double(__double_as_longlong(p) + (static_cast<long long>((n >> 8) + up) << 52));
    }
    __device__ __forceinline__ double real(float z) const { return infinite ? z == INFINITY ? 1.0 : 0.0 : scaled(z, 0); }
    __device__ __forceinline__ float below(float z) const { return (z - top_single) * rate_single; }
    // of z above minus infinity (others give anything)
    __device__ __forceinline__ Sum of(float z) const {
        if (infinite) return z == INFINITY ? 1ull << bits : 0;
        const float y = below(z);
        if (y < -20.0f) {
            const float w = __builtin_amdgcn_exp2f(y * 1.44269504f);
            return static_cast<uint32_t>(__builtin_amdgcn_ldexpf(w, bits) + 0.5f);
        }
        return static_cast<Sum>(__double_as_longlong(scaled(z, bits) + 4503599627370496.0)) & 0xfffffffffffffull;  // the low bits of the sum with 2^52
    }
    // The lowest z whose weight is at least `low`, in (0, 1], among the floats near where the logarithm says (minus infinity: all weights are).
    __device__ __forceinline__ float lowest(float low, float temperature, uint32_t lane) const {
        const double at = top + log(static_cast<double>(low)) * temperature;
        const uint32_t key = order_key(static_cast<float>(at));
        if (key <= 32) return -INFINITY;
        const float z = key_logit<float>(key - 32 + lane);
        const uint64_t enough = __ballot(z <= top_single && real(z) >= low);
        return key_logit<float>(key - 32 + __ffsll(static_cast<long long>(enough)) - 1);
    }
    // the bin of z: a 100th of the scale of y each, the largest first, everything beyond 20 in the last
    __device__ __forceinline__ uint32_t bin(float z) const {
        const float y = below(z) * -100.0f;
        return y < kBins - 1 ? static_cast<uint32_t>(y) : infinite && z == INFINITY ? 0 : kBins - 1;
    }
};

// Sums over the lanes up to each, on the vector unit's lane paths: 1, 2, 4 and 8 lanes on within the rows of 16, then the rows' last lanes to
// the rows behind.
template <int CTRL, int ROWS>
__device__ __forceinline__ Sum moved(Sum v) {
    const int low = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, false);
    const int high = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, ROWS, 0xf, false);
    return static_cast<Sum>(static_cast<uint32_t>(high)) << 32 | static_cast<uint32_t>(low);
}
__device__ __forceinline__ Sum wave_through(Sum v) {
    v += moved<0x111, 0xf>(v);
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);
    v += moved<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ Sum of_lane(Sum v, uint32_t lane) {
    const uint32_t low = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane)),
                   high = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane));
    return static_cast<Sum>(high) << 32 | low;
}
__device__ __forceinline__ Sum wave_total(Sum v) { return of_lane(wave_through(v), kWave - 1); }

// Sums over the waves: (of those before this one, of all). The values lie in `sums`, one a wave, behind a barrier.
__device__ __forceinline__ Sum waves_through(const Sum* sums) {
    const uint32_t lane = threadIdx.x % kWave;
    return wave_through(lane < kWaves ? sums[lane] : 0);
}
__device__ __forceinline__ Sum block_total(Sum v, Lds& lds) {
    v = wave_total(v);
    __syncthreads();  // the last totals were read
    if (threadIdx.x % kWave == 0) lds.sums[threadIdx.x / kWave] = v;
    __syncthreads();
    return of_lane(waves_through(lds.sums), kWaves - 1);
}
__device__ __forceinline__ uint32_t block_most(uint32_t v, Lds& lds) {
#pragma unroll
    for (int step = 1; step < kWave; step *= 2) v = max(v, static_cast<uint32_t>(__shfl_xor(v, step)));
    __syncthreads();
    if (threadIdx.x % kWave == 0) lds.words[threadIdx.x / kWave] = v;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) v = max(v, lds.words[w]);
    return v;
}

struct Threshold {
    uint32_t key;  // entries above it are kept
    Sum above;     // what they come to
    Sum at;        // what the entries at it come to
};

// Which of the bins, from the first (DOWN: the last) on, is the one with which `above` and their sums reach `target`. The bins are
// zeros afterwards.
template <bool DOWN>
__device__ __forceinline__ Threshold reach(Sum above, Lds& lds, Sum target) {
    const uint32_t lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave), pair = DOWN ? kThreads - 1 - threadIdx.x : threadIdx.x;
    __syncthreads();
    const Sum one = lds.bins[2 * pair], two = lds.bins[2 * pair + 1], first = DOWN ? two : one, second = DOWN ? one : two;
    lds.bins[2 * pair] = lds.bins[2 * pair + 1] = 0;
    const Sum through = wave_through(first + second);
    if (lane == kWave - 1) lds.sums[wave] = through;
    __syncthreads();
    const Sum waves = waves_through(lds.sums), before = above + through - first - second + (wave == 0 ? 0 : of_lane(waves, wave - 1));
    if (before < target && before + first >= target) {
        lds.digit = DOWN ? 2 * pair + 1 : 2 * pair;
        lds.above = before;
        lds.at = first;
    } else if (before + first < target && before + first + second >= target) {
        lds.digit = DOWN ? 2 * pair : 2 * pair + 1;
        lds.above = before + first;
        lds.at = second;
    }
    __syncthreads();
    return {lds.digit, lds.above, lds.at};
}

// The largest key at and above which the entries reach `target` (at least 1, at most their sum), the topmost `bits` bits of the keys
// counting, 11 at a time by histograms. each(wanted, add): for every entry of the thread with wanted(key), add(key, sum).
template <typename EACH>
__device__ __forceinline__ Threshold select(EACH&& each, Sum target, int bits, Lds& lds) {
    Threshold t = {0, 0, 0};
    uint32_t prefix = 0, mask = 0;
#pragma unroll 1
    for (int shift = 21; shift > 21 - bits; shift -= 11) {
        // the last 11 of 32 bits overlap the 11 before them by one
        const int down = shift > 0 ? shift : 0;
        each([&](uint32_t key) { return (key & mask) == prefix; }, [&](uint32_t key, Sum sum) { atomicAdd(&lds.bins[key >> down & (kBins - 1)], sum); });
        t = reach<true>(t.above, lds, target);
        prefix |= t.key << down;
        mask |= (kBins - 1) << down;
    }
    t.key = prefix;
    return t;
}

// A row, read 16 bytes of every lane at a time, 4 (bfloat16: 8) adjacent entries, or, where rows start anywhere or end inside 16
// bytes (not WHOLE), one entry of every lane.
template <typename T, bool WHOLE>
struct Row {
    static constexpr uint32_t E = WHOLE ? 16 / sizeof(T) : 1, U = WHOLE ? 4 : 8;
    struct Raw { T z[E]; };
    const T* z;
    uint32_t count;
    __device__ __forceinline__ Raw load(uint32_t first, uint32_t end) const {
        Raw raw;
        if constexpr (WHOLE) {
            const uint4 v = first < end ? *reinterpret_cast<const uint4*>(z + first) : make_uint4(0, 0, 0, 0);
            __builtin_memcpy(&raw, &v, 16);
        } else {
            raw.z[0] = first < end ? z[first] : T(0);
        }
        return raw;
    }
    // f(z, index) of the entries in [begin, end), `stride` lanes from lane `at` on; z is NaN beyond the end; U loads are in flight at a
    // time. WHOLE: begin and end are multiples of E, or end the row's.
    template <typename F>
    __device__ __forceinline__ void each(uint32_t begin, uint32_t end, uint32_t at, uint32_t stride, F&& f) const {
        each_piece(begin, end, at, stride, [&](const float (&v)[E], uint32_t first) {
#pragma unroll
            for (uint32_t e = 0; e < E; ++e) f(v[e], first + e);
        });
    }
    // the same by pieces: f(z of E entries, the first's index)
    template <typename F>
    __device__ __forceinline__ void each_piece(uint32_t begin, uint32_t end, uint32_t at, uint32_t stride, F&& f) const {
        for (uint32_t base = begin + at * E; base - at * E < end; base += U * stride * E) {
            Raw raw[U];
#pragma unroll
            for (uint32_t q = 0; q < U; ++q) raw[q] = load(base + q * stride * E, end);
#pragma unroll
            for (uint32_t q = 0; q < U; ++q) {
                const uint32_t first = base + q * stride * E;
                if (first - at * E >= end) break;
                float v[E];
#pragma unroll
                for (uint32_t e = 0; e < E; ++e) v[e] = (WHOLE ? first : first + e) < end ? widen(raw[q].z[e]) : __builtin_nanf("");
                f(v, first);
            }
        }
    }
    template <typename F>
    __device__ __forceinline__ void each(F&& f) const { each(0, count, threadIdx.x, kThreads, f); }
};

template <typename T, bool WHOLE>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleCall a, int bits) {
    __shared__ Lds lds;
    constexpr int kKeyBits = sizeof(T) == 4 ? 32 : 16;
    const uint32_t lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave), at_row = blockIdx.x;
    const float temperature = a.temperatures == nullptr ? a.temperature : a.temperatures[at_row], u = a.uniform[at_row];
    const float top_p = a.top_ps == nullptr ? a.top_p : a.top_ps[at_row], min_p = a.min_ps == nullptr ? a.min_p : a.min_ps[at_row];
    const int64_t top_k = a.top_ks == nullptr ? a.top_k : a.wide ? static_cast<const int64_t*>(a.top_ks)[at_row] : static_cast<const int32_t*>(a.top_ks)[at_row];
    const Row<T, WHOLE> row{static_cast<const T*>(a.logits) + static_cast<uint64_t>(at_row) * a.stride, a.vocab};
    const uint32_t k = top_k > 0 && top_k < row.count ? static_cast<uint32_t>(top_k) : 0;  // 0: off
    if (threadIdx.x < kTable) lds.table[threadIdx.x] = exp2(threadIdx.x * (1.0 / kTable));
    lds.bins[threadIdx.x] = lds.bins[threadIdx.x + kThreads] = 0;
    float largest = -INFINITY;
    row.each([&](float z, uint32_t) { largest = fmaxf(largest, z); });  // not a NaN
    const uint32_t own = row_key<T>(largest), most = block_most(own, lds);
    if (most == 0) {  // nothing to draw from
        if (threadIdx.x == 0) {
            a.tokens[at_row] = -1;
            a.probabilities[at_row] = 0.0f;
        }
        return;
    }
    const float top = key_logit<T>(most);
    if (!(temperature > 0.0f) || k == 1) {  // the first of the largest
        uint32_t first = 0;  // as its distance from the end
        row.each([&](float z, uint32_t index) { first = z == top ? max(first, row.count - index) : first; });
        first = block_most(first, lds);
        if (threadIdx.x == 0) {
            a.tokens[at_row] = row.count - first;
            a.probabilities[at_row] = 1.0f;
        }
        return;
    }
    const Weights weights(lds.table, top, temperature, bits);
    const bool nucleus = top_p < 1.0f;

    uint32_t held = 0;
    bool aside = false;  // whether all that is kept is among the entries aside
    // Whether all entries of wanted(z) and its(z) found room; wanted() of an entry holds for every larger one.
    const auto set_aside = [&](auto&& wanted, auto&& its) {
        __syncthreads();
        if (threadIdx.x == 0) lds.count = 0;
        __syncthreads();
        constexpr uint32_t E = Row<T, WHOLE>::E;
        row.each_piece(0, row.count, threadIdx.x, kThreads, [&](const float (&z)[E], uint32_t first) {
            float largest = z[0];
#pragma unroll
            for (uint32_t e = 1; e < E; ++e) largest = fmaxf(largest, z[e]);
            if (!(largest > -INFINITY && wanted(largest)) || *static_cast<volatile uint32_t*>(&lds.count) > kList) return;
#pragma unroll
            for (uint32_t e = 0; e < E; ++e) {
                if (!(z[e] > -INFINITY && wanted(z[e]) && its(z[e]))) continue;
                const uint32_t to = atomicAdd(&lds.count, 1u);
                if (to >= kList) continue;
                lds.keys[to] = row_key<T>(z[e]);
                lds.indices[to] = first + e;
            }
        });
        __syncthreads();
        held = uniform(lds.count);
        return held <= kList;
    };
    const auto all = [](float) { return true; };
    const auto each_aside = [&](auto&& f) {
        for (uint32_t i = threadIdx.x; i < held; i += kThreads) f(lds.keys[i], lds.indices[i]);
    };

    uint32_t least = 0;  // keys above it are kept (0: all),
    Sum ties = 0;        // and this many at it
    if (k != 0) {
        const auto count = [&](auto&& each) {
            return select([&](auto wanted, auto add) { each([&](uint32_t key, uint32_t) { if (key != 0 && wanted(key)) add(key, 1); }); }, k, kKeyBits, lds);
        };
        Threshold t = {0, 0, 0};
        if (k <= kThreads) {
            // by the distance from the largest, all maxima spread over the bins
            const uint32_t threads = static_cast<uint32_t>(block_total(own != 0, lds));
            const float spread = top - key_logit<T>(~block_most(own != 0 ? ~own : 0, lds)), scale = (kBins - 1) / spread;
            const auto bin = [&](float z) {
                const float at = (top - z) * scale;
                return at < kBins - 1 ? static_cast<uint32_t>(at) : kBins - 1;
            };
            uint32_t limit = kBins;
            if (threads >= k) {
                if (own != 0) atomicAdd(&lds.bins[bin(largest)], 1ull);
                limit = uniform(reach<false>(0, lds, k).key);
            }
            aside = set_aside([&](float z) { return limit == kBins || bin(z) <= limit; }, all);
        }
        if (aside) {  // fewer than k where the row has no more
            if (held >= k) t = count(each_aside);
        } else {
            Sum live = 0;
            row.each([&](float z, uint32_t) { live += z > -INFINITY; });
            if (block_total(live, lds) >= k) t = count([&](auto&& f) { row.each([&](float z, uint32_t index) { f(row_key<T>(z), index); }); });
        }
        if (t.at != 0) {
            least = t.key;
            ties = k - t.above;
        }
    }
    if (nucleus) {
        const auto target_of = [&](Sum mass) -> Sum {
            const double share = top_p > 0.0f ? ceil(static_cast<double>(top_p) * static_cast<double>(mass)) : 1.0;
            return share < 1.0 ? 1 : static_cast<Sum>(share);
        };
        const auto weigh = [&](auto&& each, Sum target) {
            return select([&](auto wanted, auto add) {
                each([&](uint32_t key, uint32_t) { if (key != 0 && key >= least && wanted(key)) add(key, weights.of(key_logit<T>(key))); });
            }, target, kKeyBits, lds);
        };
        const auto each_key = [&](auto&& f) { row.each([&](float z, uint32_t index) { f(row_key<T>(z), index); }); };
        Threshold t;
        Sum target;
        if (aside || least != 0) {  // of what top-k left
            const auto mass_of = [&](auto&& each) {
                Sum mass = 0, at = 0;
                each([&](uint32_t key, uint32_t) {
                    if (key > least) mass += weights.of(key_logit<T>(key));
                    at += key == least;
                });
                mass = block_total(mass, lds);
                at = block_total(at, lds);
                return least == 0 ? mass : mass + (at < ties ? at : ties) * weights.of(key_logit<T>(least));
            };
            target = target_of(aside ? mass_of(each_aside) : mass_of(each_key));
            t = aside ? weigh(each_aside, target) : weigh(each_key, target);
        } else {
            // The row's weights by bin; the bin where the target is reached; the entries up to it aside if there is room, else its own.
            Sum mass = 0, far = 0;
            row.each([&](float z, uint32_t) {
                const Sum w = z > -INFINITY ? weights.of(z) : 0;
                const uint32_t bin = weights.bin(z);
                if (bin < kBins - 1) atomicAdd(&lds.bins[bin], w);
                else far += z > -INFINITY ? w : 0;
                mass += w;
            });
            far = wave_total(far);
            if (lane == 0) atomicAdd(&lds.bins[kBins - 1], far);
            target = target_of(block_total(mass, lds));
            const Threshold bin = reach<false>(0, lds, target);
            const uint32_t limit = uniform(bin.key);
            aside = set_aside([&](float z) { return weights.bin(z) <= limit; }, all);
            if (aside) {
                t = weigh(each_aside, target);
            } else {
                const bool its_own = set_aside([&](float z) { return weights.bin(z) <= limit; }, [&](float z) { return weights.bin(z) == limit; });
                t = its_own ? weigh(each_aside, target - bin.above)
                            : weigh([&](auto&& f) { row.each([&](float z, uint32_t index) { if (z > -INFINITY && weights.bin(z) == limit) f(row_key<T>(z), index); }); },
                                    target - bin.above);
                t.above += bin.above;
            }
        }
        const Sum each = weights.of(key_logit<T>(t.key)), need = each == 0 ? ~0ull : (target - t.above + each - 1) / each;
        if (least == 0 || t.key != least || need < ties) {
            least = t.key;
            ties = need;
        }
    }
    // What is kept lies above `lowest`; of its equals the first `ties`. min-p moves it up, to just below the lowest of weight enough.
    float lowest = key_logit<T>(least);
    if (least == 0) ties = 0;
    if (min_p > 0.0f) {
        const float enough = weights.lowest(fminf(min_p, 1.0f), temperature, lane);
        if (enough > lowest) {
            const uint32_t key = order_key(enough);
            lowest = key_logit<float>(key - (key == kZeroKey ? 2 : 1));
            ties = 0;
        }
    }
    const Sum each = ties == 0 ? 0 : weights.of(lowest);
    const auto drawn = [&](Sum total) -> Sum {
        const double at = u > 0.0f ? floor(static_cast<double>(u) * static_cast<double>(total)) : 0.0;
        return at < static_cast<double>(total - 1) ? static_cast<Sum>(at) : total - 1;
    };
    const auto finish = [&](float z, uint32_t index, Sum total) {
        a.tokens[at_row] = index;
        a.probabilities[at_row] = static_cast<float>(ldexp(weights.real(z), bits) / static_cast<double>(total));
    };

    if (aside) {  // the draw is a threshold over the indices, from the lowest on
        const int spread = __clz(static_cast<int>(row.count)), place_bits = 32 - spread;
        const auto place = [&](uint32_t index) { return (row.count - index) << spread; };
        Sum at = 0, total = 0;
        each_aside([&](uint32_t key, uint32_t) {
            const float z = key_logit<T>(key);
            at += z == lowest;
            if (z > lowest) total += weights.of(z);
        });
        at = block_total(at, lds);
        total = block_total(total, lds) + (at < ties ? at : ties) * each;
        uint32_t last_tie = 0;  // ties at or above this place are kept
        if (ties != 0 && at > ties)
            last_tie = select([&](auto wanted, auto add) { each_aside([&](uint32_t key, uint32_t index) {
                if (key_logit<T>(key) == lowest && wanted(place(index))) add(place(index), 1);
            }); }, ties, place_bits, lds).key;
        const Threshold t = select([&](auto wanted, auto add) { each_aside([&](uint32_t key, uint32_t index) {
            if (!wanted(place(index))) return;
            const float z = key_logit<T>(key);
            if (z > lowest) add(place(index), weights.of(z));
            else if (z == lowest && ties != 0 && place(index) >= last_tie) add(place(index), each);
        }); }, drawn(total) + 1, place_bits, lds);
        each_aside([&](uint32_t key, uint32_t index) {
            if (place(index) == t.key) finish(key_logit<T>(key), index, total);
        });
        return;
    }
    // [first, last): where the drawn entry lies, a sixteenth of the range at a time, a wave each; from there on `draw` is counted, `ties`
    // are left
    constexpr uint32_t E = Row<T, WHOLE>::E, kEnd = E * kWave;
    uint32_t first = 0, last = row.count;
    Sum draw = 0, total = 0;
    bool begun = false;
    while (last - first > kEnd || !begun) {
        const uint32_t part = ((last - first + kWaves - 1) / kWaves + kEnd - 1) / kEnd * kEnd;
        const uint32_t begin = first + wave * part < last ? first + wave * part : last, end = last - begin < part ? last : begin + part;
        Sum mass = 0, tied = 0;
        row.each(begin, end, lane, kWave, [&](float z, uint32_t) {
            if (z > lowest) mass += weights.of(z);
            tied += z == lowest;
        });
        mass = wave_total(mass);
        tied = wave_total(tied);
        __syncthreads();
        if (lane == 0) {
            lds.sums[wave] = mass;
            lds.ties[wave] = tied;
        }
        __syncthreads();
        if (!begun) {
            Sum held_ties = 0;
            for (uint32_t w = 0; w < kWaves; ++w) {
                total += lds.sums[w];
                held_ties += lds.ties[w];
            }
            total += (held_ties < ties ? held_ties : ties) * each;
            draw = drawn(total);
            begun = true;
        }
        uint32_t w = 0;
        for (; w + 1 < kWaves; ++w) {
            const Sum kept = lds.ties[w] < ties ? lds.ties[w] : ties, in_part = lds.sums[w] + kept * each;
            if (draw < in_part) break;
            draw -= in_part;
            ties -= kept;
        }
        first = first + w * part < last ? first + w * part : last - 1;
        last = last - first < part ? last : first + part;
    }
    if (wave != 0) return;
    Sum in_lane = 0, lane_ties = 0, sums[E];
    float own_z[E];
    row.each(first, last, lane, kWave, [&](float z, uint32_t) { lane_ties += z == lowest; });
    Sum rank = wave_through(lane_ties) - lane_ties;
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) {
        const uint32_t j = first + lane * E + e;
        own_z[e] = j < last ? widen(row.z[j]) : __builtin_nanf("");
        const bool tie = own_z[e] == lowest;
        sums[e] = own_z[e] > lowest ? weights.of(own_z[e]) : tie && rank < ties ? each : 0;
        rank += tie;
        in_lane += sums[e];
    }
    Sum reached = wave_through(in_lane) - in_lane;
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) {
        if (reached <= draw && draw < reached + sums[e]) finish(own_z[e], first + lane * E + e, total);
        reached += sums[e];
    }
}

}  // namespace

hipError_t launch_sample(int vt, const SampleCall& a, hipStream_t stream) {
    int bits = 50;  // a row's weights sum to at most 2^62 (vocab 2^bits itself may pass 64 bits)
    while (a.vocab > (1ull << 62) >> bits) --bits;
    const uint32_t per = vt == kBF16 ? 8 : 4;
    const bool whole = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && a.vocab % per == 0 && a.stride % per == 0;
#define HFFN_SAMPLE(T, WHOLE) hipLaunchKernelGGL((sample_kernel<T, WHOLE>), dim3(a.n), dim3(kThreads), 0, stream, a, bits)
    if (vt == kBF16) {
        if (whole) HFFN_SAMPLE(uint16_t, true);
        else HFFN_SAMPLE(uint16_t, false);
    } else {
        if (whole) HFFN_SAMPLE(float, true);
        else HFFN_SAMPLE(float, false);
    }
#undef HFFN_SAMPLE
    return hipGetLastError();
}

}  // namespace hffn
