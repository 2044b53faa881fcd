// Softmax cross entropy of a language-model head, from hidden rows x [n, d] and the head's weight [V, d], in pieces of the
// vocabulary and without keeping the logits:
//   l_t = log sum_v exp(x_t . w_v) - x_t . w_label(t),   D = softmax - onehot(label),   gx = f D W,   gw = f D^T x,
// f the gradient's factor (1 / counted tokens for the mean). The forward leaves, per slice of the vocabulary and token, the
// maximum and the sum of exponentials of its logits, and of the last piece (of the only one, mostly) the exponentials
// themselves, where D belongs; the backward turns those into D, computes the other pieces' logits again, and multiplies D
// by the weight's rows and by x.
//
// Every product is out[b][a] = sum_k A[a, k] B[b, k] on 16-bit MFMA operands with float32 sums. bfloat16 calls multiply their
// entries as they are. Many tokens' D is rounded to bfloat16, 2^-8 of an entry as the gradients themselves are: roundings of
// many entries that do not add up (2048 tokens: the gradients' error is 1.9e-3 of them, 1.7e-3 by their own rounding alone), where
// two parts would double two products of three. A few tokens' gradients may come from a single entry of D, and their calls wait for
// the weight and for gw, not for the matrix unit: they hold D in two bfloat16 parts (a step of 1 token of 1024 x 50304 112 us,
// 106 with one).
// float32 calls hold every operand as fp16 hi + lo of the entry times a power of two of its tensor (22 bits down to 2^-12 of
// the largest entry, 2^-34 of that below; D, at most 1, to 2^-38) and take hi hi + hi lo + lo hi. Those of a few tokens read the
// weight as it is and split it where it is multiplied into three bfloat16 parts (no power of two to know first), of whose nine
// products the six down to 2^-16 count, and hold D in float32. Calls whose entries spread too far for one power of two (kSpread)
// take the three parts as well: the kernels of both forms are launched, and what the preparing launches saw says which ones do
// the work. The parts of an infinity cancel: what it enters is NaN.
//
// What bounds it: many tokens, the matrix units and their power. 8192 bfloat16 tokens of 2048 x 50304: five products per half of
// the vocabulary (844 GFLOP each) of 720 to 850 us, 1.0 to 1.17 PFLOP/s; the forward's over the whole vocabulary takes 1508 us, at
// 1.97 GHz with the units busy 54 % of the time, a library product of the same operands 1472 us, at 1.56 GHz and 71 %.
// 2048 tokens of 1024: 232 to 274 us a product (211 GFLOP). 512 float32 tokens of 1024: 184 to 245 us (158 GFLOP in fp16), and 95 us
// that pack the weight (412 MB). One bfloat16 token of 2048: 49 us for the weight's 206 MB, 4.2 TB/s.
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "launch.hpp"

namespace hffn {
namespace {

typedef float Acc __attribute__((ext_vector_type(16)));
typedef short Quad __attribute__((ext_vector_type(4)));
typedef short Frag __attribute__((ext_vector_type(8)));
typedef __bf16 FragB __attribute__((ext_vector_type(8)));
typedef _Float16 FragH __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) Quad* LdsQuad;
typedef __attribute__((address_space(3))) const Frag* LdsFrag;
typedef float Four __attribute__((ext_vector_type(4)));
typedef float Eight __attribute__((ext_vector_type(8)));
typedef uint32_t Words __attribute__((ext_vector_type(4)));
// The same 16 bytes where rows start on their entries' boundaries only; the hardware takes these in one access.
typedef float FourAnywhere __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t WordsAnywhere __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t HalvesAnywhere __attribute__((ext_vector_type(2), aligned(2)));
typedef __attribute__((address_space(3))) const Four* LdsFour;
typedef __attribute__((address_space(3))) const float* LdsFloat;

constexpr int kLift = 10;      // the entry an operand's power of two is taken from lies in [2^9, 2^10) ...
constexpr int kRoom = 5;       // ... and its largest up to kRoom binades above
constexpr int kGradLift = 14;  // |D| <= 1 is kept times 2^kGradLift
// Eight neighbouring entries of a row whose largest lies this many binades below the entry that the tensor's power of two is
// taken from would keep fewer than 20 bits of that largest: one row of 1e7 times the others cost these 1e-3 in their losses. Three
// parts in their place: losses of 512 tokens of 512 x 50304 in 226 us, not 158, steps of 1024 x 50304 in 1300, not 715; the
// launches of the form that does not run cost 1 % of either.
constexpr int kSpread = 14;
// k-tiles whose products are summed in the MFMA accumulators (float32 calls): of two parts, of three (twice the additions; logits of
// 10^3, gx's 2-norm: 1.2e-5 off with 4, below 1e-5 with 1, at the same time)
constexpr int kChain2 = 4, kChain3 = 1;

// What the first launches leave for the others: counted tokens, labels outside the vocabulary, and (float32) the bits of
// the magnitudes that the powers of two are taken from, and of the samples they were first taken from.
struct Meta {
    uint32_t valid, invalid, weight_bits, x_bits, weight_sample, x_sample;
    uint32_t wide;  // float32 of many tokens: entries spread beyond kSpread
};
__device__ __forceinline__ int lift_of(uint32_t bits) {  // e with 2^-e times that magnitude in [2^9, 2^10)
    return bits == 0 ? 0 : ilogbf(__uint_as_float(bits)) - (kLift - 1);
}
__device__ __forceinline__ float grad_factor(const Meta& meta, float scale, bool mean) {
    if (meta.invalid != 0) return __uint_as_float(0x7fc00000u);
    return mean && meta.valid != 0 ? scale / static_cast<float>(meta.valid) : scale;
}

// An exponential in [0, 1] in 16 bits: the float32 without sign, first exponent bit (both 0) and last 14 bits, to the nearest
// (2^-10 of it, down to 2^-126).
__device__ __forceinline__ uint32_t kept_bits(float e) {
    const uint32_t bits = __float_as_uint(e);
    return (bits + 0x1fff + (bits >> 14 & 1)) >> 14 & 0xffff;
}
__device__ __forceinline__ float kept_value(uint32_t bits) { return __uint_as_float((bits & 0xffff) << 14); }
__device__ __forceinline__ float half_value(uint32_t bits) { return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits))); }
__device__ __forceinline__ void split(float v, uint16_t& hi, uint16_t& lo) {
    const _Float16 h = static_cast<_Float16>(v);
    const float rest = v - static_cast<float>(h);
    const _Float16 l = static_cast<_Float16>(fabsf(v) < 65504.0f ? rest : 0.0f);
    hi = __builtin_bit_cast(uint16_t, h);
    lo = __builtin_bit_cast(uint16_t, l);
}

// ------------------------------------------------------------------------------------------------ tokens and operands

__device__ __forceinline__ int64_t label_of(const void* labels, int64_t at, bool wide) {
    return wide ? static_cast<const int64_t*>(labels)[at] : static_cast<const int32_t*>(labels)[at];
}

// What the preparing launches read and write: labels; the counted tokens in order (rows[i] the token of compact row i,
// compact[i] its label or -1 where that lies outside the vocabulary, place[t] the compact row of token t or -1); the operand
// rows of x's counted rows (zeros to the next multiple of 64) and, where it is not read in place, of the weight, as
// [rows][width] bfloat16, float32 (RAW) or, per 32 entries, 32 hi and 32 lo halves; zeros from d on.
struct Prepare {
    const void *labels, *x, *weight;
    int64_t labels_stride, ignore;
    uint64_t x_stride;
    bool wide;
    uint32_t n, d, width, vocab;
    int32_t *rows, *compact, *place;
    float* losses;
    Meta* meta;
    uint16_t *x_out, *w_out, *x_split;  // x_split: RAW, the counted rows of x as per 32 entries 3 x 32 bfloat16 parts
    uint2 *x_most, *w_most;  // float32: the Seen of each block's rows
    uint32_t x_blocks, w_blocks;
};

// Calls of more tokens than kScanTokens: the counted tokens' order, one block. (Below that every block of the preparing
// launch counts the labels itself: a launch less.)
constexpr uint32_t kScanTokens = 4096, kScanThreads = 1024, kScanAhead = 8;
__global__ __launch_bounds__(kScanThreads) void loss_scan_kernel(Prepare p) {
    __shared__ uint32_t counts[kScanThreads / kWave], bad[kScanThreads / kWave];
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    uint32_t base = 0, invalid = 0;
    int64_t ahead[kScanAhead];
    for (uint32_t first = 0; first < p.n; first += kScanThreads) {
        const uint32_t t = first + threadIdx.x, slot = first / kScanThreads % kScanAhead;
        if (slot == 0) {
#pragma unroll
            for (uint32_t k = 0; k < kScanAhead; ++k) {
                const uint32_t at = t + k * kScanThreads;
                ahead[k] = at < p.n ? label_of(p.labels, at * p.labels_stride, p.wide) : p.ignore;
            }
        }
        int64_t label = p.ignore;
#pragma unroll
        for (uint32_t k = 0; k < kScanAhead; ++k) label = slot == k ? ahead[k] : label;
        const bool counted = t < p.n && label != p.ignore, outside = counted && (label < 0 || label >= static_cast<int64_t>(p.vocab));
        const uint64_t mask = __ballot(counted);
        if (lane == 0) counts[wave] = __popcll(mask);
        invalid += outside;
        __syncthreads();
        uint32_t at = base, total = 0;
        for (uint32_t w = 0; w < kScanThreads / kWave; ++w) {
            if (w < wave) at += counts[w];
            total += counts[w];
        }
        at += __popcll(mask & ((uint64_t{1} << lane) - 1));
        if (counted) {
            p.rows[at] = static_cast<int32_t>(t);
            p.compact[at] = outside ? -1 : static_cast<int32_t>(label);
        }
        if (t < p.n) {
            p.place[t] = counted ? static_cast<int32_t>(at) : -1;
            if (!counted) p.losses[t] = 0.0f;
        }
        base += total;
        __syncthreads();
    }
    for (int step = 32; step > 0; step /= 2) invalid += __shfl_xor(invalid, step);
    if (lane == 0) bad[wave] = invalid;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 1; w < kScanThreads / kWave; ++w) invalid += bad[w];
        p.meta->valid = base;
        p.meta->invalid = invalid;
    }
}

__device__ __forceinline__ uint32_t magnitude(float v) {  // bits of |v|, 0 for what is not finite
    const uint32_t bits = __float_as_uint(v) & 0x7fffffffu;
    return bits < 0x7f800000u ? bits : 0u;
}

// What a thread saw of a tensor's finite magnitudes (bits): the largest; and of the largest of every eight neighbours, where not
// zero, the smallest, as its complement (0: none seen), so that both are joined by the larger.
struct Seen {
    uint32_t most = 0, small = 0;
    __device__ __forceinline__ void take(uint32_t of_eight) {
        most = max(most, of_eight);
        if (of_eight != 0) small = max(small, ~of_eight);
    }
    __device__ __forceinline__ void join(uint2 other) {
        most = max(most, other.x);
        small = max(small, other.y);
    }
};

constexpr uint32_t kPrepThreads = 256, kPrepWaves = kPrepThreads / kWave, kWeightRows = 16;  // weight rows a block

// The largest of the threads' values, in every thread (one barrier before and after: lds may be used again).
__device__ __forceinline__ uint32_t block_most(uint32_t v, uint32_t (&lds)[kPrepWaves]) {
    for (int step = 32; step > 0; step /= 2) v = max(v, static_cast<uint32_t>(__shfl_xor(v, step)));
    __syncthreads();
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kPrepWaves; ++w) v = max(v, lds[w]);
    return v;
}

// float32 calls take the powers of two from the largest of 1024 entries spread over a tensor, the same in every block, and
// note each block's largest: only where some entry lies kRoom binades above is the tensor packed again, by its largest.
// (A pass over the weight for its largest first took 60 us of a 1080 us step of 512 tokens of 1024 x 50304.)
constexpr uint32_t kSamples = 4;  // per thread
__device__ __forceinline__ uint32_t sample_of(const Prepare& p, bool of_x, uint32_t (&lds)[kPrepWaves]) {
    uint32_t most = 0;
#pragma unroll
    for (uint32_t k = 0; k < kSamples; ++k) {
        const uint32_t i = k * kPrepThreads + threadIdx.x, column = i * 40503u % p.d, of = kSamples * kPrepThreads;
        const uint64_t row = static_cast<uint64_t>(i) * (of_x ? p.n : p.vocab) / of;
        if (of_x && label_of(p.labels, row * p.labels_stride, p.wide) == p.ignore) continue;
        const float* from = of_x ? static_cast<const float*>(p.x) + row * p.x_stride : static_cast<const float*>(p.weight) + row * p.d;
        most = max(most, magnitude(from[column]));
    }
    return block_most(most, lds);
}

// A float32 as three bfloat16 parts whose sum it is to 2^-24: the pair (low, high)'s into words[0..2].
__device__ __forceinline__ void split_pair(float low, float high, uint32_t (&words)[3]) {
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        words[p] = bf16_pair(low, high);
        low -= __uint_as_float(words[p] << 16);
        high -= __uint_as_float(words[p] & 0xffff0000u);
    }
}

// One operand row by a wave, eight entries a lane and step; `seen`: of the lane's finite magnitudes. RAW: float32 as they are, and
// their parts to `split_to`.
template <typename T, bool RAW>
__device__ __forceinline__ void pack_row(const T* __restrict__ from, uint16_t* __restrict__ to, uint32_t d, uint32_t width, int e,
                                         Seen& seen, uint16_t* __restrict__ split_to = nullptr) {
    const uint32_t lane = threadIdx.x % kWave;
    for (uint32_t c = 8 * lane; c < width; c += 8 * kWave) {
        if constexpr (sizeof(T) == 4) {
            float v[8];
            if (c + 8 <= d) {
#pragma unroll
                for (uint32_t k = 0; k < 8; k += 4) {
                    const FourAnywhere part = *reinterpret_cast<const FourAnywhere*>(from + c + k);
                    v[k] = part[0], v[k + 1] = part[1], v[k + 2] = part[2], v[k + 3] = part[3];
                }
            } else {
#pragma unroll
                for (uint32_t k = 0; k < 8; ++k) v[k] = c + k < d ? from[c + k] : 0.0f;
            }
            if constexpr (RAW) {
                float4* out = reinterpret_cast<float4*>(to + 2 * c);
                out[0] = make_float4(v[0], v[1], v[2], v[3]);
                out[1] = make_float4(v[4], v[5], v[6], v[7]);
                uint32_t words[4][3];
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) split_pair(v[2 * k], v[2 * k + 1], words[k]);
#pragma unroll
                for (uint32_t part = 0; part < 3; ++part)
                    *reinterpret_cast<uint4*>(split_to + c / 32 * 96 + part * 32 + c % 32) =
                        make_uint4(words[0][part], words[1][part], words[2][part], words[3][part]);
                continue;
            }
            uint32_t hi[4], lo[4], most = 0;
#pragma unroll
            for (uint32_t k = 0; k < 8; k += 2) {
                uint16_t h[2], l[2];
                most = max(most, max(magnitude(v[k]), magnitude(v[k + 1])));
                split(ldexpf(v[k], -e), h[0], l[0]);
                split(ldexpf(v[k + 1], -e), h[1], l[1]);
                hi[k / 2] = h[0] | static_cast<uint32_t>(h[1]) << 16;
                lo[k / 2] = l[0] | static_cast<uint32_t>(l[1]) << 16;
            }
            if (c < d && c + 8 > d)  // the row's last entries: with those before them
                for (uint32_t k = d < 8 ? d : 8; k > 0; --k) most = max(most, magnitude(from[d - k]));
            seen.take(most);
            uint16_t* out = to + c / 32 * 64 + c % 32;
            *reinterpret_cast<uint4*>(out) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(out + 32) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        } else {
            WordsAnywhere v;
            if (c + 8 <= d) {
                v = *reinterpret_cast<const WordsAnywhere*>(from + c);
            } else {
                uint32_t words[4];
#pragma unroll
                for (uint32_t k = 0; k < 8; k += 2)
                    words[k / 2] = (c + k < d ? from[c + k] : 0u) | (c + k + 1 < d ? static_cast<uint32_t>(from[c + k + 1]) : 0u) << 16;
                v = WordsAnywhere{words[0], words[1], words[2], words[3]};
            }
            *reinterpret_cast<uint4*>(to + c) = make_uint4(v[0], v[1], v[2], v[3]);
        }
    }
}

// The weight's rows of block `block`.
template <typename T>
__device__ __forceinline__ void pack_weight(const Prepare& p, uint32_t block, int e, Seen& seen) {
    constexpr uint64_t kParts = sizeof(T) == 4 ? 2 : 1;
    for (uint32_t r = threadIdx.x / kWave; r < kWeightRows; r += kPrepWaves) {
        const uint64_t row = static_cast<uint64_t>(block) * kWeightRows + r;
        if (row < p.vocab) pack_row<T, false>(static_cast<const T*>(p.weight) + row * p.d, p.w_out + row * kParts * p.width, p.d, p.width, e, seen);
    }
}

// Compact row i of x_split to zeros, by a wave.
__device__ __forceinline__ void clear_split(const Prepare& p, uint32_t i) {
    uint4* parts = reinterpret_cast<uint4*>(p.x_split + static_cast<uint64_t>(i) * 3 * p.width);
    for (uint32_t c = threadIdx.x % kWave; c < 3 * p.width / 8; c += kWave) parts[c] = make_uint4(0, 0, 0, 0);
}

// A block per kPrepWaves tokens (a wave each, and the compact row of the same number where zeros belong) and, after those,
// one per kWeightRows weight rows to pack.
template <typename T, bool RAW>
__global__ __launch_bounds__(kPrepThreads) void loss_prepare_kernel(Prepare p) {
    constexpr uint64_t kParts = sizeof(T) == 4 ? 2 : 1;
    constexpr bool kScaled = sizeof(T) == 4 && !RAW;
    __shared__ uint32_t most_lds[kPrepWaves], sums[kPrepWaves][3];
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    if (!RAW && blockIdx.x >= p.x_blocks) {
        const uint32_t block = blockIdx.x - p.x_blocks;
        int e = 0;
        if constexpr (kScaled) {
            const uint32_t sample = sample_of(p, false, most_lds);
            e = lift_of(sample);
            if (block == 0 && threadIdx.x == 0) p.meta->weight_sample = sample;
        }
        Seen seen;
        pack_weight<T>(p, block, e, seen);
        if constexpr (kScaled) {
            const uint2 all = make_uint2(block_most(seen.most, most_lds), block_most(seen.small, most_lds));
            if (threadIdx.x == 0) p.w_most[block] = all;
        }
        return;
    }
    const uint32_t first = blockIdx.x * kPrepWaves, i = first + wave;
    uint32_t valid, at = 0;
    bool counted = false;
    if (p.n > kScanTokens) {
        valid = p.meta->valid;
        const int32_t here = i < p.n ? p.place[i] : -1;
        counted = here >= 0;
        at = static_cast<uint32_t>(here);
    } else {
        uint32_t before = 0, all = 0, outside = 0;  // counted tokens before the block's, all, and those outside, of this wave
        for (uint32_t t = threadIdx.x; t < (p.n + kWave - 1) / kWave * kWave; t += kPrepThreads) {
            const int64_t label = t < p.n ? label_of(p.labels, t * p.labels_stride, p.wide) : p.ignore;
            const bool is = t < p.n && label != p.ignore;
            all += __popcll(__ballot(is));
            before += __popcll(__ballot(is && t < first));
            outside += __popcll(__ballot(is && (label < 0 || label >= static_cast<int64_t>(p.vocab))));
        }
        if (lane == 0) {
            sums[wave][0] = before;
            sums[wave][1] = all;
            sums[wave][2] = outside;
        }
        __syncthreads();
        at = valid = outside = 0;
#pragma unroll
        for (uint32_t w = 0; w < kPrepWaves; ++w) {
            at += sums[w][0];
            valid += sums[w][1];
            outside += sums[w][2];
        }
        for (uint32_t t = first; t <= i && t < p.n; ++t) {
            const int64_t label = label_of(p.labels, t * p.labels_stride, p.wide);
            counted = label != p.ignore;
            if (t < i) {
                at += counted;
            } else if (lane == 0) {
                p.place[t] = counted ? static_cast<int32_t>(at) : -1;
                if (counted) {
                    p.rows[at] = static_cast<int32_t>(t);
                    p.compact[at] = label < 0 || label >= static_cast<int64_t>(p.vocab) ? -1 : static_cast<int32_t>(label);
                } else {
                    p.losses[t] = 0.0f;
                }
            }
        }
        counted = counted && i < p.n;
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            p.meta->valid = valid;
            p.meta->invalid = outside;
        }
    }
    int e = 0;
    if constexpr (kScaled) {
        const uint32_t sample = sample_of(p, true, most_lds);
        e = lift_of(sample);
        if (blockIdx.x == 0 && threadIdx.x == 0) p.meta->x_sample = sample;
    }
    Seen seen;
    if (counted)
        pack_row<T, RAW>(static_cast<const T*>(p.x) + i * p.x_stride, p.x_out + at * kParts * p.width, p.d, p.width, e, seen,
                         RAW ? p.x_split + static_cast<uint64_t>(at) * 3 * p.width : nullptr);
    if (i >= valid && i < (valid + 63) / 64 * 64) {
        uint4* out = reinterpret_cast<uint4*>(p.x_out + i * kParts * p.width);
        for (uint32_t c = lane; c < kParts * p.width / 8; c += kWave) out[c] = make_uint4(0, 0, 0, 0);
        if constexpr (RAW) clear_split(p, i);
    }
    if constexpr (kScaled) {
        const uint2 all = make_uint2(block_most(seen.most, most_lds), block_most(seen.small, most_lds));
        if (threadIdx.x == 0) p.x_most[blockIdx.x] = all;
    }
}

// float32: the powers of two that hold, from the blocks' largest magnitudes, and the operands packed again where the
// sample's did not. Where entries spread beyond kSpread, x's counted rows are packed as they are and as three parts instead
// (the weight is read in place then).
__global__ __launch_bounds__(kPrepThreads) void loss_settle_kernel(Prepare p) {
    __shared__ uint32_t lds[kPrepWaves];
    bool wide = false;
    const auto settled = [&](const uint2* blocks_seen, uint32_t blocks, uint32_t sample) -> uint32_t {
        Seen seen;
        for (uint32_t i = threadIdx.x; i < blocks; i += kPrepThreads) seen.join(blocks_seen[i]);
        const uint32_t largest = block_most(seen.most, lds), small = block_most(seen.small, lds);
        const uint32_t bits = largest == 0 || (sample != 0 && lift_of(largest) - lift_of(sample) <= kRoom) ? sample : largest;
        wide = wide || (small != 0 && lift_of(bits) - lift_of(~small) > kSpread);
        return bits;
    };
    const uint32_t x_sample = p.meta->x_sample, w_sample = p.meta->weight_sample, valid = p.meta->valid;
    const uint32_t x_bits = settled(p.x_most, p.x_blocks, x_sample), w_bits = settled(p.w_most, p.w_blocks, w_sample);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        p.meta->x_bits = x_bits;
        p.meta->weight_bits = w_bits;
        p.meta->wide = wide;
    }
    Seen again;
    if (wide || x_bits != x_sample)
        for (uint32_t i = blockIdx.x * kPrepWaves + threadIdx.x / kWave; i < (valid + 63) / 64 * 64; i += gridDim.x * kPrepWaves) {
            if (i >= valid) {  // x_out's rows are zeros already
                if (wide) clear_split(p, i);
                continue;
            }
            const float* from = static_cast<const float*>(p.x) + p.rows[i] * p.x_stride;
            uint16_t* to = p.x_out + static_cast<uint64_t>(i) * 2 * p.width;
            if (wide) pack_row<float, true>(from, to, p.d, p.width, 0, again, p.x_split + static_cast<uint64_t>(i) * 3 * p.width);
            else pack_row<float, false>(from, to, p.d, p.width, lift_of(x_bits), again);
        }
    if (!wide && w_bits != w_sample)
        for (uint32_t block = blockIdx.x; block < p.w_blocks; block += gridDim.x) pack_weight<float>(p, block, lift_of(w_bits), again);
}

// --------------------------------------------------------------------------------------------------------- the product

// Index permutation of the 32 rows of an MFMA operand: with it a lane's 16 results of a 32 x 32 tile are 16 consecutive
// indexes (16 (lane / 32) on) of the row operand.
__device__ __forceinline__ uint32_t permuted(uint32_t r) { return (r >> 2 & 1) * 16 + (r >> 3) * 4 + (r & 3); }

// An operand's tile in LDS, TILE indexes x 64 / PARTS k (128 bytes an index), 16-byte chunks swizzled so that the lanes of
// a read touch every bank: index-major (memory rows are the operand's indexes, k contiguous; a row's 8 chunks) or k-major
// (TR: memory rows are k, read through the LDS transpose reads). Transfers of 1 KB go straight from memory to LDS.
// Entries in memory: PARTS 1 bfloat16; PARTS 2 fp16 hi and lo; PARTS 3 float32 as they are, split into three bfloat16 parts
// by the wave that reads them (RAW; k-major tiles of these are read entry by entry). GRAIN: bytes a lane transfers at a time, 4 for
// rows of float32 that start on their own boundaries only.
template <int PARTS, bool TR, int TILE, int WAVES, uint32_t GRAIN = 16>
struct Operand {
    static constexpr bool RAW = PARTS == 3;
    static constexpr uint32_t kWords = PARTS == 1 ? 1 : 2;  // 16-bit words of an entry
    static constexpr uint32_t kBytes = TILE * 128, kPiece = GRAIN * kWave, kPieces = kBytes / kPiece, kPerWave = kPieces / WAVES;
    static constexpr uint32_t kRow = TR ? TILE * 2 * kWords : 128, kDepth = 64 / kWords;
    static_assert(kPieces % WAVES == 0, "every wave transfers as many pieces");
    static_assert(GRAIN == 16 || (GRAIN == 4 && RAW), "16-byte transfers, or single float32");
    static_assert(!TR || RAW || kRow >= 256, "the swizzle stays within a row");

    const char* base;        // of the tile at k = 0 (index-major) or of its first column (k-major)
    uint64_t stride;         // bytes of a memory row
    uint32_t offset[kPerWave];  // index-major: a lane's byte offset of each piece
    uint32_t back[kPerWave], whole;  // index-major: bytes back to the tile's first chunk where k-tile `whole`, the last, has no more
    uint32_t row[kPerWave], last;  // k-major: the lane's k row of each piece (offset: its column); the last k row to read

    __device__ __forceinline__ static uint32_t swizzle(uint32_t r) {
        if constexpr (TR && RAW) return 0;
        else if constexpr (TR) return (r & 1) * 4 + (r >> 1 & 1) * 9;
        else return ((r & 3) | (r >> 4 & 1) << 2) ^ (r >> 2 & 1);
    }
    // first: the tile's first index; indexes: memory rows (index-major) or columns, a multiple of 8 (k-major), there are; depth:
    // k there are. What lies beyond reads as something else: results that are dropped, or k where the other operand holds
    // zeros.
    __device__ __forceinline__ void begin(const uint16_t* p, uint64_t row_entries, uint32_t first, uint32_t indexes, uint32_t depth) {
        const uint32_t wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
        stride = row_entries * 2;
        last = depth - 1;
        whole = depth * kWords / 64;
        if (!TR && first >= indexes) first = indexes - 1;
        if constexpr (TR) base = reinterpret_cast<const char*>(p) + static_cast<uint64_t>(first) * 2 * kWords;
        else base = reinterpret_cast<const char*>(p) + first * stride;
#pragma unroll
        for (uint32_t j = 0; j < kPerWave; ++j) {
            const uint32_t at = (wave * kPerWave + j) * kPiece + lane * GRAIN, r = at / kRow, chunk = at % kRow / 16 ^ swizzle(r);
            if constexpr (TR) {
                const uint32_t byte = chunk * 16 + at % 16, end = (indexes - first) * kWords * 2;  // of the memory row
                row[j] = r;
                offset[j] = byte < end ? byte : end - GRAIN;
            } else {
                const uint32_t left = indexes - first - 1;  // clamped rows repeat the last
                const uint32_t byte = chunk * 16 + at % 16;
                offset[j] = (r < left ? r : left) * static_cast<uint32_t>(stride) + byte;
                back[j] = byte >= depth * kWords * 2 % 128 ? byte : 0;
            }
        }
    }
    __device__ __forceinline__ static void transfer(const char* from, uint32_t at, const char* lds) {
        if constexpr (GRAIN == 16) dma16(from, at, lds);
        else dma4(from, at, lds);
    }
    // the tile of k-tile kt into LDS, from `shift` bytes on
    __device__ __forceinline__ void fetch(uint32_t kt, const char* lds, uint64_t shift = 0) const {
        const uint32_t wave = uniform(threadIdx.x / kWave);
        if constexpr (TR) {
            const uint32_t k0 = kt * kDepth;
            const char* from = base + shift + k0 * stride;
#pragma unroll
            for (uint32_t j = 0; j < kPerWave; ++j) {
                const uint32_t r = k0 + row[j] <= last ? row[j] : last - k0;  // beyond: the other operand holds zeros
                transfer(from, r * static_cast<uint32_t>(stride) + offset[j], lds + (wave * kPerWave + j) * kPiece);
            }
        } else {
            const char* from = base + shift + kt * 128;
#pragma unroll
            for (uint32_t j = 0; j < kPerWave; ++j) transfer(from, kt == whole ? offset[j] - back[j] : offset[j], lds + (wave * kPerWave + j) * kPiece);
        }
    }
    // a lane's place in the tile for the 32-index blocks from `first` on
    __device__ __forceinline__ static uint32_t place(uint32_t first) {
        const uint32_t lane = threadIdx.x % kWave, half = lane / 32;
        if constexpr (TR && RAW) {
            return half * 8 * kRow + (first + permuted(lane % 32)) * 4;
        } else if constexpr (TR) {
            const uint32_t in = lane % 16, block = (lane / 16 & 1) * 4 + in % 4, k = in / 4;
            const uint32_t column = first * 2 * kWords + (block & 1) * 32 + (block >> 1) * 8;
            return (half * 8 + k) * kRow + (column ^ swizzle(k) * 16);
        } else {
            const uint32_t r = first + permuted(lane % 32);
            return r * 128 + ((RAW ? 2 * half : half) ^ swizzle(r)) * 16;
        }
    }
    // entries k = 16 step + 8 (lane / 32) + 0..7 of index permuted(lane % 32) of block i
    __device__ __forceinline__ static Frag read(uint32_t tile, uint32_t place, int i, int step, int part) {
        if constexpr (TR) {
            const uint32_t at = tile + (place ^ (i * 64 * kWords + part * 64)) + step * 16 * kRow;
            const Quad a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<LdsQuad>(at));
            const Quad b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<LdsQuad>(at + 4 * kRow));
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            return *reinterpret_cast<LdsFrag>(tile + i * 4096 + (place ^ (part * 64 + step * 32)));
        }
    }
    __device__ __forceinline__ static Eight read_raw(uint32_t tile, uint32_t place, int i, int step) {
        if constexpr (TR) {
            Eight v;
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = *reinterpret_cast<LdsFloat>(tile + place + i * 128 + (step * 16 + k) * kRow);
            return v;
        } else {
            const Four a = *reinterpret_cast<LdsFour>(tile + i * 4096 + (place ^ (step * 64)));
            const Four b = *reinterpret_cast<LdsFour>(tile + i * 4096 + (place ^ (step * 64 + 16)));
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

// float32 entries already split into three bfloat16 parts (memory: per 32 entries 3 x 32), index-major, in LDS as a plane of
// TILE x 64 bytes a part: x's rows for the weight's products, which every wave of a block reads (splitting them where they are
// read took four waves' time: losses of 64 tokens of 2048 x 50304 143 us, 123 so).
template <int TILE, int WAVES>
struct SplitOperand {
    static constexpr uint32_t kPlane = TILE * 64, kBytes = 3 * kPlane, kPieces = kBytes / 1024, kPerWave = kPieces / WAVES, kDepth = 32;
    static_assert(kPieces % WAVES == 0 && kPlane % 1024 == 0, "every wave transfers as many pieces, each of one plane");

    const char* base;
    uint32_t offset[kPerWave];

    __device__ __forceinline__ static uint32_t swizzle(uint32_t r) { return ((r >> 1 ^ r >> 2) & 1) | (r >> 4 & 1) << 1; }
    __device__ __forceinline__ void begin(const uint16_t* p, uint64_t row_entries, uint32_t first, uint32_t indexes, uint32_t) {
        const uint32_t wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, left = indexes - first - 1;
        base = reinterpret_cast<const char*>(p) + first * row_entries * 2;
#pragma unroll
        for (uint32_t j = 0; j < kPerWave; ++j) {
            const uint32_t at = (wave * kPerWave + j) * 1024 + lane * 16, part = at / kPlane, r = at % kPlane / 64, chunk = at % 64 / 16 ^ swizzle(r);
            offset[j] = min(r, left) * static_cast<uint32_t>(row_entries * 2) + part * 64 + chunk * 16;
        }
    }
    __device__ __forceinline__ void fetch(uint32_t kt, const char* lds) const {
        const uint32_t wave = uniform(threadIdx.x / kWave);
        const char* from = base + kt * 192;
#pragma unroll
        for (uint32_t j = 0; j < kPerWave; ++j) dma16(from, offset[j], lds + (wave * kPerWave + j) * 1024);
    }
    __device__ __forceinline__ static uint32_t place(uint32_t first) {
        const uint32_t lane = threadIdx.x % kWave, r = first + permuted(lane % 32);
        return r * 64 + (lane / 32 ^ swizzle(r)) * 16;
    }
    __device__ __forceinline__ static Frag read(uint32_t tile, uint32_t place, int i, int step, int part) {
        return *reinterpret_cast<LdsFrag>(tile + part * kPlane + i * 2048 + (place ^ (step * 32)));
    }
};

// The same entries as `count` MFMA operands: the parts as read, or three bfloat16 ones whose sum is the float32 to 2^-24.
template <int PARTS>
struct Parts {
    Frag part[PARTS];
    template <typename OP>
    __device__ __forceinline__ void read(uint32_t tile, uint32_t place, int i, int step) {
#pragma unroll
        for (int k = 0; k < PARTS; ++k) part[k] = OP::read(tile, place, i, step, k);
    }
    __device__ __forceinline__ const Parts& parts() const { return *this; }
};
struct Raw {
    Eight value;
    template <typename OP>
    __device__ __forceinline__ void read(uint32_t tile, uint32_t place, int i, int step) {
        value = OP::read_raw(tile, place, i, step);
    }
    __device__ __forceinline__ Parts<3> parts() const {
        uint32_t words[4][3];
#pragma unroll
        for (int k = 0; k < 4; ++k) split_pair(value[2 * k], value[2 * k + 1], words[k]);
        Parts<3> out;
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            const Words w{words[0][p], words[1][p], words[2][p], words[3][p]};
            out.part[p] = __builtin_bit_cast(Frag, w);
        }
        return out;
    }
};

template <int PARTS>
__device__ __forceinline__ Acc multiply(Frag a, Frag b, Acc c) {
    if constexpr (PARTS != 2) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(FragB, a), __builtin_bit_cast(FragB, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(FragH, a), __builtin_bit_cast(FragH, b), c, 0, 0, 0);
}

// float32 calls keep the exponential's last bits; bfloat16 ones round it to 8.
template <int PARTS>
__device__ __forceinline__ float exponential(float v) {
    if constexpr (PARTS != 1) return v < -150.0f ? 0.0f : exp_split(v);  // also -inf, of which exp_split makes a NaN
    else return __expf(v);
}

// Where a slice's maximum and sum of token t lie: a few tokens' slices token by token, which one block a token reads in whole
// lines (losses of 1 token 2.4 us of 31 or 57 less), many tokens' slice by slice.
template <bool FEW>
__device__ __forceinline__ uint64_t slice_at(uint32_t slice, uint32_t t, uint32_t pitch) {
    return FEW ? static_cast<uint64_t>(t) * pitch + slice : static_cast<uint64_t>(slice) * pitch + t;
}

// Stats: slices' maxima and sums; Keep: those, and the exponentials kept where D belongs; Grad: D.
enum class Use { Stats, Keep, Grad, GradX, GradW };

// float32 calls of many tokens: whether a launch is for entries that lie near enough for one power of two a tensor, or for others.
enum class Spread : uint8_t { Any, Near, Wide };
__device__ __forceinline__ bool skipped(Spread only, const Meta& meta) { return only != Spread::Any && (only == Spread::Wide) != (meta.wide != 0); }

// One product of a loss call: which operands, how far they go, and what becomes of the results.
struct Product {
    const uint16_t *a, *b;
    uint64_t a_stride, b_stride;  // 16-bit entries from one memory row to the next
    uint32_t a_columns, b_columns;  // entries of a memory row: the weight's d in place, padded widths else
    uint32_t a_first;             // first vocabulary row of the piece
    uint32_t a_count, b_count;    // GradX, GradW: columns of the output; GradW: its rows
    uint32_t vocab;
    uint32_t k_tiles;             // all (GradX: of the piece)
    uint32_t a_tiles, b_tiles, splits;
    uint32_t height, a_columns_out;  // vocabulary rows of a tile (Stats, Keep, Grad; kA at most), columns of D to write
    const Meta* meta;
    const int32_t* labels;        // compact
    const float* lse;             // Grad, compact
    float* picked;                // Stats, Keep: the label's logit, compact
    float2* slices;               // Stats, Keep: a slice's maximum and sum of exponentials per token
    uint32_t slice_pitch;         // slices of many tokens [slice][n_pad]; of a few [n_pad][slice]: n_pad, or the slices there are
    uint32_t slice_first;         // the piece's first
    uint16_t* grad;               // Grad: D, [n_pad][piece]; Keep: the exponentials
    uint64_t grad_stride, grad_low;  // LOW: 16-bit entries from D's first part to its second
    uint32_t n_pad;
    float* partial;               // GradX: [split][n_pad][d]
    bool add;
    void* out;                    // GradW: [V, d]
    uint64_t out_stride;
    float scale;
    bool mean, out_bf16;
    Spread only;                  // the calls that this launch does the work of
};

// WA x WB waves of TA x TB 32 x 32 results each; k-tiles go through a ring of kStages tile pairs. LOW: bfloat16 calls that hold D as
// two bfloat16 parts, its rounding and what that left, a plane each; its products multiply the other operand by both.
template <int PARTS_, Use USE_, int WA_, int WB_, int TA_, int TB_, uint32_t GRAIN = 16, bool LOW_ = false>
struct Shape {
    static constexpr int PARTS = PARTS_, WA = WA_, WB = WB_, TA = TA_, TB = TB_;
    static constexpr Use USE = USE_;
    static constexpr bool LOW = LOW_, kLowB = LOW && (USE == Use::GradX || USE == Use::GradW);
    static_assert(!LOW || PARTS == 1, "other parts hold D to more bits by themselves");
    static constexpr bool kATr = USE == Use::GradX || USE == Use::GradW, kBTr = USE == Use::GradW;
    static constexpr int kA = WA * TA * 32, kB = WB * TB * 32, kWaves = WA * WB;
    using OpA = Operand<PARTS, kATr, kA, kWaves, GRAIN>;
    // float32 as it is: x's rows come split, D's do not
    static constexpr bool kBSplit = PARTS == 3 && USE != Use::GradX && USE != Use::GradW;
    using OpB = typename std::conditional<kBSplit, SplitOperand<kB, kWaves>, Operand<PARTS, kBTr, kB, kWaves>>::type;
    static constexpr uint32_t kPlanes = kLowB ? 2 : 1, kStage = OpA::kBytes + kPlanes * OpB::kBytes;
    static constexpr uint32_t kTransfers = OpA::kPerWave + kPlanes * OpB::kPerWave;
    static constexpr int kStages = kWaves == 4 ? 81920 / kStage : 163840 / kStage < 4 ? 163840 / kStage : 4;  // 4 waves: two blocks a CU
    static constexpr uint32_t kLds = kStage * kStages;
    static_assert(kStages >= 1, "a stage at least");
};

// Tiles in groups of kGroup inner ones, a group's outer tiles one after the other: the 32 blocks that an XCD runs at a time
// share kGroup inner and 4 outer tiles, 12 tiles' transfers through its L2 where rows of 32 inner ones would take 33
// (8192 tokens of 2048 x 50304: the forward's product 1510 -> 1460 us).
constexpr uint32_t kGroup = 8;
struct TilePlace {
    uint32_t inner, outer;
};
__device__ __forceinline__ TilePlace tile_place(uint32_t block, uint32_t inner, uint32_t outer) {
    const uint32_t group = block / (kGroup * outer), rest = block % (kGroup * outer), left = inner - group * kGroup;
    const uint32_t width = left < kGroup ? left : kGroup;
    return {group * kGroup + rest % width, rest / width};
}

// Where a tile's results lie: a0 <= indexes of A < a_end, a_tile its whole tile along A.
struct TileAt {
    uint32_t a0, b0, split, a_tile, a_end;
};

// One tile: where it lies, its operands and its k-tiles.
template <typename S>
struct Tile {
    TileAt at;
    uint32_t k_begin, k_end;
    typename S::OpA a;
    typename S::OpB b;
    uint64_t low;  // bytes from D's first part to its second

    // part `part` (of tiles WHOLE::kA x WHOLE::kB cut into tiles of this shape) of tile `index` of the live_b token tiles;
    // false where it has no results
    template <typename WHOLE>
    __device__ __forceinline__ bool begin(const Product& p, uint32_t valid, uint32_t live_b, uint32_t index, uint32_t part) {
        constexpr Use USE = S::USE;
        constexpr bool kTokensFirst = USE == Use::Stats || USE == Use::Keep || USE == Use::Grad;
        const uint32_t per_split = p.a_tiles * live_b;
        at.split = index / per_split;
        const TilePlace tile = tile_place(index % per_split, kTokensFirst ? live_b : p.a_tiles, kTokensFirst ? p.a_tiles : live_b);
        constexpr uint32_t kPartsA = WHOLE::kA / S::kA;
        at.a_tile = kTokensFirst ? tile.outer : tile.inner;
        at.a0 = at.a_tile * (kTokensFirst ? p.height : WHOLE::kA) + part % kPartsA * S::kA;
        at.a_end = kTokensFirst ? min((at.a_tile + 1) * p.height, p.a_columns_out) : p.a_count;
        at.b0 = (kTokensFirst ? tile.inner : tile.outer) * WHOLE::kB + part / kPartsA * S::kB;
        k_begin = 0;
        k_end = p.k_tiles;
        if constexpr (S::kLowB) low = p.grad_low * 2;
        if constexpr (kTokensFirst) {
            if (at.b0 >= valid) return false;
            a.begin(p.a, p.a_stride, p.a_first + at.a0, min(p.vocab, p.a_first + at.a_end), p.a_columns);
            b.begin(p.b, p.b_stride, at.b0, p.n_pad, p.b_columns);
        } else if constexpr (USE == Use::GradX) {
            if (at.b0 >= valid || at.a0 >= p.a_columns) return false;
            k_begin = static_cast<uint64_t>(p.k_tiles) * at.split / p.splits;
            k_end = static_cast<uint64_t>(p.k_tiles) * (at.split + 1) / p.splits;
            a.begin(p.a, p.a_stride, at.a0, p.a_columns, p.vocab - p.a_first);
            b.begin(p.b, p.b_stride, at.b0, p.n_pad, p.b_columns);
        } else {
            if (at.b0 >= p.b_count || at.a0 >= p.a_count) return false;
            k_end = (valid + S::OpA::kDepth - 1) / S::OpA::kDepth;
            a.begin(p.a, p.a_stride, at.a0, p.a_columns, p.n_pad);
            b.begin(p.b, p.b_stride, at.b0, p.b_columns, p.n_pad);
        }
        return true;
    }
    __device__ __forceinline__ void fetch(uint32_t kt, const char* ring) const {
        const char* stage = ring + (kt - k_begin) % S::kStages * S::kStage;
        a.fetch(kt, stage);
        b.fetch(kt, stage + S::OpA::kBytes);
        if constexpr (S::kLowB) b.fetch(kt, stage + S::OpA::kBytes + S::OpB::kBytes, low);
    }
    __device__ __forceinline__ void ahead(const char* ring) const {  // the first k-tiles
        for (uint32_t kt = k_begin; kt < k_end && kt < k_begin + S::kStages; ++kt) fetch(kt, ring);
    }
};

// Every wave's LDS reads so far and, of its transfers, all but the last `kLater` are done.
template <int kLater>
__device__ __forceinline__ void meet() {
    wait_loads<kLater>();
    asm volatile("" ::: "memory");  // LDS reads stay on their side
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// The sums of a tile whose first k-tiles are under way. Operands of a step (16 k) are read from LDS while the step before it
// multiplies; the last step of a k-tile reads the first of the next, behind the barrier that says every wave's transfers
// of it have landed and every wave has read the last of the k-tile before it, whose stage the transfers of k-tile
// kt + kStages then take. float32: sums of kChain2 or kChain3 k-tiles in the MFMA accumulators (whose own sums round downwards), added to
// others.
template <typename S>
__device__ __forceinline__ void accumulate(const Tile<S>& tile, const char* ring, Acc (&sums)[S::TA][S::TB]) {
    constexpr int PARTS = S::PARTS, TA = S::TA, TB = S::TB, kSteps = PARTS == 1 ? 4 : 2, kTransfers = static_cast<int>(S::kTransfers);
    constexpr uint32_t kChain = PARTS == 3 ? kChain3 : kChain2;
    static_assert(kSteps % 2 == 0, "a k-tile's first step always reads into the same registers");
    const uint32_t wave = threadIdx.x / kWave, lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(ring));
    const uint32_t a_place = S::OpA::place(wave % S::WA * TA * 32), b_place = S::OpB::place(wave / S::WA * TB * 32);
    const uint32_t k_begin = tile.k_begin, k_end = tile.k_end;
#pragma unroll
    for (int i = 0; i < TA; ++i)
#pragma unroll
        for (int j = 0; j < TB; ++j) sums[i][j] = 0.0f;
    if (k_begin >= k_end) return;
    Acc chain[PARTS != 1 ? TA : 1][PARTS != 1 ? TB : 1];
    if constexpr (PARTS != 1) {
#pragma unroll
        for (int i = 0; i < TA; ++i)
#pragma unroll
            for (int j = 0; j < TB; ++j) chain[i][j] = 0.0f;
    }
    const auto acc = [&](int i, int j) -> Acc& {
        if constexpr (PARTS != 1) return chain[i][j];
        else return sums[i][j];
    };
    typename std::conditional<PARTS == 3, Raw, Parts<PARTS>>::type fa[2][TA];
    typename std::conditional<PARTS == 3 && !S::kBSplit, Raw, Parts<PARTS>>::type fb[2][TB];
    Parts<PARTS> fb_low[2][S::kLowB ? TB : 1];
    const auto read = [&](uint32_t kt, int step, int to) {
        const uint32_t tile_a = lds + (kt - k_begin) % S::kStages * S::kStage, tile_b = tile_a + S::OpA::kBytes;
#pragma unroll
        for (int i = 0; i < TA; ++i) fa[to][i].template read<typename S::OpA>(tile_a, a_place, i, step);
#pragma unroll
        for (int j = 0; j < TB; ++j) {
            fb[to][j].template read<typename S::OpB>(tile_b, b_place, j, step);
            if constexpr (S::kLowB) fb_low[to][j].template read<typename S::OpB>(tile_b + S::OpB::kBytes, b_place, j, step);
        }
    };
    if (k_end - k_begin >= static_cast<uint32_t>(S::kStages)) meet<kTransfers * (S::kStages - 1)>();
    else meet<0>();
    read(k_begin, 0, 0);
    for (uint32_t kt = k_begin; kt < k_end; ++kt) {
#pragma unroll
        for (int step = 0; step < kSteps; ++step) {
            const int now = step % 2;
            if (step + 1 < kSteps) {
                read(kt, step + 1, 1 - now);
            } else if (kt + 1 < k_end) {
                constexpr int kLater = S::kStages > 1 ? kTransfers * (S::kStages - 2) : 0;
                if (k_end - kt >= static_cast<uint32_t>(S::kStages)) meet<kLater>();
                else meet<0>();
                if (kt + S::kStages < k_end) tile.fetch(kt + S::kStages, ring);
                if constexpr (S::kStages == 1) meet<0>();  // the only stage: its transfers have only begun
                read(kt + 1, 0, 1 - now);
            }
            Parts<PARTS> a[TA], b[TB];
#pragma unroll
            for (int i = 0; i < TA; ++i) a[i] = fa[now][i].parts();
#pragma unroll
            for (int j = 0; j < TB; ++j) b[j] = fb[now][j].parts();
#pragma unroll
            for (int i = 0; i < TA; ++i)
#pragma unroll
                for (int j = 0; j < TB; ++j) {
                    if constexpr (S::kLowB) acc(i, j) = multiply<PARTS>(a[i].part[0], fb_low[now][j].part[0], acc(i, j));
#pragma unroll
                    for (int q = 0; q < PARTS; ++q) {  // the parts' products down to the last part's weight; three parts: the least first
                        const int sum = PARTS == 3 ? PARTS - 1 - q : q;
#pragma unroll
                        for (int k = 0; k <= sum; ++k) acc(i, j) = multiply<PARTS>(a[i].part[k], b[j].part[sum - k], acc(i, j));
                    }
                }
        }
        if constexpr (PARTS != 1) {
            if ((kt - k_begin) % kChain == kChain - 1 || kt + 1 == k_end) {
#pragma unroll
                for (int i = 0; i < TA; ++i)
#pragma unroll
                    for (int j = 0; j < TB; ++j) {
                        sums[i][j] += chain[i][j];
                        chain[i][j] = 0.0f;
                    }
            }
        }
    }
}

// What becomes of a tile's sums. A lane's: index b0 + (wb TB + j) 32 + permuted(lane % 32) of B, indexes
// a0 + (wa TA + i) 32 + 16 (lane / 32) + 0..15 of A. SLICES: the forward's slices of a whole tile, of which a wave of a
// whole tile fills several (one with its sums, the others empty).
template <typename S, uint32_t SLICES, int WHOLE_A>
__device__ __forceinline__ void finish(const Product& p, const Meta& meta, const TileAt& tile, Acc (&sums)[S::TA][S::TB]) {
    constexpr int PARTS = S::PARTS, WA = S::WA, TA = S::TA, TB = S::TB;
    constexpr Use USE = S::USE;
    const uint32_t wave = threadIdx.x / kWave, wa = wave % WA, wb = wave / WA, lane = threadIdx.x % kWave, half = lane / 32;
    const uint32_t a0 = tile.a0, b0 = tile.b0, split_at = tile.split, a_end = tile.a_end, a_lane = a0 + wa * TA * 32 + 16 * half;
    float power = 1.0f;
    if constexpr (PARTS == 2) {
        const int ew = lift_of(meta.weight_bits), ex = lift_of(meta.x_bits);
        power = ldexpf(1.0f, USE == Use::GradX ? ew - kGradLift : USE == Use::GradW ? ex - kGradLift : 0);
        if constexpr (USE == Use::Stats || USE == Use::Keep || USE == Use::Grad) {
#pragma unroll
            for (int i = 0; i < TA; ++i)
#pragma unroll
                for (int j = 0; j < TB; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r) sums[i][j][r] = ldexpf(sums[i][j][r], ew + ex);
        }
    }
    const auto result = [&](int i, int j, int r) -> float { return sums[i][j][r]; };
    // 16 consecutive entries of a lane into row t of D, from its block i on: 16-bit ones (PARTS 2: hi and lo; LOW: the two planes'),
    // or the bits of 16 float32 (PARTS 3: eight and eight)
    const auto store = [&](uint32_t t, int i, const uint32_t (&hi)[8], const uint32_t (&lo)[8]) {
        if (a_lane + i * 32 >= a_end) return;
        uint16_t* to = p.grad + t * p.grad_stride + (a_lane - 16 * half + i * 32) * (PARTS == 1 ? 1 : 2) + (PARTS == 3 ? 32 : 16) * half;
        *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(to + 8) = make_uint4(hi[4], hi[5], hi[6], hi[7]);
        if constexpr (PARTS != 1 || S::LOW) {
            uint16_t* const low = to + (S::LOW ? p.grad_low : PARTS == 3 ? 16 : 32);
            *reinterpret_cast<uint4*>(low) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            *reinterpret_cast<uint4*>(low + 8) = make_uint4(lo[4], lo[5], lo[6], lo[7]);
        }
    };
    if constexpr (USE == Use::Stats || USE == Use::Keep) {
        constexpr uint32_t kFill = SLICES * S::kA / (WHOLE_A * WA);  // slices a wave fills
        const uint32_t slice = p.slice_first + tile.a_tile * SLICES + ((a0 - tile.a_tile * p.height) / (WA * TA * 32) * WA + wa) * kFill;
        const uint32_t first = p.a_first + a_lane, end = min(p.vocab, p.a_first + a_end);  // vocabulary rows: the lane's first, the tile's end
        if (p.a_first + a0 + S::kA > end) {  // what lies beyond adds nothing
#pragma unroll
            for (int i = 0; i < TA; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (first + i * 32 + r >= end)
#pragma unroll
                        for (int j = 0; j < S::TB; ++j) sums[i][j][r] = -__builtin_huge_valf();
        }
#pragma unroll
        for (int j = 0; j < S::TB; ++j) {
            const uint32_t t = b0 + (wb * S::TB + j) * 32 + permuted(lane % 32);
            float most = -__builtin_huge_valf();
#pragma unroll
            for (int i = 0; i < TA; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) most = fmaxf(most, result(i, j, r));
            most = fmaxf(most, __shfl_xor(most, 32));
            const float shift = most == -__builtin_huge_valf() ? 0.0f : most;
            float sum = 0.0f;
            const uint32_t label = t < meta.valid ? static_cast<uint32_t>(p.labels[t]) - first : 0xffffffffu;  // outside: far from every lane
            if (label < TA * 32 && (label & 16) == 0 && first + label < end) {
                float logit = 0.0f;
#pragma unroll
                for (int i = 0; i < TA; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) logit = label == static_cast<uint32_t>(i * 32 + r) ? result(i, j, r) : logit;
                p.picked[t] = logit;
            }
#pragma unroll
            for (int i = 0; i < TA; ++i) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    const float e[2] = {exponential<PARTS>(result(i, j, r) - shift), exponential<PARTS>(result(i, j, r + 1) - shift)};
                    sum += e[0];
                    sum += e[1];
                    if constexpr (USE == Use::Keep && PARTS == 1) {
                        hi[r / 2] = kept_bits(e[0]) | kept_bits(e[1]) << 16;
                    } else if constexpr (USE == Use::Keep && PARTS == 3) {
                        uint32_t* const to = r < 8 ? hi : lo;
                        to[r % 8] = __float_as_uint(e[0]);
                        to[r % 8 + 1] = __float_as_uint(e[1]);
                    } else if constexpr (USE == Use::Keep) {
                        uint16_t h[2], l[2];
                        split(e[0] * (1 << kGradLift), h[0], l[0]);
                        split(e[1] * (1 << kGradLift), h[1], l[1]);
                        hi[r / 2] = h[0] | static_cast<uint32_t>(h[1]) << 16;
                        lo[r / 2] = l[0] | static_cast<uint32_t>(l[1]) << 16;
                    }
                }
                if constexpr (USE == Use::Keep)
                    if (t < meta.valid) store(t, i, hi, lo);
            }
            sum += __shfl_xor(sum, 32);
            if (t >= meta.valid || half != 0) continue;
#pragma unroll
            for (uint32_t k = 0; k < kFill; ++k) p.slices[slice_at<S::kWaves == 4>(slice + k, t, p.slice_pitch)] = make_float2(most, k == 0 ? sum : 0.0f);
        }
    } else if constexpr (USE == Use::Grad) {
#pragma unroll
        for (int j = 0; j < TB; ++j) {
            const uint32_t t = b0 + (wb * TB + j) * 32 + permuted(lane % 32);
            const bool live = t < meta.valid;
            const float lse = live ? p.lse[t] : 0.0f;  // not counted: zeros below
            const uint32_t label = live ? static_cast<uint32_t>(p.labels[t]) - p.a_first - a_lane : 0xffffffffu;  // from the lane's first
            const bool whole = p.a_first + a0 + S::kA <= p.vocab;
#pragma unroll
            for (int i = 0; i < TA; ++i) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    float v[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        v[k] = exponential<PARTS>(result(i, j, r + k) - lse) - (label == static_cast<uint32_t>(i * 32 + r + k) ? 1.0f : 0.0f);
                        if (!live || (!whole && p.a_first + a_lane + i * 32 + r + k >= p.vocab)) v[k] = 0.0f;
                    }
                    if constexpr (PARTS == 1) {
                        hi[r / 2] = bf16_pair(v[0], v[1]);
                        if constexpr (S::LOW) lo[r / 2] = bf16_pair(v[0] - __uint_as_float(hi[r / 2] << 16), v[1] - __uint_as_float(hi[r / 2] & 0xffff0000u));
                    } else if constexpr (PARTS == 3) {
                        uint32_t* const to = r < 8 ? hi : lo;
                        to[r % 8] = __float_as_uint(v[0]);
                        to[r % 8 + 1] = __float_as_uint(v[1]);
                    } else {
                        uint16_t h[2], l[2];
                        split(v[0] * (1 << kGradLift), h[0], l[0]);
                        split(v[1] * (1 << kGradLift), h[1], l[1]);
                        hi[r / 2] = h[0] | static_cast<uint32_t>(h[1]) << 16;
                        lo[r / 2] = l[0] | static_cast<uint32_t>(l[1]) << 16;
                    }
                }
                store(t, i, hi, lo);
            }
        }
    } else {
        const float factor = USE == Use::GradW ? power * grad_factor(meta, p.scale, p.mean) : power;
        const uint32_t rows = USE == Use::GradX ? meta.valid : p.b_count;
#pragma unroll
        for (int j = 0; j < TB; ++j) {
            const uint32_t at_b = b0 + (wb * TB + j) * 32 + permuted(lane % 32);
            if (at_b >= rows) continue;
#pragma unroll
            for (int i = 0; i < TA; ++i) {
                const uint32_t at_a = a_lane + i * 32;
                if constexpr (USE == Use::GradX) {
                    float* to = p.partial + (static_cast<uint64_t>(split_at) * p.n_pad + at_b) * p.out_stride + at_a;
#pragma unroll
                    for (int r = 0; r < 16; r += 4) {
                        if (at_a + r >= p.a_count) continue;  // a_count, the padded width, is a multiple of 4
                        float4 v = make_float4(result(i, j, r), result(i, j, r + 1), result(i, j, r + 2), result(i, j, r + 3));
                        v = make_float4(v.x * factor, v.y * factor, v.z * factor, v.w * factor);
                        if (p.add) {
                            const float4 w = *reinterpret_cast<const float4*>(to + r);
                            v = make_float4(w.x + v.x, w.y + v.y, w.z + v.z, w.w + v.w);
                        }
                        *reinterpret_cast<float4*>(to + r) = v;
                    }
                } else {
                    const uint64_t to = at_b * p.out_stride + at_a;
                    float v[16];
#pragma unroll
                    for (int r = 0; r < 16; ++r) v[r] = factor * result(i, j, r);
                    if (at_a + 16 <= p.a_count && p.out_bf16) {
#pragma unroll
                        for (int r = 0; r < 16; r += 8)
                            *reinterpret_cast<WordsAnywhere*>(static_cast<uint16_t*>(p.out) + to + r) =
                                WordsAnywhere{bf16_pair(v[r], v[r + 1]), bf16_pair(v[r + 2], v[r + 3]), bf16_pair(v[r + 4], v[r + 5]), bf16_pair(v[r + 6], v[r + 7])};
                    } else if (at_a + 16 <= p.a_count) {
#pragma unroll
                        for (int r = 0; r < 16; r += 4)
                            *reinterpret_cast<FourAnywhere*>(static_cast<float*>(p.out) + to + r) = FourAnywhere{v[r], v[r + 1], v[r + 2], v[r + 3]};
                    } else {
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            if (at_a + r >= p.a_count) continue;
                            if (p.out_bf16) static_cast<uint16_t*>(p.out)[to + r] = bf16_bits(v[r]);
                            else static_cast<float*>(p.out)[to + r] = v[r];
                        }
                    }
                }
            }
        }
    }
}

// Part `part` of tile `index`, alone.
template <typename S, typename WHOLE, uint32_t SLICES>
__device__ __forceinline__ void take_part(const Product& p, const Meta& meta, uint32_t live_b, uint32_t index, uint32_t part, const char* ring) {
    Tile<S> tile;
    if (!tile.template begin<WHOLE>(p, meta.valid, live_b, index, part)) return;
    tile.ahead(ring);
    Acc sums[S::TA][S::TB];
    accumulate<S>(tile, ring, sums);
    finish<S, SLICES, WHOLE::kA>(p, meta, tile.at, sums);
}

// A launch's blocks stay: block b, on XCD b % 8, takes every (blocks / 8)-th tile of the XCD's share and requests a tile's
// first k-tiles before it finishes the tile before. Tiles that would leave most CUs idle in a last round are cut into halves
// or quarters, one a block (1 / 2 or 1 / 4 of the whole shape): 788 tiles of 256 blocks take 3.25 rounds, not 4. bfloat16 tiles
// are of 8 waves of 128 x 64 results (4 of 128 x 128: the forward's product of 8192 tokens of 2048 1540 -> 1780 us).
constexpr int kXcds = 8;
template <int PARTS, Use USE, int WA, int WB, int TA, int TB, uint32_t GRAIN, bool LOW>
__global__ __launch_bounds__(WA* WB* kWave) __attribute__((amdgpu_waves_per_eu(2, 2))) void loss_product_kernel(Product p) {
    constexpr bool kCut = TA % 2 == 0 && TB % 2 == 0;
    using Whole = Shape<PARTS, USE, WA, WB, TA, TB, GRAIN, LOW>;
    using Half = Shape<PARTS, USE, WA, WB, TA, kCut ? TB / 2 : TB, GRAIN, LOW>;
    using Quarter = Shape<PARTS, USE, WA, WB, kCut ? TA / 2 : TA, kCut ? TB / 2 : TB, GRAIN, LOW>;
    constexpr uint32_t kSlices = kCut ? 2 * WA : WA;
    constexpr uint32_t kLds = Whole::kLds > Quarter::kLds ? (Whole::kLds > Half::kLds ? Whole::kLds : Half::kLds)
                                                          : (Quarter::kLds > Half::kLds ? Quarter::kLds : Half::kLds);
    __shared__ __attribute__((aligned(1024))) char ring[kLds];
    const Meta meta = *p.meta;
    if (PARTS != 1 && skipped(p.only, meta)) return;
    const uint32_t live_b = USE == Use::GradW ? p.b_tiles : (meta.valid + Whole::kB - 1) / Whole::kB;
    const uint64_t tiles = static_cast<uint64_t>(p.a_tiles) * live_b * p.splits;
    const uint32_t xcd = blockIdx.x % kXcds, local = blockIdx.x / kXcds, blocks = gridDim.x / kXcds;
    const uint32_t first = static_cast<uint32_t>(tiles * xcd / kXcds), share = static_cast<uint32_t>(tiles * (xcd + 1) / kXcds) - first;
    const uint32_t rest = share % blocks, pieces = !kCut || rest == 0 || 2 * rest > blocks ? 1 : 4 * rest > blocks ? 2 : 4;
    const uint32_t whole = pieces == 1 ? share : share - rest;
    {
        Tile<Whole> tile;
        uint32_t index = local;
        bool live = false;
        const auto next = [&]() {  // the block's next tile that has results
            for (live = false; index < whole && !live; index += blocks) live = tile.template begin<Whole>(p, meta.valid, live_b, first + index, 0);
            if (live) tile.ahead(ring);
        };
        next();
        Acc sums[TA][TB];
        while (live) {
            accumulate<Whole>(tile, ring, sums);
            const TileAt at = tile.at;
            meet<0>();  // every wave has read its last
            next();
            finish<Whole, kSlices, Whole::kA>(p, meta, at, sums);
        }
    }
    if constexpr (kCut) {
        if (pieces == 1 || local >= pieces * rest) return;
        const uint32_t index = first + whole + local / pieces, part = local % pieces;
        if (pieces == 2) take_part<Half, Whole, kSlices>(p, meta, live_b, index, part, ring);
        else take_part<Quarter, Whole, kSlices>(p, meta, live_b, index, part, ring);
    }
}

// ------------------------------------------------------------------------------------------- the sums over the vocabulary

// Where a product left its slices: how many there are, and the pitch of slice_at.
struct Slices {
    const float2* at;
    uint32_t count, pitch;
};

// lse and loss of every counted token from the slices: TOKENS tokens a block, 1024 / TOKENS threads each over the slices. `wide`:
// the slices, token by token, of calls whose entries spread (null: there are no such calls).
constexpr uint32_t kLseThreads = 1024, kLseWaves = kLseThreads / kWave;
__device__ __forceinline__ float2 joined(float2 a, float2 b) {
    const float most = fmaxf(a.x, b.x);
    if (most == -__builtin_huge_valf()) return make_float2(most, a.y + b.y);
    return make_float2(most, a.y * exponential<2>(a.x - most) + b.y * exponential<2>(b.x - most));
}
template <uint32_t TOKENS>
__device__ __forceinline__ float2 joined_lanes(float2 v) {  // over the lanes of a wave that share a token
#pragma unroll
    for (uint32_t step = TOKENS; step < kWave; step *= 2) v = joined(v, make_float2(__shfl_xor(v.x, step), __shfl_xor(v.y, step)));
    return v;
}
template <uint32_t TOKENS>
__global__ __launch_bounds__(kLseThreads) void loss_lse_kernel(Slices near, Slices wide, const float* __restrict__ picked, const int32_t* __restrict__ rows,
                                                              const int32_t* __restrict__ labels, const Meta* __restrict__ meta,
                                                              float* __restrict__ lse, float* __restrict__ losses) {
    const bool by_token = wide.at != nullptr && meta->wide != 0;
    constexpr uint32_t kLanes = kLseThreads / TOKENS;
    __shared__ float2 lds[kLseWaves * TOKENS];
    const uint32_t in = threadIdx.x % TOKENS, t = blockIdx.x * TOKENS + in, valid = meta->valid, lane = threadIdx.x % kWave;
    if (blockIdx.x * TOKENS >= valid) return;
    float2 all = make_float2(-__builtin_huge_valf(), 0.0f);
    if (t < valid && by_token) {
        for (uint32_t s = threadIdx.x / TOKENS; s < wide.count; s += kLanes) all = joined(all, wide.at[slice_at<true>(s, t, wide.pitch)]);
    } else if (t < valid) {
#pragma unroll 4
        for (uint32_t s = threadIdx.x / TOKENS; s < near.count; s += kLanes) all = joined(all, near.at[slice_at<TOKENS == 1>(s, t, near.pitch)]);
    }
    all = joined_lanes<TOKENS>(all);
    if (lane < TOKENS) lds[threadIdx.x / kWave * TOKENS + in] = all;
    __syncthreads();
    if (threadIdx.x >= kWave) return;
    all = make_float2(-__builtin_huge_valf(), 0.0f);
#pragma unroll
    for (uint32_t k = 0; k < kLseWaves * TOKENS; k += kWave)
        if (k + lane < kLseWaves * TOKENS) all = joined(all, lds[k + lane]);  // a multiple of TOKENS apart: the lane's token
    all = joined_lanes<TOKENS>(all);
    if (lane >= TOKENS || t >= valid) return;
    const float value = all.x + logf(all.y);
    lse[t] = value;
    losses[rows[t]] = labels[t] < 0 ? __uint_as_float(0x7fc00000u) : value - picked[t];
}

// The kept exponentials of a piece, taken against their slice's maximum m, turned into D in place: e exp(m - lse) - onehot;
// zero rows from the counted tokens to the next multiple of 64. bfloat16 calls keep them to 2^-10 (kept_bits; D is then rounded
// to 2^-8), float32 ones as hi + lo. A block per row and kTurnThreads groups of 8 entries. For a piece that fits, this and the
// stores take less than its logits again: 2048 tokens of 1024 x 50304 bfloat16 75 + 25 against 283 us, 512 float32 40 + 5
// against 222 us.
constexpr uint32_t kTurnThreads = 256;
// What the product that kept them was: its slices (of the piece's first on), vocabulary rows of a tile, slices of a tile and
// rows of a slice.
struct Kept {
    const float2* slices;
    uint32_t height, per_tile, slice_rows, pitch;
};
template <int PARTS>
__device__ __forceinline__ void turn(uint16_t* __restrict__ grad, uint64_t stride, uint32_t first, uint32_t count, uint32_t across, const Kept& kept_by,
                                     const float* __restrict__ lse, const int32_t* __restrict__ labels, const Meta* __restrict__ meta) {
    const uint32_t t = blockIdx.x / across, valid = meta->valid, c = (blockIdx.x % across * kTurnThreads + threadIdx.x) * 8;
    if (t >= (valid + 63) / 64 * 64 || c >= count) return;
    uint4* const at = reinterpret_cast<uint4*>(grad + t * stride + (PARTS == 1 ? c : PARTS == 2 ? c / 32 * 64 + c % 32 : 2 * c));
    uint4* const low = at + (PARTS == 2 ? 4 : 1);  // PARTS 2: the lo halves, 3: the last four
    if (t >= valid) {
        *at = make_uint4(0, 0, 0, 0);
        if constexpr (PARTS != 1) *low = make_uint4(0, 0, 0, 0);
        return;
    }
    const uint32_t slice = c / kept_by.height * kept_by.per_tile + c % kept_by.height / kept_by.slice_rows;
    const float most = kept_by.slices[slice_at<PARTS == 3>(slice, t, kept_by.pitch)].x;
    const float factor = exponential<2>(most - lse[t]) * (PARTS == 2 ? 1.0f / (1 << kGradLift) : 1.0f);
    const uint32_t label = static_cast<uint32_t>(labels[t]) - first - c;
    const uint4 kept = *at, rest = PARTS != 1 ? *low : make_uint4(0, 0, 0, 0);
    const uint32_t hi[4] = {kept.x, kept.y, kept.z, kept.w}, lo[4] = {rest.x, rest.y, rest.z, rest.w};
    float v[8];
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k) {
        const uint32_t shift = 16 * (k % 2);
        float e;
        if constexpr (PARTS == 1) e = kept_value(hi[k / 2] >> shift);
        else if constexpr (PARTS == 2) e = half_value(hi[k / 2] >> shift) + half_value(lo[k / 2] >> shift);
        else e = __uint_as_float(k < 4 ? hi[k] : lo[k - 4]);
        v[k] = e * factor - (label == k ? 1.0f : 0.0f);
    }
    if constexpr (PARTS == 1) {
        *at = make_uint4(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7]));
    } else if constexpr (PARTS == 3) {
        *reinterpret_cast<float4*>(at) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(low) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t h[4], l[4];
#pragma unroll
        for (uint32_t k = 0; k < 8; k += 2) {
            uint16_t a[2], b[2];
            split(v[k] * (1 << kGradLift), a[0], b[0]);
            split(v[k + 1] * (1 << kGradLift), a[1], b[1]);
            h[k / 2] = a[0] | static_cast<uint32_t>(a[1]) << 16;
            l[k / 2] = b[0] | static_cast<uint32_t>(b[1]) << 16;
        }
        *at = make_uint4(h[0], h[1], h[2], h[3]);
        *low = make_uint4(l[0], l[1], l[2], l[3]);
    }
}
template <int PARTS>
__global__ __launch_bounds__(kTurnThreads) void loss_turn_kernel(uint16_t* __restrict__ grad, uint64_t stride, uint32_t first, uint32_t count,
                                                                uint32_t across, Kept near, Kept wide, const float* __restrict__ lse,
                                                                const int32_t* __restrict__ labels, const Meta* __restrict__ meta) {
    if constexpr (PARTS == 2)
        if (meta->wide != 0) return turn<3>(grad, stride, first, count, across, wide, lse, labels, meta);
    turn<PARTS>(grad, stride, first, count, across, near, lse, labels, meta);
}

// gx of every token: the splits' sums in order times the factor; zeros for tokens that do not count. A wave per token and 256
// columns, four a lane; from kFinishWaves splits on a block, each wave every fourth of the splits (ways), the waves' sums added
// in order (one token, 64 splits of 1024 columns: 5 us, 35 by one wave). The last block: the loss, the tokens' losses added
// in a fixed order.
constexpr uint32_t kFinishThreads = 256, kFinishWaves = kFinishThreads / kWave, kFinishColumns = 4 * kWave;
template <typename T, uint32_t WAYS>
__global__ __launch_bounds__(kFinishThreads) void loss_finish_kernel(const float* __restrict__ partial, uint32_t splits, uint32_t n_pad, uint32_t width,
                                                                    const int32_t* __restrict__ place, const Meta* __restrict__ meta,
                                                                    uint32_t n, uint32_t d, float scale, bool mean, const float* __restrict__ losses,
                                                                    float* __restrict__ loss, T* __restrict__ gx) {
    const Meta m = *meta;
    if (blockIdx.x == gridDim.x - 1) {
        __shared__ double lds[kFinishThreads];
        double sum = 0.0;
#pragma unroll 8
        for (uint32_t i = threadIdx.x; i < n; i += kFinishThreads) sum += losses[i];
        lds[threadIdx.x] = sum;
        __syncthreads();
        for (uint32_t half = kFinishThreads / 2; half > 0; half /= 2) {
            if (threadIdx.x < half) lds[threadIdx.x] += lds[threadIdx.x + half];
            __syncthreads();
        }
        if (threadIdx.x == 0) *loss = static_cast<float>(mean && m.valid != 0 ? lds[0] / m.valid : lds[0]);
        return;
    }
    __shared__ Four sums[kFinishWaves][kWave];
    const uint32_t lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave), across = (d + kFinishColumns - 1) / kFinishColumns;
    const uint32_t unit = blockIdx.x * (kFinishWaves / WAYS) + wave / WAYS, t = unit / across, c = unit % across * kFinishColumns + 4 * lane;
    const int32_t row = t < n ? place[t] : -1;
    const float factor = grad_factor(m, scale, mean);
    Four v = 0.0f;
    if (row >= 0 && c < d) {
        const float* from = partial + static_cast<uint64_t>(row) * width + c;
        const uint64_t next = static_cast<uint64_t>(n_pad) * width;
#pragma unroll 4
        for (uint32_t s = wave % WAYS; s < splits; s += WAYS) v += *reinterpret_cast<const Four*>(from + s * next);
    }
    if constexpr (WAYS != 1) {
        sums[wave][lane] = v;
        __syncthreads();
        if (wave != 0) return;
#pragma unroll
        for (uint32_t w = 1; w < kFinishWaves; ++w) v += sums[w][lane];
    }
    if (t >= n || c >= d) return;
    if (row >= 0) v *= factor;
    else if (m.invalid != 0) v = factor;  // NaN: a label was outside the vocabulary
    T* to = gx + static_cast<uint64_t>(t) * d + c;
    if (c + 4 <= d) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<FourAnywhere*>(to) = v;
        else *reinterpret_cast<HalvesAnywhere*>(to) = HalvesAnywhere{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3])};
    } else {
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
            if (c + k < d) {
                if constexpr (sizeof(T) == 4) to[k] = v[k];
                else to[k] = bf16_bits(v[k]);
            }
    }
}

// ------------------------------------------------------------------------------------------------------------ the host

constexpr uint32_t kTile = 256;                      // vocabulary rows and width of a tile
constexpr uint32_t kFewTokens = 64, kFewTile = 128;  // a few tokens: tiles of 128 x 64, two blocks a CU
constexpr uint32_t kFewRows = 16384;                 // float32: vocabulary rows from which reading them as they are pays
constexpr uint32_t kCus = 256;

uint32_t ceil_div(uint64_t a, uint32_t b) { return static_cast<uint32_t>((a + b - 1) / b); }
uint32_t padded(uint32_t v, uint32_t to) { return ceil_div(v, to) * to; }

// How a call runs. parts: 1 bfloat16, 2 float32 as fp16 hi + lo, 3 float32 as three bfloat16 parts split where they are
// multiplied. A few tokens wait for the weight, not for the matrix unit, and packing it reads and writes it once more: float32
// calls then read it as it is (in 4-byte transfers where its rows are not made of whole 16-byte pieces: losses of one token
// of 1001 x 50304 in 69 us, packed 164). Losses, width 1024, as it is against packed: 1
// token of 50304 rows 67 against 161 us, 128 tokens 110 / 159, 192 156 / 195, 256 202 / 202; of 32768 rows 128 tokens 107 /
// 115, 192 151 / 126; of 16384 rows 64 tokens 58 / 62, 128 102 / 64; of 10000 rows 64 tokens 57 / 48. Steps gain less (their
// products with D split what they read): 64 tokens of 50304 rows 229 / 324 us, 128 362 / 350. The width moves little: losses of
// 50304 rows, width 512, 192 tokens 90 / 118, 256 116 / 122, of 16384 rows 64 tokens 37 / 40, 128 60 / 42; width 2048 192 tokens
// 315 / 371, 256 413 / 376, 64 of 16384 rows 110 / 115, 128 198 / 115; steps of 50304 rows, width 512, 64 tokens 139 / 188, 128
// 224 / 214, width 2048 440 / 595 and 726 / 652.
// bfloat16 calls of up to 64 tokens take tiles of 128 x 64, two blocks a CU, instead of 256 x 256 (D in one part on either
// side): losses of 64 tokens of 50304 rows at widths 512, 1024 and 2048 21 / 29, 31 / 44 and 58 / 78 us, of 96 27 / 29, 42 / 44 and
// 75 / 77; steps of 64 75 / 87, 116 / 127, 204 / 215. (Of 8192 rows 64 tokens 24 / 20 and 57 / 45: few tiles favour the large ones.)
struct Plan {
    uint32_t parts, words, planes, n_pad, width, vocab_tile, token_tile, height, per_tile, slices, piece, pieces, last, stats_tiles, keep_tiles, splits;
    bool whole, few, in_place, keeps;  // whole: the weight's rows are made of whole 16-byte pieces
    uint64_t meta, rows, labels, place, lse, picked, losses, slice_sums, x_most, w_most, x, x_split, weight, grad, partial, bytes;
};

// `aligned`: the weight starts on a 16-byte boundary.
Plan plan_of(int vt, uint32_t n, uint32_t d, uint32_t vocab, bool aligned, bool gradients, uint64_t piece_bytes) {
    Plan p{};
    p.words = vt == kBF16 ? 1 : 2;
    p.whole = d % (8 / p.words) == 0 && aligned;
    if (vt == kBF16) p.few = n <= kFewTokens;
    else p.few = n <= (gradients ? 1 : 3) * kFewTokens && vocab >= ceil_div(n, kFewTokens) * kFewRows;
    p.parts = vt == kBF16 ? 1 : p.few ? 3 : 2;
    p.vocab_tile = p.few ? kFewTile : kTile;
    p.token_tile = p.few ? kFewTokens : p.parts == 1 ? 256 : 128;
    p.n_pad = padded(n, p.few ? kFewTokens : 256);
    p.width = padded(d, 64 / p.words);
    p.in_place = p.parts == 3 || (p.parts == 1 && p.whole);
    p.per_tile = p.parts == 2 ? 8 : 4;  // slices: as many as waves of quarter tiles (few: of tiles) along the vocabulary
    p.pieces = 1;
    p.piece = padded(vocab, kTile);
    if (gradients) {
        // A tile of D's rows is read by 32-bit byte offsets from its first (Operand::begin), which its last row must not pass; a
        // launch has below 2^32 threads, and loss_turn_kernel's one for 8 entries of D, in whole blocks of a row.
        p.planes = p.few && p.parts == 1 ? 2 : 1;
        const uint64_t reach = ((1ull << 32) - 256) / (2ull * p.words * (p.token_tile - 1) * kTile);
        const uint64_t turned = (1ull << 32) / (kTile / 8 * static_cast<uint64_t>(p.n_pad)) - 8 * kTurnThreads / kTile;
        const uint64_t asked = (piece_bytes == 0 ? kLossPieceBytes : piece_bytes) / (2ull * p.words * p.planes * p.n_pad * kTile);
        const uint64_t most = std::min({asked, reach, turned});
        const uint32_t tiles = ceil_div(vocab, kTile), fit = most < 1 ? 1 : most < tiles ? static_cast<uint32_t>(most) : tiles;
        p.piece = ceil_div(tiles, ceil_div(tiles, fit)) * kTile;
        p.pieces = ceil_div(vocab, p.piece);
    }
    // The last piece's exponentials stay where its D belongs. Not those of a few bfloat16 tokens, whose products wait for the
    // weight.
    p.keeps = gradients && !(p.few && p.parts == 1);
    p.last = p.keeps ? (p.pieces - 1) * p.piece : vocab;
    // A few tokens' vocabulary tiles share the rows evenly between the blocks that the CUs hold (50304 rows: 99 or 112 of 128
    // a block, 512 blocks, where whole tiles would be 393); their results go out in sixteens where D is written.
    p.height = p.vocab_tile;
    if (p.few) {
        const uint32_t blocks = 2 * kCus, even = ceil_div(vocab, blocks * ceil_div(vocab, blocks * kFewTile));
        p.height = gradients ? padded(even, 16) : even < 16 ? 16 : even;
    }
    p.stats_tiles = ceil_div(p.last, p.height);
    p.keep_tiles = p.keeps ? ceil_div(padded(vocab - p.last, kTile), p.height) : 0;
    p.slices = (p.stats_tiles + p.keep_tiles) * p.per_tile;
    uint64_t at = 0;
    const auto take = [&](uint64_t bytes) {
        const uint64_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    p.meta = take(sizeof(Meta));
    p.rows = take(4ull * p.n_pad);
    p.labels = take(4ull * p.n_pad);
    p.place = take(4ull * p.n_pad);
    p.lse = take(4ull * p.n_pad);
    p.picked = take(4ull * p.n_pad);
    p.losses = take(4ull * p.n_pad);
    p.slice_sums = take(sizeof(float2) * p.slices * p.n_pad);
    if (p.parts == 2) {
        p.x_most = take(sizeof(uint2) * ceil_div(p.n_pad, kPrepWaves));
        p.w_most = take(sizeof(uint2) * ceil_div(vocab, kWeightRows));
    }
    p.x = take(2ull * p.words * p.n_pad * p.width);
    p.weight = p.in_place ? 0 : take(2ull * p.words * vocab * p.width);
    // (packed weights are not read by the form that reads x split, which then may lie in their place)
    const bool within = p.parts == 2 && 6ull * p.n_pad <= 4ull * vocab;
    p.x_split = p.parts == 1 ? 0 : within ? p.weight : take(6ull * p.n_pad * p.width);
    if (gradients) {
        // splits of the vocabulary that give every CU a block (few tokens: two), each of 8 k-tiles at least
        const uint32_t blocks = ceil_div(p.width, p.vocab_tile) * (p.n_pad / p.token_tile), k_tiles = p.piece / (64 / p.words);
        const uint32_t fill = ceil_div(p.few ? 2 * kCus : kCus, blocks), limit = k_tiles / 8 < 1 ? 1 : k_tiles / 8;
        p.splits = fill < limit ? fill : limit;
        p.grad = take(2ull * p.words * p.planes * p.n_pad * p.piece);
        p.partial = take(4ull * p.splits * p.n_pad * p.width);
    }
    p.bytes = at;
    return p;
}

template <int PARTS, Use USE, int WA, int WB, int TA, int TB, uint32_t GRAIN = 16, bool LOW = false>
hipError_t launch_product(const Product& p, hipStream_t stream) {
    constexpr uint32_t kBlocks = WA * WB == 4 ? 2 * kCus : kCus;  // as many as the CUs hold
    hipLaunchKernelGGL((loss_product_kernel<PARTS, USE, WA, WB, TA, TB, GRAIN, LOW>), dim3(kBlocks), dim3(WA * WB * kWave), 0, stream, p);
    return hipGetLastError();
}

// One way to run a call's products: where the operands lie, and the tiles of the kernels that multiply them.
struct Form {
    uint32_t parts;
    Spread only;
    const uint16_t *weight, *x;  // x: as the weight's products read it
    uint32_t w_columns;
    uint64_t w_row, x_row;
    uint32_t vocab_tile, height, per_tile, stats_tiles, keep_tiles, gw_tile, gw_rows;
    Slices slices;
};

template <Use USE>
hipError_t product(const Plan& plan, const Form& form, const Product& p, hipStream_t stream) {
    if constexpr (USE != Use::GradW)  // which does not read the weight
        if (form.parts == 3 && !plan.whole) return launch_product<3, USE, 4, 1, 1, 2, 4>(p, stream);
    if (form.parts == 3) return launch_product<3, USE, 4, 1, 1, 2>(p, stream);
    if constexpr (USE == Use::Stats)
        if (plan.few) return launch_product<1, USE, 4, 1, 1, 2>(p, stream);
    // gw of a few bfloat16 tokens, one k-tile a tile: 128 x 128 in one stage, two blocks a CU (1 token of 1024 x 50304: a step of 112 us,
    // 123 with 8 waves and one block a CU)
    if constexpr (USE == Use::GradW)
        if (plan.few) return launch_product<1, USE, 4, 1, 1, 4, 16, true>(p, stream);
    if constexpr (USE == Use::Grad || USE == Use::GradX)
        if (plan.few) return launch_product<1, USE, 4, 1, 1, 2, 16, true>(p, stream);
    return form.parts == 1 ? launch_product<1, USE, 2, 4, 4, 2>(p, stream) : launch_product<2, USE, 4, 2, 2, 2>(p, stream);
}

template <typename T>
hipError_t run(const LossCall& c, hipStream_t stream) {
    const bool gradients = c.gw != nullptr;
    const Plan plan = plan_of(c.value_type, c.n, c.d, c.vocab, reinterpret_cast<uintptr_t>(c.weight) % 16 == 0, gradients, c.piece_bytes);
    char* const work = static_cast<char*>(c.workspace);
    Meta* const meta = reinterpret_cast<Meta*>(work + plan.meta);
    int32_t *const rows = reinterpret_cast<int32_t*>(work + plan.rows), *const labels = reinterpret_cast<int32_t*>(work + plan.labels),
            *const place = reinterpret_cast<int32_t*>(work + plan.place);
    float *const lse = reinterpret_cast<float*>(work + plan.lse), *const picked = reinterpret_cast<float*>(work + plan.picked);
    float* const losses = c.losses != nullptr ? c.losses : reinterpret_cast<float*>(work + plan.losses);
    uint16_t* const x = reinterpret_cast<uint16_t*>(work + plan.x);
    const uint16_t *const given = static_cast<const uint16_t*>(c.weight), *const x_split = reinterpret_cast<const uint16_t*>(work + plan.x_split);
    const uint32_t depth = 64 / plan.words;
    const uint64_t x_row = static_cast<uint64_t>(plan.width) * plan.words;
    const auto failed = [](hipError_t& status) { return (status = hipGetLastError()) != hipSuccess; };
    hipError_t status;

    const Prepare prepare{c.labels, c.x, c.weight, c.labels_stride, c.ignore, c.x_stride, c.wide_labels, c.n, c.d, plan.width, c.vocab, rows, labels,
                          place, losses, meta, x, reinterpret_cast<uint16_t*>(work + plan.weight), reinterpret_cast<uint16_t*>(work + plan.x_split),
                          reinterpret_cast<uint2*>(work + plan.x_most), reinterpret_cast<uint2*>(work + plan.w_most),
                          ceil_div(padded(c.n, 64), kPrepWaves), plan.in_place ? 0 : ceil_div(c.vocab, kWeightRows)};
    if (c.n > kScanTokens) {
        hipLaunchKernelGGL(loss_scan_kernel, dim3(1), dim3(kScanThreads), 0, stream, prepare);
        if (failed(status)) return status;
    }
    const dim3 prepare_grid(prepare.x_blocks + prepare.w_blocks);
    if constexpr (sizeof(T) == 4) {
        if (plan.parts == 3) hipLaunchKernelGGL((loss_prepare_kernel<T, true>), prepare_grid, dim3(kPrepThreads), 0, stream, prepare);
        else hipLaunchKernelGGL((loss_prepare_kernel<T, false>), prepare_grid, dim3(kPrepThreads), 0, stream, prepare);
        if (failed(status)) return status;
        if (plan.parts == 2) hipLaunchKernelGGL(loss_settle_kernel, dim3(2 * kCus), dim3(kPrepThreads), 0, stream, prepare);
    } else {
        hipLaunchKernelGGL((loss_prepare_kernel<T, false>), prepare_grid, dim3(kPrepThreads), 0, stream, prepare);
    }
    if (failed(status)) return status;

    float2* const slice_sums = reinterpret_cast<float2*>(work + plan.slice_sums);
    const uint32_t kept = plan.keeps ? padded(c.vocab - plan.last, kTile) : 0;
    const auto of_raw = [&](uint32_t height, Spread only) {  // float32: the weight as it is, x split
        const uint32_t stats_tiles = ceil_div(plan.last, height), keep_tiles = ceil_div(kept, height), slices = (stats_tiles + keep_tiles) * 4;
        return Form{3, only, given, x_split, c.d, 2ull * c.d, 3ull * plan.width, kFewTile, height, 4, stats_tiles, keep_tiles, kFewTile, 64,
                    {slice_sums, slices, slices}};
    };
    Form forms[2];
    uint32_t form_count = 1;
    if (plan.parts == 3) {
        forms[0] = of_raw(plan.height, Spread::Any);
    } else {
        const uint32_t w_columns = plan.in_place ? c.d : plan.width;
        forms[0] = {plan.parts, plan.parts == 2 ? Spread::Near : Spread::Any, plan.in_place ? given : reinterpret_cast<const uint16_t*>(work + plan.weight), x,
                    w_columns, static_cast<uint64_t>(w_columns) * plan.words, x_row, plan.vocab_tile, plan.height, plan.per_tile, plan.stats_tiles,
                    plan.keep_tiles, plan.few ? kFewTile : kTile, plan.few || plan.parts == 2 ? 128u : 256u,
                    {slice_sums, plan.slices, plan.few ? plan.slices : plan.n_pad}};
        if (plan.parts == 2) forms[form_count++] = of_raw(kFewTile, Spread::Wide);
    }
    // `what` of every form, until one fails
    const auto each = [&](auto what) -> hipError_t {
        for (uint32_t k = 0; k < form_count; ++k)
            if (hipError_t failure = what(forms[k]); failure != hipSuccess) return failure;
        return hipSuccess;
    };
    const auto begun = [&](const Form& form) {
        Product p{};
        p.meta = meta;
        p.labels = labels;
        p.lse = lse;
        p.vocab = c.vocab;
        p.n_pad = plan.n_pad;
        p.scale = c.scale;
        p.mean = c.mean;
        p.out_bf16 = c.value_type == kBF16;
        p.splits = 1;
        p.only = form.only;
        return p;
    };
    const uint64_t grad_row = static_cast<uint64_t>(plan.piece) * plan.words;
    // the logits of `rows` vocabulary rows from `first` on
    const auto logits = [&](const Form& form, uint32_t first, uint32_t rows) {
        Product p = begun(form);
        p.a = form.weight;
        p.a_stride = form.w_row;
        p.a_columns = form.w_columns;
        p.a_first = first;
        p.a_tiles = ceil_div(rows, form.height);
        p.a_columns_out = rows;
        p.b = form.x;
        p.b_stride = form.x_row;
        p.b_columns = plan.width;
        p.k_tiles = plan.width / depth;
        p.height = form.height;
        p.picked = picked;
        p.slices = slice_sums;
        p.slice_pitch = form.slices.pitch;
        p.slice_first = first == plan.last ? form.stats_tiles * form.per_tile : 0;
        p.grad = reinterpret_cast<uint16_t*>(work + plan.grad);
        p.grad_stride = grad_row;
        p.grad_low = plan.n_pad * grad_row;
        return p;
    };
    if (plan.last != 0 && (status = each([&](const Form& form) { return product<Use::Stats>(plan, form, logits(form, 0, plan.last), stream); })) != hipSuccess)
        return status;
    if (plan.keeps && (status = each([&](const Form& form) { return product<Use::Keep>(plan, form, logits(form, plan.last, kept), stream); })) != hipSuccess)
        return status;
    const Slices none{};
    const auto lse_of = [&](auto tokens) {
        constexpr uint32_t kTokens = decltype(tokens)::value;
        hipLaunchKernelGGL(loss_lse_kernel<kTokens>, dim3(ceil_div(c.n, kTokens)), dim3(kLseThreads), 0, stream, forms[0].slices,
                           form_count == 2 ? forms[1].slices : none, picked, rows, labels, meta, lse, losses);
    };
    // tokens a block: one where few are all there are, more where that still fills the CUs (runs of 128 bytes of a slice; 8192
    // tokens: 15 us, in fours 46; 512 float32 tokens in fours 10 us, in sixteens 16)
    if (plan.few) lse_of(std::integral_constant<uint32_t, 1>{});
    else if (c.n < 1024) lse_of(std::integral_constant<uint32_t, 4>{});
    else lse_of(std::integral_constant<uint32_t, 16>{});
    if (failed(status)) return status;
    if (!gradients) return hipSuccess;

    for (uint32_t piece = plan.pieces; piece-- > 0;) {
        const uint32_t first = piece * plan.piece, count = c.vocab - first < plan.piece ? c.vocab - first : plan.piece, columns = padded(count, kTile);
        uint16_t* const grad = reinterpret_cast<uint16_t*>(work + plan.grad);
        if (first == plan.last) {
            const uint32_t across = ceil_div(columns, 8 * kTurnThreads);
            const auto kept_by = [&](const Form& form) {
                const uint64_t before = static_cast<uint64_t>(form.stats_tiles) * form.per_tile;
                return Kept{slice_sums + before * (plan.few || form.parts == 3 ? 1 : form.slices.pitch), form.height, form.per_tile,
                            form.vocab_tile / form.per_tile, form.slices.pitch};
            };
            const auto turned = [&](auto parts) {
                constexpr int kParts = decltype(parts)::value;
                hipLaunchKernelGGL(loss_turn_kernel<kParts>, dim3(across * padded(c.n, 64)), dim3(kTurnThreads), 0, stream, grad, grad_row, first, columns,
                                   across, kept_by(forms[0]), kept_by(forms[form_count - 1]), lse, labels, meta);
            };
            if (plan.parts == 1) turned(std::integral_constant<int, 1>{});
            else if (plan.parts == 2) turned(std::integral_constant<int, 2>{});
            else turned(std::integral_constant<int, 3>{});
            if (failed(status)) return status;
        } else if ((status = each([&](const Form& form) { return product<Use::Grad>(plan, form, logits(form, first, columns), stream); })) != hipSuccess) {
            return status;
        }

        status = each([&](const Form& form) {
            Product gx = begun(form);
            gx.a = form.weight + first * form.w_row;
            gx.a_stride = form.w_row;
            gx.a_columns = form.w_columns;
            gx.b = grad;
            gx.b_stride = grad_row;
            gx.grad_low = plan.n_pad * grad_row;
            gx.b_columns = plan.piece;
            gx.a_first = first;
            gx.a_count = plan.width;
            gx.k_tiles = ceil_div(count, depth);
            gx.a_tiles = ceil_div(form.w_columns, form.vocab_tile);
            gx.splits = plan.splits;
            gx.partial = reinterpret_cast<float*>(work + plan.partial);
            gx.out_stride = plan.width;
            gx.add = piece + 1 != plan.pieces;
            return product<Use::GradX>(plan, form, gx, stream);
        });
        if (status != hipSuccess) return status;

        status = each([&](const Form& form) {
            Product gw = begun(form);
            gw.a = x;
            gw.a_stride = x_row;
            gw.a_columns = plan.width;
            gw.b = grad;
            gw.b_stride = grad_row;
            gw.grad_low = plan.n_pad * grad_row;
            gw.b_columns = plan.piece;
            gw.a_count = c.d;
            gw.b_count = count;
            gw.a_tiles = ceil_div(c.d, form.gw_tile);
            gw.b_tiles = ceil_div(count, form.gw_rows);
            gw.out = static_cast<T*>(c.gw) + static_cast<uint64_t>(first) * c.d;
            gw.out_stride = c.d;
            return product<Use::GradW>(plan, form, gw, stream);
        });
        if (status != hipSuccess) return status;
    }
    const auto finish = [&](auto ways) {
        constexpr uint32_t kWays = decltype(ways)::value;
        const uint32_t blocks = ceil_div(static_cast<uint64_t>(c.n) * ceil_div(c.d, kFinishColumns), kFinishWaves / kWays);
        hipLaunchKernelGGL((loss_finish_kernel<T, kWays>), dim3(blocks + 1), dim3(kFinishThreads), 0, stream,
                           reinterpret_cast<const float*>(work + plan.partial), plan.splits, plan.n_pad, plan.width, place, meta, c.n, c.d, c.scale, c.mean,
                           losses, c.loss, static_cast<T*>(c.gx));
    };
    if (plan.splits < kFinishWaves) finish(std::integral_constant<uint32_t, 1>{});
    else finish(std::integral_constant<uint32_t, kFinishWaves>{});
    return hipGetLastError();
}

}  // namespace

uint64_t loss_workspace_bytes(int vt, uint32_t n, uint32_t d, uint32_t vocab, bool aligned, bool gradients, uint64_t piece_bytes) {
    return plan_of(vt, n, d, vocab, aligned, gradients, piece_bytes).bytes;
}

hipError_t launch_loss(const LossCall& call, hipStream_t stream) {
    return call.value_type == kBF16 ? run<uint16_t>(call, stream) : run<float>(call, stream);
}

}  // namespace hffn
