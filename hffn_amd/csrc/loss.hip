// Softmax cross entropy of a language-model head, from hidden rows x [n, d] and the head's weight [V, d], in pieces of the
// vocabulary and without keeping the logits:
//   l_t = log sum_v exp(x_t . w_v) - x_t . w_label(t),   D = softmax - onehot(label),   gx = f D W,   gw = f D^T x,
// f the gradient's factor (1 / counted tokens for the mean). The forward leaves, per slice of the vocabulary and token, the
// maximum and the sum of exponentials of its logits; the backward computes a piece's logits again, turns them into D
// (16 bits) and multiplies D by the weight's rows and by x.
//
// Every product is out[b][a] = sum_k A[a, k] B[b, k] on 16-bit MFMA operands with float32 sums. bfloat16 calls multiply
// their entries as they are (D rounded to bfloat16: 2^-8 of an entry, as the gradients themselves are rounded). float32
// calls hold every operand as fp16 hi + lo of the entry times a power of two of its tensor (the largest entry at
// 2^12..2^13; 22 bits down to 2^-16 of it) and take hi hi + hi lo + lo hi.
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

constexpr uint32_t kThreads = 512, kWaves = kThreads / kWave;
constexpr int kLift = 13;      // operands' largest entries lie below 2^kLift
constexpr int kGradLift = 14;  // |D| <= 1 is kept times 2^kGradLift
constexpr int kChain = 4;      // k-tiles whose products are summed in the MFMA accumulators (float32 calls)

// What the first launches leave for the others: counted tokens, labels outside the vocabulary, and (float32) the bits of
// the largest finite magnitudes of the weight and of the counted rows of x.
struct Meta {
    uint32_t valid, invalid, weight_bits, x_bits;
};
__device__ __forceinline__ int lift_of(uint32_t bits) {  // e with 2^-e times the largest entry in [2^12, 2^13)
    return bits == 0 ? 0 : ilogbf(__uint_as_float(bits)) - (kLift - 1);
}
__device__ __forceinline__ float grad_factor(const Meta& meta, float scale, bool mean) {
    if (meta.invalid != 0) return __uint_as_float(0x7fc00000u);
    return mean && meta.valid != 0 ? scale / static_cast<float>(meta.valid) : scale;
}

__device__ __forceinline__ void split(float v, uint16_t& hi, uint16_t& lo) {
    const _Float16 h = static_cast<_Float16>(v);
    const float rest = v - static_cast<float>(h);
    const _Float16 l = static_cast<_Float16>(fabsf(v) < 65504.0f ? rest : 0.0f);
    hi = __builtin_bit_cast(uint16_t, h);
    lo = __builtin_bit_cast(uint16_t, l);
}

// ------------------------------------------------------------------------------------------------ tokens and operands

// The counted tokens in order: rows[i] the token of compact row i and labels[i] its label; place[t] the compact row of
// token t or -1. A label outside the vocabulary counts as a token whose loss is NaN. One block.
constexpr uint32_t kScanThreads = 1024;
__global__ __launch_bounds__(kScanThreads) void loss_scan_kernel(const void* __restrict__ labels, int64_t stride, bool wide, int64_t ignore,
                                                                 uint32_t n, uint32_t vocab, int32_t* __restrict__ rows,
                                                                 int32_t* __restrict__ compact, int32_t* __restrict__ place,
                                                                 float* __restrict__ losses, Meta* __restrict__ meta) {
    __shared__ uint32_t counts[kScanThreads / kWave], bad[kScanThreads / kWave];
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    uint32_t base = 0, invalid = 0;
    for (uint32_t first = 0; first < n; first += kScanThreads) {
        const uint32_t t = first + threadIdx.x;
        int64_t label = ignore;
        if (t < n) label = wide ? static_cast<const int64_t*>(labels)[t * stride] : static_cast<const int32_t*>(labels)[t * stride];
        const bool counted = t < n && label != ignore, outside = counted && (label < 0 || label >= static_cast<int64_t>(vocab));
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
            rows[at] = static_cast<int32_t>(t);
            compact[at] = outside ? -1 : static_cast<int32_t>(label);
        }
        if (t < n) {
            place[t] = counted ? static_cast<int32_t>(at) : -1;
            if (!counted) losses[t] = 0.0f;
        }
        base += total;
        __syncthreads();
    }
    for (int step = 32; step > 0; step /= 2) invalid += __shfl_xor(invalid, step);
    if (lane == 0) bad[wave] = invalid;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 1; w < kScanThreads / kWave; ++w) invalid += bad[w];
        *meta = {base, invalid, 0u, 0u};
    }
}

// float32: the largest finite magnitudes of the weight and of x's counted rows (maxima: any order gives the same).
__device__ __forceinline__ uint32_t magnitude(float v) {
    const uint32_t bits = __float_as_uint(v) & 0x7fffffffu;
    return bits < 0x7f800000u ? bits : 0u;
}
constexpr uint32_t kRangeThreads = 256;
__global__ __launch_bounds__(kRangeThreads) void loss_range_kernel(const float* __restrict__ weight, uint64_t entries, const float* __restrict__ x,
                                                                  uint64_t x_stride, uint32_t d, const int32_t* __restrict__ rows,
                                                                  Meta* __restrict__ meta, uint32_t weight_blocks) {
    __shared__ uint32_t lds[kRangeThreads / kWave];
    uint32_t most = 0;
    const bool of_weight = blockIdx.x < weight_blocks;
    if (of_weight) {
        const uint64_t quads = reinterpret_cast<uintptr_t>(weight) % 16 == 0 ? entries / 4 : 0;
        const uint64_t step = static_cast<uint64_t>(weight_blocks) * kRangeThreads, first = static_cast<uint64_t>(blockIdx.x) * kRangeThreads + threadIdx.x;
#pragma unroll 4
        for (uint64_t i = first; i < quads; i += step) {
            const float4 v = reinterpret_cast<const float4*>(weight)[i];
            most = max(max(most, max(magnitude(v.x), magnitude(v.y))), max(magnitude(v.z), magnitude(v.w)));
        }
        for (uint64_t i = 4 * quads + first; i < entries; i += step) most = max(most, magnitude(weight[i]));
    } else {
        const uint32_t valid = meta->valid;
        for (uint32_t i = blockIdx.x - weight_blocks; i < valid; i += gridDim.x - weight_blocks)
            for (uint32_t c = threadIdx.x; c < d; c += kRangeThreads) most = max(most, magnitude(x[rows[i] * x_stride + c]));
    }
    for (int step = 32; step > 0; step /= 2) most = max(most, static_cast<uint32_t>(__shfl_xor(most, step)));
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = most;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 1; w < kRangeThreads / kWave; ++w) most = max(most, lds[w]);
        atomicMax(of_weight ? &meta->weight_bits : &meta->x_bits, most);
    }
}

// Operand rows: x's counted rows (zeros to the next multiple of 64) and, where it is not read in place, the weight's, as
// [rows][width] bfloat16 or, per 32 entries, 32 hi and 32 lo halves; zeros from d on. A wave per row.
constexpr uint32_t kPackThreads = 256, kPackRows = kPackThreads / kWave;
template <typename T>
__global__ __launch_bounds__(kPackThreads) void loss_pack_kernel(const T* __restrict__ x, uint64_t x_stride, const T* __restrict__ weight, uint32_t vocab,
                                                                uint32_t d, uint32_t width, const int32_t* __restrict__ rows,
                                                                const Meta* __restrict__ meta, uint16_t* __restrict__ x_out,
                                                                uint16_t* __restrict__ w_out, uint32_t x_blocks) {
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const bool of_x = blockIdx.x < x_blocks;
    const uint32_t row = (of_x ? blockIdx.x : blockIdx.x - x_blocks) * kPackRows + wave;
    const uint32_t valid = meta->valid;
    if (of_x ? row >= (valid + 63) / 64 * 64 : row >= vocab) return;
    const bool zero = of_x && row >= valid;
    const T* from = of_x ? (zero ? x : x + rows[row] * x_stride) : weight + static_cast<uint64_t>(row) * d;
    if constexpr (sizeof(T) == 4) {
        const int e = lift_of(of_x ? meta->x_bits : meta->weight_bits);
        uint16_t* to = (of_x ? x_out : w_out) + static_cast<uint64_t>(row) * 2 * width;
        for (uint32_t c = lane; c < width; c += kWave) {
            uint16_t hi, lo;
            split(zero || c >= d ? 0.0f : ldexpf(from[c], -e), hi, lo);
            to[c / 32 * 64 + c % 32] = hi;
            to[c / 32 * 64 + 32 + c % 32] = lo;
        }
    } else {
        uint16_t* to = (of_x ? x_out : w_out) + static_cast<uint64_t>(row) * width;
        for (uint32_t c = lane; c < width; c += kWave) to[c] = zero || c >= d ? 0 : from[c];
    }
}

// --------------------------------------------------------------------------------------------------------- the product

// Index permutation of the 32 rows of an MFMA operand: with it a lane's 16 results of a 32 x 32 tile are 16 consecutive
// indexes (16 (lane / 32) on) of the row operand.
__device__ __forceinline__ uint32_t permuted(uint32_t r) { return (r >> 2 & 1) * 16 + (r >> 3) * 4 + (r & 3); }

// An operand's tile in LDS, TILE indexes x 64 / PARTS k (128 bytes an index), 16-byte chunks swizzled so that the lanes of
// a read touch every bank: index-major (memory rows are the operand's indexes, k contiguous; a row's 8 chunks) or k-major
// (TR: memory rows are k, read through the LDS transpose reads). Transfers of 1 KB go straight from memory to LDS.
template <int PARTS, bool TR, int TILE>
struct Operand {
    static constexpr uint32_t kBytes = TILE * 128, kPieces = kBytes / 1024, kPerWave = kPieces / kWaves;
    static constexpr uint32_t kRow = TR ? TILE * 2 * PARTS : 128, kDepth = 64 / PARTS;
    static_assert(kPieces % kWaves == 0, "every wave transfers as many pieces");

    const char* base;        // of the tile at k = 0 (index-major) or of its first column (k-major)
    uint64_t stride;         // bytes of a memory row
    uint32_t offset[kPerWave];  // index-major: a lane's byte offset of each piece
    uint32_t row[kPerWave], last;  // k-major: the lane's k row of each piece (offset: its column); the last k row to read

    __device__ __forceinline__ static uint32_t swizzle(uint32_t r) {
        if constexpr (TR) return (r & 1) * 4 + (r >> 1 & 1) * 9;
        else return ((r & 3) | (r >> 4 & 1) << 2) ^ (r >> 2 & 1);
    }
    // first: the tile's first index; indexes: memory rows (index-major) or, padded, columns (k-major) there are; depth: k
    // rows there are (k-major)
    __device__ __forceinline__ void begin(const uint16_t* p, uint64_t row_entries, uint32_t first, uint32_t indexes, uint32_t depth) {
        const uint32_t wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
        stride = row_entries * 2;
        last = depth - 1;
        if constexpr (TR) base = reinterpret_cast<const char*>(p) + static_cast<uint64_t>(first) * 2 * PARTS;
        else base = reinterpret_cast<const char*>(p) + first * stride;
#pragma unroll
        for (uint32_t j = 0; j < kPerWave; ++j) {
            const uint32_t at = (wave * kPerWave + j) * 1024 + lane * 16, r = at / kRow, chunk = at % kRow / 16 ^ swizzle(r);
            if constexpr (TR) {
                const uint32_t chunks = (indexes - first) * PARTS / 8;  // to the end of the memory row
                row[j] = r;
                offset[j] = (chunk < chunks ? chunk : chunks - 1) * 16;
            } else {
                const uint32_t left = indexes - first - 1;  // clamped rows repeat the last: their results are dropped
                offset[j] = (r < left ? r : left) * static_cast<uint32_t>(stride) + chunk * 16;
            }
        }
    }
    // the tile of k-tile kt into LDS
    __device__ __forceinline__ void fetch(uint32_t kt, const char* lds) const {
        const uint32_t wave = threadIdx.x / kWave;
        if constexpr (TR) {
            const uint32_t k0 = kt * kDepth;
            const char* from = base + k0 * stride;
#pragma unroll
            for (uint32_t j = 0; j < kPerWave; ++j) {
                const uint32_t r = k0 + row[j] <= last ? row[j] : last - k0;  // beyond: the other operand holds zeros
                dma16(from, r * static_cast<uint32_t>(stride) + offset[j], lds + (wave * kPerWave + j) * 1024);
            }
        } else {
            const char* from = base + kt * 128;
#pragma unroll
            for (uint32_t j = 0; j < kPerWave; ++j) dma16(from, offset[j], lds + (wave * kPerWave + j) * 1024);
        }
    }
    // a lane's place in the tile for the 32-index blocks from `first` on
    __device__ __forceinline__ static uint32_t place(uint32_t first) {
        const uint32_t lane = threadIdx.x % kWave, half = lane / 32;
        if constexpr (TR) {
            const uint32_t in = lane % 16, block = (lane / 16 & 1) * 4 + in % 4, k = in / 4;
            const uint32_t column = first * 2 * PARTS + (block & 1) * 32 + (block >> 1) * 8;
            return (half * 8 + k) * kRow + (column ^ swizzle(k) * 16);
        } else {
            const uint32_t r = first + permuted(lane % 32);
            return r * 128 + (half ^ swizzle(r)) * 16;
        }
    }
    // entries k = 16 step + 8 (lane / 32) + 0..7 of index permuted(lane % 32) of block i
    __device__ __forceinline__ static Frag read(uint32_t tile, uint32_t place, int i, int step, int part) {
        if constexpr (TR) {
            const uint32_t at = tile + (place ^ (i * 64 * PARTS + part * 64)) + step * 16 * kRow;
            const Quad a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<LdsQuad>(at));
            const Quad b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<LdsQuad>(at + 4 * kRow));
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            return *reinterpret_cast<LdsFrag>(tile + i * 4096 + (place ^ (part * 64 + step * 32)));
        }
    }
};

template <int PARTS>
__device__ __forceinline__ Acc multiply(Frag a, Frag b, Acc c) {
    if constexpr (PARTS == 1) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(FragB, a), __builtin_bit_cast(FragB, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(FragH, a), __builtin_bit_cast(FragH, b), c, 0, 0, 0);
}

// float32 calls keep the exponential's last bits; bfloat16 ones round it to 8.
template <int PARTS>
__device__ __forceinline__ float exponential(float v) {
    if constexpr (PARTS == 2) return v < -150.0f ? 0.0f : exp_split(v);  // also -inf, of which exp_split makes a NaN
    else return __expf(v);
}

enum class Use { Stats, Grad, GradX, GradW };

// One product of a loss call: which operands, how far they go, and what becomes of the results.
struct Product {
    const uint16_t *a, *b;
    uint64_t a_stride, b_stride;  // entries (16 bits) of a memory row
    uint32_t a_first;             // Stats, Grad: first vocabulary row of the piece
    uint32_t a_count, b_count;    // GradX, GradW: columns of the output; GradW: its rows
    uint32_t vocab;
    uint32_t k_tiles;             // all (GradX: of the piece)
    uint32_t a_tiles, b_tiles, splits;
    const Meta* meta;
    const int32_t* labels;        // compact
    const float* lse;             // Grad, compact
    float* picked;                // Stats: the label's logit, compact
    float2* slices;               // Stats: [slice][n_pad] maximum and sum of exponentials
    uint16_t* grad;               // Grad: D, [n_pad][piece]
    uint64_t grad_stride;
    uint32_t n_pad;
    float* partial;               // GradX: [split][n_pad][d]
    bool add;
    void* out;                    // GradW: [V, d]
    uint64_t out_stride;
    float scale;
    bool mean, out_bf16;
};

// A block of 8 waves takes WA TA 32 x WB TB 32 results, k-tiles through a ring of STAGES tile pairs: a k-tile's transfers
// are issued STAGES - 1 k-tiles ahead, one barrier a k-tile.
template <int PARTS, Use USE, int WA, int WB, int TA, int TB>
struct Shape {
    static constexpr bool kATr = USE == Use::GradX || USE == Use::GradW, kBTr = USE == Use::GradW;
    static constexpr int kA = WA * TA * 32, kB = WB * TB * 32;
    using OpA = Operand<PARTS, kATr, kA>;
    using OpB = Operand<PARTS, kBTr, kB>;
    static constexpr uint32_t kStage = OpA::kBytes + OpB::kBytes;
    static constexpr int kStages = 163840 / kStage < 4 ? 163840 / kStage : 4;
    static constexpr uint32_t kLds = kStage * kStages;
    static_assert(WA * WB == static_cast<int>(kWaves) && kStages >= 2, "8 waves, two stages at least");
};

template <int PARTS, Use USE, int WA, int WB, int TA, int TB>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void loss_product_kernel(Product p) {
    using S = Shape<PARTS, USE, WA, WB, TA, TB>;
    using OpA = typename S::OpA;
    using OpB = typename S::OpB;
    __shared__ __attribute__((aligned(1024))) char ring[S::kLds];
    constexpr int kSteps = 4 / PARTS;
    const Meta meta = *p.meta;
    const uint32_t per_split = p.a_tiles * p.b_tiles, block = xcd_order(blockIdx.x, gridDim.x);
    const uint32_t split_at = block / per_split, in_split = block % per_split;
    // Stats, Grad: the token tiles of a vocabulary tile are neighbours; the others: the width tiles of a row tile
    const bool tokens_first = USE == Use::Stats || USE == Use::Grad;
    const uint32_t ta = tokens_first ? in_split / p.b_tiles : in_split % p.a_tiles, tb = tokens_first ? in_split % p.b_tiles : in_split / p.a_tiles;
    const uint32_t a0 = ta * S::kA, b0 = tb * S::kB;
    if (USE != Use::GradW && b0 >= meta.valid) return;

    uint32_t k_begin = 0, k_end = p.k_tiles;
    if (USE == Use::GradX) {
        k_begin = static_cast<uint64_t>(p.k_tiles) * split_at / p.splits;
        k_end = static_cast<uint64_t>(p.k_tiles) * (split_at + 1) / p.splits;
    }
    if (USE == Use::GradW) k_end = (meta.valid + OpA::kDepth - 1) / OpA::kDepth;

    OpA a;
    OpB b;
    if constexpr (USE == Use::Stats || USE == Use::Grad) {
        a.begin(p.a, p.a_stride, p.a_first + a0, p.vocab, 0);
        b.begin(p.b, p.b_stride, b0, p.n_pad, 0);
    } else if constexpr (USE == Use::GradX) {
        a.begin(p.a, p.a_stride, a0, static_cast<uint32_t>(p.a_stride / PARTS), p.vocab - p.a_first);
        b.begin(p.b, p.b_stride, b0, p.n_pad, 0);
    } else {
        a.begin(p.a, p.a_stride, a0, static_cast<uint32_t>(p.a_stride / PARTS), p.n_pad);
        b.begin(p.b, p.b_stride, b0, static_cast<uint32_t>(p.b_stride / PARTS), p.n_pad);
    }

    const uint32_t wave = threadIdx.x / kWave, wa = wave % WA, wb = wave / WA, lane = threadIdx.x % kWave;
    const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(ring));
    const uint32_t a_place = OpA::place(wa * TA * 32), b_place = OpB::place(wb * TB * 32);
    constexpr uint32_t kTransfers = OpA::kPerWave + OpB::kPerWave;
    const auto fetch = [&](uint32_t kt) {
        char* stage = ring + (kt - k_begin) % S::kStages * S::kStage;
        a.fetch(kt, stage);
        b.fetch(kt, stage + OpA::kBytes);
    };

    Acc acc[TA][TB], sums[PARTS == 2 ? TA : 1][PARTS == 2 ? TB : 1];
#pragma unroll
    for (int i = 0; i < TA; ++i)
#pragma unroll
        for (int j = 0; j < TB; ++j) {
            acc[i][j] = 0.0f;
            if constexpr (PARTS == 2) sums[i][j] = 0.0f;
        }
    for (uint32_t kt = k_begin; kt < k_end && kt < k_begin + S::kStages - 1; ++kt) fetch(kt);
    for (uint32_t kt = k_begin; kt < k_end; ++kt) {
        if (k_end - kt >= static_cast<uint32_t>(S::kStages) - 1) wait_loads<kTransfers * (S::kStages - 2)>();
        else wait_loads<0>();
        asm volatile("" ::: "memory");  // the last k-tile's LDS reads stay before the barrier, this one's behind it
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (kt + S::kStages - 1 < k_end) fetch(kt + S::kStages - 1);
        const uint32_t tile_a = lds + (kt - k_begin) % S::kStages * S::kStage, tile_b = tile_a + OpA::kBytes;
#pragma unroll
        for (int step = 0; step < kSteps; ++step) {
            Frag fa[TA][PARTS], fb[TB][PARTS];
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
#pragma unroll
                for (int i = 0; i < TA; ++i) fa[i][part] = OpA::read(tile_a, a_place, i, step, part);
#pragma unroll
                for (int j = 0; j < TB; ++j) fb[j][part] = OpB::read(tile_b, b_place, j, step, part);
            }
#pragma unroll
            for (int i = 0; i < TA; ++i)
#pragma unroll
                for (int j = 0; j < TB; ++j) {
                    acc[i][j] = multiply<PARTS>(fa[i][0], fb[j][0], acc[i][j]);
                    if constexpr (PARTS == 2) {
                        acc[i][j] = multiply<PARTS>(fa[i][0], fb[j][1], acc[i][j]);
                        acc[i][j] = multiply<PARTS>(fa[i][1], fb[j][0], acc[i][j]);
                    }
                }
        }
        if constexpr (PARTS == 2) {
            if ((kt - k_begin) % kChain == kChain - 1 || kt + 1 == k_end) {
#pragma unroll
                for (int i = 0; i < TA; ++i)
#pragma unroll
                    for (int j = 0; j < TB; ++j) {
                        sums[i][j] += acc[i][j];
                        acc[i][j] = 0.0f;
                    }
            }
        }
    }

    // a lane's results: index b0 + (wb TB + j) 32 + permuted(lane % 32) of B, indexes a0 + (wa TA + i) 32 + 16 (lane / 32)
    // + 0..15 of A
    const uint32_t half = lane / 32;
    float power = 1.0f;
    if constexpr (PARTS == 2) {
        const int ew = lift_of(meta.weight_bits), ex = lift_of(meta.x_bits);
        power = ldexpf(1.0f, USE == Use::GradX ? ew - kGradLift : USE == Use::GradW ? ex - kGradLift : 0);
        if constexpr (USE == Use::Stats || USE == Use::Grad) {
#pragma unroll
            for (int i = 0; i < TA; ++i)
#pragma unroll
                for (int j = 0; j < TB; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r) sums[i][j][r] = ldexpf(sums[i][j][r], ew + ex);
        }
    }
    const auto result = [&](int i, int j, int r) -> float {
        if constexpr (PARTS == 2) return sums[i][j][r];
        else return acc[i][j][r];
    };
    const uint32_t a_lane = a0 + wa * TA * 32 + 16 * half;
    // the value held for result (i, j, r)
    const auto at = [&](int i, int j) -> Acc& {
        if constexpr (PARTS == 2) return sums[i][j];
        else return acc[i][j];
    };
    if constexpr (USE == Use::Stats) {
        const uint32_t slice = ta * WA + wa;
        if (a0 + S::kA > p.vocab) {  // the last vocabulary tile: what lies beyond adds nothing
#pragma unroll
            for (int i = 0; i < TA; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (a_lane + i * 32 + r >= p.vocab)
#pragma unroll
                        for (int j = 0; j < TB; ++j) at(i, j)[r] = -__builtin_huge_valf();
        }
#pragma unroll
        for (int j = 0; j < TB; ++j) {
            const uint32_t t = b0 + (wb * TB + j) * 32 + permuted(lane % 32);
            float most = -__builtin_huge_valf();
#pragma unroll
            for (int i = 0; i < TA; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) most = fmaxf(most, result(i, j, r));
            most = fmaxf(most, __shfl_xor(most, 32));
            const float shift = most == -__builtin_huge_valf() ? 0.0f : most;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < TA; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) sum += exponential<PARTS>(result(i, j, r) - shift);
            sum += __shfl_xor(sum, 32);
            if (t >= meta.valid) continue;
            if (half == 0) p.slices[static_cast<uint64_t>(slice) * p.n_pad + t] = make_float2(most, sum);
            const uint32_t label = static_cast<uint32_t>(p.labels[t]) - a_lane;  // a label outside: far from every lane
            if (label < TA * 32 && (label & 16) == 0) {
                float logit = 0.0f;
#pragma unroll
                for (int i = 0; i < TA; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) logit = label == static_cast<uint32_t>(i * 32 + r) ? result(i, j, r) : logit;
                p.picked[t] = logit;
            }
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
                    } else {
                        uint16_t h[2], l[2];
                        split(v[0] * (1 << kGradLift), h[0], l[0]);
                        split(v[1] * (1 << kGradLift), h[1], l[1]);
                        hi[r / 2] = h[0] | static_cast<uint32_t>(h[1]) << 16;
                        lo[r / 2] = l[0] | static_cast<uint32_t>(l[1]) << 16;
                    }
                }
                uint16_t* to = p.grad + t * p.grad_stride + (a_lane - 16 * half + i * 32) * PARTS + 16 * half;
                *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4*>(to + 8) = make_uint4(hi[4], hi[5], hi[6], hi[7]);
                if constexpr (PARTS == 2) {
                    *reinterpret_cast<uint4*>(to + 32) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    *reinterpret_cast<uint4*>(to + 40) = make_uint4(lo[4], lo[5], lo[6], lo[7]);
                }
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
                    const uint64_t at = at_b * p.out_stride + at_a;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        if (at_a + r >= p.a_count) continue;
                        const float v = factor * result(i, j, r);
                        if (p.out_bf16) static_cast<uint16_t*>(p.out)[at + r] = bf16_bits(v);
                        else static_cast<float*>(p.out)[at + r] = v;
                    }
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------- the sums over the vocabulary

// lse and loss of every counted token from the slices: 16 tokens a block, 64 threads each over the slices.
constexpr uint32_t kLseTokens = 16, kLseLanes = 64;
__global__ __launch_bounds__(kLseTokens* kLseLanes) void loss_lse_kernel(const float2* __restrict__ slices, uint32_t count, uint32_t n_pad,
                                                                        const float* __restrict__ picked, const int32_t* __restrict__ rows,
                                                                        const int32_t* __restrict__ labels, const Meta* __restrict__ meta,
                                                                        float* __restrict__ lse, float* __restrict__ losses) {
    __shared__ float2 lds[kLseLanes][kLseTokens];
    const uint32_t in = threadIdx.x % kLseTokens, first = threadIdx.x / kLseTokens, t = blockIdx.x * kLseTokens + in, valid = meta->valid;
    if (blockIdx.x * kLseTokens >= valid) return;
    const auto join = [](float2 a, float2 b) {
        const float most = fmaxf(a.x, b.x);
        if (most == -__builtin_huge_valf()) return make_float2(most, a.y + b.y);
        return make_float2(most, a.y * expf(a.x - most) + b.y * expf(b.x - most));
    };
    float2 all = make_float2(-__builtin_huge_valf(), 0.0f);
    if (t < valid)
        for (uint32_t s = first; s < count; s += kLseLanes) all = join(all, slices[static_cast<uint64_t>(s) * n_pad + t]);
    lds[first][in] = all;
    __syncthreads();
    for (uint32_t step = kLseLanes / 2; step > 0; step /= 2) {
        if (first < step) lds[first][in] = join(lds[first][in], lds[first + step][in]);
        __syncthreads();
    }
    if (first != 0 || t >= valid) return;
    const float2 total = lds[0][in];
    const float value = total.x + logf(total.y);
    lse[t] = value;
    losses[rows[t]] = labels[t] < 0 ? __uint_as_float(0x7fc00000u) : value - picked[t];
}

// gx of every token: the splits' sums in order times the factor; zeros for tokens that do not count. The last block: the
// loss, the tokens' losses added in a fixed order.
constexpr uint32_t kFinishThreads = 256;
template <typename T>
__global__ __launch_bounds__(kFinishThreads) void loss_finish_kernel(const float* __restrict__ partial, uint32_t splits, uint32_t n_pad, uint32_t width,
                                                                    const int32_t* __restrict__ place, const Meta* __restrict__ meta, uint32_t n,
                                                                    uint32_t d, float scale, bool mean, const float* __restrict__ losses,
                                                                    float* __restrict__ loss, T* __restrict__ gx) {
    const Meta m = *meta;
    const uint32_t t = blockIdx.x;
    if (t == n) {
        __shared__ double lds[kFinishThreads];
        double sum = 0.0;
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
    const int32_t row = place[t];
    const float factor = grad_factor(m, scale, mean);
    for (uint32_t c = threadIdx.x; c < d; c += kFinishThreads) {
        float sum = 0.0f;
        if (row >= 0) {
            for (uint32_t s = 0; s < splits; ++s) sum += partial[(static_cast<uint64_t>(s) * n_pad + row) * width + c];
            sum *= factor;
        } else if (m.invalid != 0) {
            sum = factor;  // NaN: a label was outside the vocabulary
        }
        if constexpr (sizeof(T) == 4) gx[static_cast<uint64_t>(t) * d + c] = sum;
        else gx[static_cast<uint64_t>(t) * d + c] = bf16_bits(sum);
    }
}

// ------------------------------------------------------------------------------------------------------------ the host

constexpr uint32_t kTile = 256;               // vocabulary rows and width of a tile
constexpr uint64_t kGradBytes = 256ull << 20;  // a piece's D at most (or one vocabulary tile's)
constexpr uint32_t kBlocks = 256;             // CUs

uint32_t ceil_div(uint64_t a, uint32_t b) { return static_cast<uint32_t>((a + b - 1) / b); }
uint32_t padded(uint32_t v, uint32_t to) { return ceil_div(v, to) * to; }

struct Plan {
    uint32_t parts, n_pad, width, token_tile, slices, piece, pieces, splits;
    bool in_place;
    uint64_t meta, rows, labels, place, lse, picked, losses, slice_sums, x, weight, grad, partial, bytes;
};

Plan plan_of(int vt, uint32_t n, uint32_t d, uint32_t vocab, bool aligned, bool gradients) {
    Plan p{};
    p.parts = vt == kBF16 ? 1 : 2;
    p.token_tile = p.parts == 1 ? 256 : 128;
    p.n_pad = padded(n, 256);
    p.width = padded(d, 64 / p.parts);
    p.in_place = p.parts == 1 && d % 64 == 0 && aligned;
    p.slices = ceil_div(vocab, kTile) * (p.parts == 1 ? 2 : 4);
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
    p.x = take(2ull * p.parts * p.n_pad * p.width);
    p.weight = p.in_place ? 0 : take(2ull * p.parts * vocab * p.width);
    if (gradients) {
        const uint64_t per_row = 2ull * p.parts * p.n_pad;
        const uint64_t most = kGradBytes / (per_row * kTile);
        const uint32_t tiles = ceil_div(vocab, kTile), fit = most < 1 ? 1 : most < tiles ? static_cast<uint32_t>(most) : tiles;
        p.pieces = ceil_div(tiles, fit);
        p.piece = ceil_div(tiles, p.pieces) * kTile;
        p.pieces = ceil_div(vocab, p.piece);
        const uint32_t blocks = ceil_div(p.width, kTile) * (p.n_pad / p.token_tile), k_tiles = p.piece / (64 / p.parts);
        const uint32_t fill = ceil_div(kBlocks, blocks);  // splits that give every CU a block
        p.splits = fill < 1 ? 1 : fill > k_tiles / 8 ? (k_tiles / 8 < 1 ? 1 : k_tiles / 8) : fill;
        p.grad = take(per_row * p.piece);
        p.partial = take(4ull * p.splits * p.n_pad * p.width);
    }
    p.bytes = at;
    return p;
}

template <int PARTS, Use USE, int WA, int WB, int TA, int TB>
hipError_t launch_product(const Product& p, hipStream_t stream) {
    const auto kernel = loss_product_kernel<PARTS, USE, WA, WB, TA, TB>;
    hipLaunchKernelGGL(kernel, dim3(p.a_tiles * p.b_tiles * p.splits), dim3(kThreads), 0, stream, p);
    return hipGetLastError();
}

template <Use USE>
hipError_t product(uint32_t parts, const Product& p, hipStream_t stream) {
    return parts == 1 ? launch_product<1, USE, 2, 4, 4, 2>(p, stream) : launch_product<2, USE, 4, 2, 2, 2>(p, stream);
}

template <typename T>
hipError_t run(const LossCall& c, hipStream_t stream) {
    const bool gradients = c.gw != nullptr;
    const Plan plan = plan_of(c.value_type, c.n, c.d, c.vocab, reinterpret_cast<uintptr_t>(c.weight) % 16 == 0, gradients);
    char* const work = static_cast<char*>(c.workspace);
    Meta* const meta = reinterpret_cast<Meta*>(work + plan.meta);
    int32_t *const rows = reinterpret_cast<int32_t*>(work + plan.rows), *const labels = reinterpret_cast<int32_t*>(work + plan.labels),
            *const place = reinterpret_cast<int32_t*>(work + plan.place);
    float *const lse = reinterpret_cast<float*>(work + plan.lse), *const picked = reinterpret_cast<float*>(work + plan.picked);
    float* const losses = c.losses != nullptr ? c.losses : reinterpret_cast<float*>(work + plan.losses);
    uint16_t* const x = reinterpret_cast<uint16_t*>(work + plan.x);
    uint16_t* const packed = reinterpret_cast<uint16_t*>(work + plan.weight);
    const uint16_t* const weight = plan.in_place ? static_cast<const uint16_t*>(c.weight) : packed;
    const uint64_t row = static_cast<uint64_t>(plan.width) * plan.parts;
    const auto done = [](hipError_t& status) { return (status = hipGetLastError()) != hipSuccess; };
    hipError_t status;

    hipLaunchKernelGGL(loss_scan_kernel, dim3(1), dim3(kScanThreads), 0, stream, c.labels, c.labels_stride, c.wide_labels, c.ignore, c.n, c.vocab, rows,
                       labels, place, losses, meta);
    if (done(status)) return status;
    if constexpr (sizeof(T) == 4) {
        const uint32_t weight_blocks = 8 * kBlocks, x_blocks = c.n < kBlocks ? c.n : kBlocks;
        hipLaunchKernelGGL(loss_range_kernel, dim3(weight_blocks + x_blocks), dim3(kRangeThreads), 0, stream, static_cast<const float*>(c.weight),
                           static_cast<uint64_t>(c.vocab) * c.d, static_cast<const float*>(c.x), c.x_stride, c.d, rows, meta, weight_blocks);
        if (done(status)) return status;
    }
    const uint32_t x_blocks = ceil_div(padded(c.n, 64), kPackRows), w_blocks = plan.in_place ? 0 : ceil_div(c.vocab, kPackRows);
    hipLaunchKernelGGL(loss_pack_kernel<T>, dim3(x_blocks + w_blocks), dim3(kPackThreads), 0, stream, static_cast<const T*>(c.x), c.x_stride,
                       static_cast<const T*>(c.weight), c.vocab, c.d, plan.width, rows, meta, x, packed, x_blocks);
    if (done(status)) return status;

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
    const uint32_t token_tiles = ceil_div(c.n, plan.token_tile), width_tiles = ceil_div(plan.width, kTile);
    Product stats = p;
    stats.a = weight;
    stats.a_stride = row;
    stats.b = x;
    stats.b_stride = row;
    stats.k_tiles = plan.width / (64 / plan.parts);
    stats.a_tiles = ceil_div(c.vocab, kTile);
    stats.b_tiles = token_tiles;
    stats.picked = picked;
    stats.slices = reinterpret_cast<float2*>(work + plan.slice_sums);
    if ((status = product<Use::Stats>(plan.parts, stats, stream)) != hipSuccess) return status;
    hipLaunchKernelGGL(loss_lse_kernel, dim3(ceil_div(c.n, kLseTokens)), dim3(kLseTokens * kLseLanes), 0, stream, stats.slices, plan.slices, plan.n_pad,
                       picked, rows, labels, meta, lse, losses);
    if (done(status)) return status;
    if (!gradients) return hipSuccess;

    for (uint32_t first = 0; first < c.vocab; first += plan.piece) {
        const uint32_t count = c.vocab - first < plan.piece ? c.vocab - first : plan.piece;
        Product grad = stats;
        grad.a_first = first;
        grad.a_tiles = ceil_div(count, kTile);
        grad.grad = reinterpret_cast<uint16_t*>(work + plan.grad);
        grad.grad_stride = static_cast<uint64_t>(plan.piece) * plan.parts;
        if ((status = product<Use::Grad>(plan.parts, grad, stream)) != hipSuccess) return status;

        Product gx = p;
        gx.a = weight + first * row;
        gx.a_stride = row;
        gx.b = grad.grad;
        gx.b_stride = grad.grad_stride;
        gx.a_first = first;
        gx.a_count = plan.width;
        gx.k_tiles = ceil_div(count, 64 / plan.parts);
        gx.a_tiles = width_tiles;
        gx.b_tiles = token_tiles;
        gx.splits = plan.splits;
        gx.partial = reinterpret_cast<float*>(work + plan.partial);
        gx.out_stride = plan.width;
        gx.add = first != 0;
        if ((status = product<Use::GradX>(plan.parts, gx, stream)) != hipSuccess) return status;

        Product gw = p;
        gw.a = x;
        gw.a_stride = row;
        gw.b = grad.grad;
        gw.b_stride = grad.grad_stride;
        gw.a_count = c.d;
        gw.b_count = count;
        gw.a_tiles = width_tiles;
        gw.b_tiles = ceil_div(count, plan.token_tile);
        gw.out = static_cast<T*>(c.gw) + static_cast<uint64_t>(first) * c.d;
        gw.out_stride = c.d;
        if ((status = product<Use::GradW>(plan.parts, gw, stream)) != hipSuccess) return status;
    }
    hipLaunchKernelGGL(loss_finish_kernel<T>, dim3(c.n + 1), dim3(kFinishThreads), 0, stream, reinterpret_cast<const float*>(work + plan.partial), plan.splits,
                       plan.n_pad, plan.width, place, meta, c.n, c.d, c.scale, c.mean, losses, c.loss, static_cast<T*>(c.gx));
    return hipGetLastError();
}

}  // namespace

uint64_t loss_workspace_bytes(int vt, uint32_t n, uint32_t d, uint32_t vocab, bool aligned, bool gradients) {
    return plan_of(vt, n, d, vocab, aligned, gradients).bytes;
}

hipError_t launch_loss(const LossCall& call, hipStream_t stream) {
    return call.value_type == kBF16 ? run<uint16_t>(call, stream) : run<float>(call, stream);
}

}  // namespace hffn
