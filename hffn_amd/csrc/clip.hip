// The global norm over many tensors and the clipping of their entries to it: two launches per table of kClipArrays arrays.
// The first leaves one float64 partial per block; every block of the second adds the partials up again (8 KB a table out
// of L2), so that no block waits for another, and scales its share.
//
// Bound by memory: 152 million entries in 145 tensors (506 MB; two tables) take 93 us for the norm, 5.4 TB/s, and 217 us scaled into 609 MB
// of others, 5.1 TB/s, a copy's rate. 36 tensors, 10 MB in all: 5.2 and 3.3 us, less than the host's part of the calls (24 us).
#include <vector>

#include "common.hpp"
#include "launch.hpp"

namespace hffn {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint64_t kChunk = 8192;  // entries of an array that a block takes at a time

// The table of a launch, in the kernel's arguments: the arrays and the chunk each begins with.
struct Table {
    const void* p[kClipArrays];
    void* out[kClipArrays];
    uint64_t count[kClipArrays];
    uint32_t first[kClipArrays + 1];
    uint8_t types[kClipArrays];  // bit 0: entries are bfloat16, bit 1: the scaled ones are
    uint32_t arrays;
};
static_assert(sizeof(Table) + 64 <= 4096, "a kernel's arguments end at 4 KB");

__device__ __forceinline__ uint32_t array_of(const Table& table, uint32_t chunk) {
    uint32_t low = 0, high = table.arrays;  // first[low] <= chunk < first[high]
    while (high - low > 1) {
        const uint32_t middle = (low + high) / 2;
        if (table.first[middle] <= chunk) low = middle;
        else high = middle;
    }
    return low;
}

// The larger magnitude; a NaN stays.
__device__ __forceinline__ double larger(double a, double b) { return b > a || b != b ? b : a; }

template <bool LARGEST>
__device__ __forceinline__ void take(double& into, float v) {
    const double w = static_cast<double>(v);  // squares of every float32 are float64 values: nothing overflows
    if constexpr (LARGEST) into = larger(into, fabs(w));
    else into = fma(w, w, into);
}

template <bool LARGEST>
__device__ __forceinline__ double joined(double a, double b) {
    return LARGEST ? larger(a, b) : a + b;
}

// The block's value from its threads' (a tree of fixed order), in every thread.
template <bool LARGEST>
__device__ __forceinline__ double block_join(double v, double (&lds)[kThreads]) {
    lds[threadIdx.x] = v;
    __syncthreads();
#pragma unroll
    for (uint32_t half = kThreads / 2; half > 0; half /= 2) {
        if (threadIdx.x < half) lds[threadIdx.x] = joined<LARGEST>(lds[threadIdx.x], lds[threadIdx.x + half]);
        __syncthreads();
    }
    return lds[0];
}

template <typename T, bool LARGEST>
__device__ __forceinline__ void take_chunk(const T* __restrict__ p, uint64_t count, double& into) {
    constexpr uint32_t V = 16 / sizeof(T);
    const uint32_t lead = static_cast<uint32_t>((16 - reinterpret_cast<uintptr_t>(p) % 16) % 16 / sizeof(T));
    const uint32_t all = static_cast<uint32_t>(count), before = lead < all ? lead : all, pieces = (all - before) / V;
    if (threadIdx.x < before) take<LARGEST>(into, widen(p[threadIdx.x]));
    const uint4* q = reinterpret_cast<const uint4*>(p + before);
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < pieces; i += kThreads) {
        const uint4 v = q[i];
        const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (sizeof(T) == 4) {
                take<LARGEST>(into, __uint_as_float(words[k]));
            } else {
                take<LARGEST>(into, __uint_as_float(words[k] << 16));
                take<LARGEST>(into, __uint_as_float(words[k] & 0xffff0000u));
            }
        }
    }
    const uint32_t rest = before + pieces * V + threadIdx.x;
    if (rest < all) take<LARGEST>(into, widen(p[rest]));  // fewer than V entries
}

template <bool LARGEST>
__global__ __launch_bounds__(kThreads) void norm_partials_kernel(Table table, double* __restrict__ partials) {
    __shared__ double lds[kThreads];
    double mine = 0.0;
    for (uint32_t chunk = blockIdx.x; chunk < table.first[table.arrays]; chunk += gridDim.x) {
        const uint32_t which = array_of(table, chunk);
        const uint64_t start = (chunk - table.first[which]) * kChunk, left = table.count[which] - start, count = left < kChunk ? left : kChunk;
        if (table.types[which] & 1) take_chunk<uint16_t, LARGEST>(static_cast<const uint16_t*>(table.p[which]) + start, count, mine);
        else take_chunk<float, LARGEST>(static_cast<const float*>(table.p[which]) + start, count, mine);
    }
    const double sum = block_join<LARGEST>(mine, lds);
    if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

template <bool LARGEST>
__device__ __forceinline__ double norm_of(const double* __restrict__ partials, uint32_t count, double (&lds)[kThreads]) {
    double mine = 0.0;
    for (uint32_t i = threadIdx.x; i < count; i += kThreads) mine = joined<LARGEST>(mine, partials[i]);
    const double sum = block_join<LARGEST>(mine, lds);
    return LARGEST ? sum : sqrt(sum);
}

template <bool LARGEST>
__global__ __launch_bounds__(kThreads) void norm_kernel(const double* __restrict__ partials, uint32_t count, float* __restrict__ norm) {
    __shared__ double lds[kThreads];
    const double value = norm_of<LARGEST>(partials, count, lds);
    if (threadIdx.x == 0) *norm = static_cast<float>(value);
}

template <typename T>
__device__ __forceinline__ void put(T* out, float v) {
    if constexpr (sizeof(T) == 4) *out = v;
    else *out = bf16_bits(v);
}

template <typename T, typename U>
__device__ __forceinline__ void scale_chunk(const T* p, U* out, uint64_t count, float factor) {
    constexpr uint32_t V = 16 / sizeof(T);
    const uint32_t lead = static_cast<uint32_t>((16 - reinterpret_cast<uintptr_t>(p) % 16) % 16 / sizeof(T));
    const uint32_t all = static_cast<uint32_t>(count), before = lead < all ? lead : all;
    // whole pieces where the scaled entries' pieces start on 16-byte boundaries too; else entry by entry
    const bool whole = reinterpret_cast<uintptr_t>(out + before) % 16 == 0;
    const uint32_t pieces = whole ? (all - before) / V : 0;
    if (threadIdx.x < before) put(out + threadIdx.x, factor * widen(p[threadIdx.x]));
    const uint4* q = reinterpret_cast<const uint4*>(p + before);
    constexpr uint32_t kAhead = 4;  // pieces of a thread requested before the first is written (p and out may be one array)
    for (uint32_t first = threadIdx.x; first < pieces; first += kAhead * kThreads) {
        uint4 v[kAhead];
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j)
            if (first + j * kThreads < pieces) v[j] = q[first + j * kThreads];
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            const uint32_t i = first + j * kThreads;
            if (i >= pieces) break;
            const uint32_t words[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
            float w[V];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (sizeof(T) == 4) {
                    w[k] = factor * __uint_as_float(words[k]);
                } else {
                    w[2 * k] = factor * __uint_as_float(words[k] << 16);
                    w[2 * k + 1] = factor * __uint_as_float(words[k] & 0xffff0000u);
                }
            }
            U* to = out + before + i * V;
            if constexpr (sizeof(U) == 4) {
#pragma unroll
                for (uint32_t k = 0; k < V; k += 4) {
                    typedef float Four __attribute__((ext_vector_type(4)));
                    __builtin_nontemporal_store((Four{w[k], w[k + 1], w[k + 2], w[k + 3]}), reinterpret_cast<Four*>(to + k));
                }
            } else {
#pragma unroll
                for (uint32_t k = 0; k < V; k += 4)
                    *reinterpret_cast<uint2*>(to + k) = make_uint2(bf16_pair(w[k], w[k + 1]), bf16_pair(w[k + 2], w[k + 3]));
            }
        }
    }
    for (uint32_t i = before + pieces * V + threadIdx.x; i < all; i += kThreads) put(out + i, factor * widen(p[i]));
}

// The arrays of one table scaled, last entries first: they were read last and lie in the caches. float32 entries are stored past the
// caches (331 -> 311 us of the call above, into other tensors; in place, and with an AdamW step behind, the same time either way:
// 101 million entries 85 us, 719 with the step). `count` partials are all tables'. In place with a factor of one
// nothing is written: every entry would be itself.
template <bool LARGEST>
__global__ __launch_bounds__(kThreads) void clip_kernel(Table table, const double* __restrict__ partials, uint32_t count, double limit,
                                                       bool in_place, float* __restrict__ norm) {
    __shared__ double lds[kThreads];
    const double value = norm_of<LARGEST>(partials, count, lds);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(value);
    const double quotient = limit / (value + 1e-6);
    const float factor = quotient >= 1.0 ? 1.0f : static_cast<float>(quotient);  // a NaN norm makes every entry NaN
    if (in_place && factor == 1.0f) return;
    const uint32_t chunks = table.first[table.arrays];
    for (uint32_t turn = blockIdx.x; turn < chunks; turn += gridDim.x) {
        const uint32_t chunk = chunks - 1 - turn, which = array_of(table, chunk);
        const uint64_t start = (chunk - table.first[which]) * kChunk, left = table.count[which] - start, n = left < kChunk ? left : kChunk;
        const float* p = static_cast<const float*>(table.p[which]) + start;
        const uint16_t* q = static_cast<const uint16_t*>(table.p[which]) + start;
        float* out = static_cast<float*>(table.out[which]) + start;
        uint16_t* out16 = static_cast<uint16_t*>(table.out[which]) + start;
        switch (table.types[which]) {
            case 0: scale_chunk(p, out, n, factor); break;
            case 1: scale_chunk(q, out, n, factor); break;
            case 2: scale_chunk(p, out16, n, factor); break;
            default: scale_chunk(q, out16, n, factor); break;
        }
    }
}

// The table of up to kClipArrays arrays from arrays[*next] on (empty ones left out); returns its chunks, which fit 32
// bits (kMaxClipEntries).
uint32_t fill(Table& table, const ClipArray* arrays, uint32_t count, uint32_t* next) {
    table.arrays = 0;
    uint64_t chunks = 0;
    table.first[0] = 0;
    while (*next < count && table.arrays < kClipArrays) {
        const ClipArray& a = arrays[*next];
        const uint64_t more = (a.count + kChunk - 1) / kChunk;
        ++*next;
        if (more == 0) continue;
        const uint32_t k = table.arrays++;
        table.p[k] = a.p;
        table.out[k] = a.out;
        table.count[k] = a.count;
        table.types[k] = static_cast<uint8_t>((a.type == kBF16 ? 1 : 0) | (a.out_type == kBF16 ? 2 : 0));
        chunks += more;
        table.first[k + 1] = static_cast<uint32_t>(chunks);
    }
    return static_cast<uint32_t>(chunks);
}

template <bool LARGEST>
hipError_t partials_of(const ClipArray* arrays, uint32_t count, double* partials, uint32_t* used, hipStream_t stream) {
    Table table;
    *used = 0;
    for (uint32_t next = 0; next < count;) {
        const uint32_t chunks = fill(table, arrays, count, &next);
        if (chunks == 0) continue;
        const uint32_t blocks = chunks < kClipPartials ? chunks : kClipPartials;
        hipLaunchKernelGGL(norm_partials_kernel<LARGEST>, dim3(blocks), dim3(kThreads), 0, stream, table, partials + *used);
        if (hipError_t status = hipGetLastError(); status != hipSuccess) return status;
        *used += blocks;
    }
    return hipSuccess;
}

template <bool LARGEST>
hipError_t norm_and_clip(const ClipArray* arrays, uint32_t count, bool clip, double limit, bool in_place, double* partials, float* norm,
                         hipStream_t stream) {
    uint32_t used;
    if (hipError_t status = partials_of<LARGEST>(arrays, count, partials, &used, stream); status != hipSuccess) return status;
    if (!clip || used == 0) {
        hipLaunchKernelGGL(norm_kernel<LARGEST>, dim3(1), dim3(kThreads), 0, stream, partials, used, norm);
        return hipGetLastError();
    }
    Table table;
    std::vector<uint32_t> starts;  // the tables' first arrays
    for (uint32_t next = 0; next < count;) {
        starts.push_back(next);
        fill(table, arrays, count, &next);
    }
    for (size_t k = starts.size(); k-- > 0;) {
        uint32_t next = starts[k];
        const uint32_t chunks = fill(table, arrays, count, &next);
        if (chunks == 0) continue;
        const uint32_t blocks = chunks < 2 * kClipPartials ? chunks : 2 * kClipPartials;
        hipLaunchKernelGGL(clip_kernel<LARGEST>, dim3(blocks), dim3(kThreads), 0, stream, table, partials, used, limit, in_place, norm);
        if (hipError_t status = hipGetLastError(); status != hipSuccess) return status;
    }
    return hipSuccess;
}

}  // namespace

uint64_t clip_workspace_bytes(uint32_t arrays) {
    return (static_cast<uint64_t>(arrays) / kClipArrays + 1) * kClipPartials * sizeof(double);
}

hipError_t launch_grad_norm(const ClipArray* arrays, uint32_t count, bool largest, double* partials, float* norm, hipStream_t stream) {
    return largest ? norm_and_clip<true>(arrays, count, false, 0.0, false, partials, norm, stream)
                   : norm_and_clip<false>(arrays, count, false, 0.0, false, partials, norm, stream);
}

hipError_t launch_clip(const ClipArray* arrays, uint32_t count, bool largest, double limit, bool in_place, double* partials, float* norm,
                       hipStream_t stream) {
    return largest ? norm_and_clip<true>(arrays, count, true, limit, in_place, partials, norm, stream)
                   : norm_and_clip<false>(arrays, count, true, limit, in_place, partials, norm, stream);
}

}  // namespace hffn
