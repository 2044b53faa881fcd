// The boundary between two blocks of a residual stack, forward and backward, one pass over the rows each:
//   u = post_norm(f) (or f),  r = x + scale gate u,  h = norm(r)
// with layer norms (v - mean) / sqrt(var + eps) w + b or RMS norms v / sqrt(mean(v^2) + eps) w. Rows stay in registers between
// the statistics (float32) and their use, so each is read and written once; statistics are computed again by the backward
// rather than kept: a row costs its reading either way.
#include <type_traits>

#include "common.hpp"
#include "launch.hpp"

namespace hffn {
namespace {

// V consecutive entries of a row as they lie in memory: 16 bytes, or one entry where rows start anywhere.
template <typename T, int V>
struct Piece {
    static_assert(V * sizeof(T) == 16 || V == 1, "16 bytes or an entry");
    using Raw = typename std::conditional<V == 1, T, uint4>::type;
    Raw raw;
    __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const Raw*>(p); }
    __device__ __forceinline__ void clear() {
        if constexpr (V == 1) raw = 0;
        else raw = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void widened(float* out) const {
        if constexpr (V == 1) {
            out[0] = widen(raw);
        } else {
            const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (sizeof(T) == 4) {
                    out[k] = __uint_as_float(words[k]);
                } else {
                    out[2 * k] = __uint_as_float(words[k] << 16);
                    out[2 * k + 1] = __uint_as_float(words[k] & 0xffff0000u);
                }
            }
        }
    }
};

template <typename T, int V>
__device__ __forceinline__ void store_row(T* p, const float* in) {
    if constexpr (sizeof(T) == 4) {
        if constexpr (V == 1) *p = in[0];
        else *reinterpret_cast<float4*>(p) = make_float4(in[0], in[1], in[2], in[3]);
    } else if constexpr (V == 1) {
        *p = bf16_bits(in[0]);
    } else {
        *reinterpret_cast<uint4*>(p) = make_uint4(bf16_pair(in[0], in[1]), bf16_pair(in[2], in[3]), bf16_pair(in[4], in[5]), bf16_pair(in[6], in[7]));
    }
}

// A thread's share of a row of d entries: C pieces of V, one every LANES pieces, E entries in all.
template <typename T, int V, int C, int LANES>
struct Share {
    static constexpr int E = V * C;
    uint32_t lane, d;
    __device__ __forceinline__ uint32_t at(int c) const { return (c * LANES + lane) * V; }
    __device__ __forceinline__ void request(const void* rows, uint64_t stride, uint32_t row, bool live, Piece<T, V> (&to)[C]) const {
        const T* p = static_cast<const T*>(rows) + row * stride;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (live && at(c) < d) to[c].load(p + at(c));
            else to[c].clear();
        }
    }
    __device__ __forceinline__ static void widened(const Piece<T, V> (&from)[C], float (&to)[E]) {
#pragma unroll
        for (int c = 0; c < C; ++c) from[c].widened(to + c * V);
    }
    __device__ __forceinline__ void store(void* rows, uint32_t row, const float (&from)[E]) const {
        T* p = static_cast<T*>(rows) + static_cast<uint64_t>(row) * d;
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (at(c) < d) store_row<T, V>(p + at(c), from + c * V);
    }
    // a float32 parameter, `otherwise` where there is none and beyond the row
    __device__ __forceinline__ void parameter(const float* p, float otherwise, float (&to)[E]) const {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int k = 0; k < V; ++k) to[c * V + k] = otherwise;
        if (p == nullptr) return;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (at(c) >= d) continue;
#pragma unroll
            for (int k = 0; k < V; k += V < 4 ? V : 4) {
                if constexpr (V == 1) {
                    to[c] = p[at(c)];
                } else {
                    const float4 v = *reinterpret_cast<const float4*>(p + at(c) + k);
                    to[c * V + k] = v.x; to[c * V + k + 1] = v.y; to[c * V + k + 2] = v.z; to[c * V + k + 3] = v.w;
                }
            }
        }
    }
    // entries beyond the row to zero
    __device__ __forceinline__ void cut(float (&v)[E]) const {
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (at(c) >= d)
#pragma unroll
                for (int k = 0; k < V; ++k) v[c * V + k] = 0.0f;
    }
};

// Sums of K values over the WPR waves of a row; every thread receives the same totals (waves in order). Two rows in turn use
// places of their own (`step` + kSteps): a place is written again only after a barrier that every reader of its last
// use has passed.
constexpr int kSteps = 4;  // sums of one row at most
template <int WPR, int K>
__device__ __forceinline__ void row_sums(float (&v)[K], float (*lds)[16 * 2], uint32_t step) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = wave_sum(v[k]);
    if constexpr (WPR > 1) {
        const uint32_t wave = threadIdx.x / kWave, first = wave / WPR * WPR;
        if (threadIdx.x % kWave == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) lds[step][2 * wave + k] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < WPR; ++w) sum += lds[step][2 * (first + w) + k];
            v[k] = sum;
        }
    }
}

// A block takes THREADS / LANES rows at a time and requests its next ones before it finishes these. Bound by memory: 8192 bfloat16
// rows of 2560 with f and a post norm 29.9 us for 168 MB, 5.6 TB/s; one row 2.6 us, a launch.
template <typename T, int V, int C, int WPR, int THREADS, bool LAYER, bool POST>
__global__ __launch_bounds__(THREADS) void residual_norm_kernel(NormForward a) {
    constexpr int LANES = kWave * WPR, ROWS = THREADS / LANES;
    using S = Share<T, V, C, LANES>;
    constexpr int E = S::E;
    __shared__ float lds[2 * kSteps][16 * 2];
    const S s{threadIdx.x % LANES, a.d};
    const float inv_d = 1.0f / static_cast<float>(a.d);
    uint32_t row = blockIdx.x * ROWS + threadIdx.x / LANES;
    Piece<T, V> px[C], pf[C];
    const auto request = [&](uint32_t from) {
        s.request(a.x, a.x_stride, from, from < a.n, px);
        if (a.f != nullptr) s.request(a.f, a.f_stride, from, from < a.n, pf);
    };
    request(row);
    float weight[E], bias[E], post_weight[POST ? E : 1], post_bias[POST && LAYER ? E : 1], gate[E];
    s.parameter(a.weight, 0.0f, weight);
    if constexpr (LAYER) s.parameter(a.bias, 0.0f, bias);
    if constexpr (POST) s.parameter(a.post_weight, 0.0f, post_weight);
    if constexpr (POST && LAYER) s.parameter(a.post_bias, 0.0f, post_bias);
    s.parameter(a.gate, 1.0f, gate);
    for (uint32_t base = blockIdx.x * ROWS, parity = 0; base < a.n; base += gridDim.x * ROWS, parity ^= 1) {
        float r[E], u[E];
        uint32_t step = parity * kSteps;
        S::widened(px, r);
        if (a.f != nullptr) S::widened(pf, u);
        const uint32_t here = row;
        row += gridDim.x * ROWS;
        request(row);
        if (a.f != nullptr) {
            if constexpr (POST) {
                float mean = 0.0f;
                if constexpr (LAYER) {
                    float sum[1] = {0.0f};
#pragma unroll
                    for (int e = 0; e < E; ++e) sum[0] += u[e];
                    row_sums<WPR, 1>(sum, lds, step++);
                    mean = sum[0] * inv_d;
                }
                float square[1] = {0.0f};
#pragma unroll
                for (int e = 0; e < E; ++e) u[e] -= mean;
                s.cut(u);
#pragma unroll
                for (int e = 0; e < E; ++e) square[0] = fmaf(u[e], u[e], square[0]);
                row_sums<WPR, 1>(square, lds, step++);
                const float inverse = rsqrtf(square[0] * inv_d + a.eps);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    u[e] *= inverse * post_weight[e];
                    if constexpr (LAYER) u[e] += post_bias[e];
                }
            }
#pragma unroll
            for (int e = 0; e < E; ++e) r[e] = fmaf(a.scale * gate[e], u[e], r[e]);
            if (here < a.n) s.store(a.r, here, r);
        }
        float mean = 0.0f;
        if constexpr (LAYER) {
            float sum[1] = {0.0f};
#pragma unroll
            for (int e = 0; e < E; ++e) sum[0] += r[e];
            row_sums<WPR, 1>(sum, lds, step++);
            mean = sum[0] * inv_d;
        }
        float square[1] = {0.0f};
#pragma unroll
        for (int e = 0; e < E; ++e) r[e] -= mean;
        s.cut(r);
#pragma unroll
        for (int e = 0; e < E; ++e) square[0] = fmaf(r[e], r[e], square[0]);
        row_sums<WPR, 1>(square, lds, step++);
        const float inverse = rsqrtf(square[0] * inv_d + a.eps);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            r[e] *= inverse * weight[e];
            if constexpr (LAYER) r[e] += bias[e];
        }
        if (here < a.n) s.store(a.h, here, r);
    }
}

// Column sums of a block's rows stay in its threads' registers and go out once per block, the block's rows added up in
// order, as rows of partials [kNormGrads][blocks][width] in the order weight, bias, gate, post_weight, post_bias;
// column_sums_kernel adds them. 2048 float32 rows of 1024 with f: 16.5 us for 50 MB, and 3.9 us for the 256 blocks' partials: three
// reductions over a row's two waves and few rows a block, latency rather than memory. (A block per row and atomics on the
// parameters' gradients would make their sums depend on the order.)
constexpr uint32_t kSumsLds = 4096;  // floats: the rows of a block side by side
template <typename T, int V, int C, int WPR, int THREADS, bool LAYER, bool POST>
__global__ __launch_bounds__(THREADS) void residual_norm_back_kernel(NormBackward a, uint32_t width) {
    constexpr int LANES = kWave * WPR, ROWS = THREADS / LANES;
    using S = Share<T, V, C, LANES>;
    constexpr int E = S::E;
    static_assert(ROWS == 1 || ROWS * LANES * E <= static_cast<int>(kSumsLds), "a block's rows fit");
    __shared__ float lds[2 * kSteps][16 * 2];
    __shared__ float rows_lds[ROWS > 1 ? kSumsLds : 1];
    const S s{threadIdx.x % LANES, a.d};
    const float inv_d = 1.0f / static_cast<float>(a.d);
    const bool with_f = POST || a.gate != nullptr;
    uint32_t row = blockIdx.x * ROWS + threadIdx.x / LANES;
    Piece<T, V> pr[C], pf[C], pgr[C], pgh[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        pf[c].clear();
        pgr[c].clear();
    }
    const auto request = [&](uint32_t from) {
        s.request(a.r, a.r_stride, from, from < a.n, pr);
        s.request(a.gh, a.gh_stride, from, from < a.n, pgh);
        if (with_f) s.request(a.f, a.f_stride, from, from < a.n, pf);
        if (a.gr != nullptr) s.request(a.gr, a.gr_stride, from, from < a.n, pgr);
    };
    request(row);
    float weight[E], gate[E], post_weight[POST ? E : 1], post_bias[POST && LAYER ? E : 1];
    s.parameter(a.weight, 0.0f, weight);
    s.parameter(a.gate, 1.0f, gate);
    if constexpr (POST) s.parameter(a.post_weight, 0.0f, post_weight);
    if constexpr (POST && LAYER) s.parameter(a.post_bias, 0.0f, post_bias);
    float sums[kNormGrads][E];
#pragma unroll
    for (int q = 0; q < kNormGrads; ++q)
#pragma unroll
        for (int e = 0; e < E; ++e) sums[q][e] = 0.0f;
    for (uint32_t base = blockIdx.x * ROWS, parity = 0; base < a.n; base += gridDim.x * ROWS, parity ^= 1) {
        float r[E], g[E], f[E], v[E];  // r, then its normalised entries; gh, then what comes back to f; f, then its normalised entries; gx
        uint32_t step = parity * kSteps;
        S::widened(pr, r);
        S::widened(pgh, g);
        S::widened(pf, f);
        S::widened(pgr, v);
        const uint32_t here = row;
        const bool live = here < a.n;
        row += gridDim.x * ROWS;
        request(row);
        float mean[2] = {0.0f, 0.0f}, square[2] = {0.0f, 0.0f};
        if constexpr (LAYER) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                mean[0] += r[e];
                if (POST) mean[1] += f[e];
            }
            row_sums<WPR, 2>(mean, lds, step++);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                r[e] -= mean[0] * inv_d;
                if (POST) f[e] -= mean[1] * inv_d;
            }
            s.cut(r);
            if (POST) s.cut(f);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            square[0] = fmaf(r[e], r[e], square[0]);
            if (POST) square[1] = fmaf(f[e], f[e], square[1]);
        }
        row_sums<WPR, 2>(square, lds, step++);
        const float inverse = rsqrtf(square[0] * inv_d + a.eps), post_inverse = POST ? rsqrtf(square[1] * inv_d + a.eps) : 1.0f;
        // through the norm of r: inverse (gh w - hat mean(gh w hat) [- mean(gh w)]), and gr
        float along[2] = {0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < E; ++e) {
            r[e] *= inverse;
            if (POST) f[e] *= post_inverse;
            if (live) {  // a row beyond the last may hold NaN (eps 0)
                sums[0][e] = fmaf(g[e], r[e], sums[0][e]);
                if (LAYER) sums[1][e] += g[e];
            }
            g[e] *= weight[e];
            along[0] = fmaf(g[e], r[e], along[0]);
            along[1] += g[e];
        }
        row_sums<WPR, 2>(along, lds, step++);
        along[0] *= inv_d;
        along[1] = LAYER ? along[1] * inv_d : 0.0f;
        float back[2] = {0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] += inverse * (g[e] - r[e] * along[0] - along[1]);
        s.cut(v);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float gu = a.scale * v[e], u = f[e];
            if constexpr (POST) {
                u *= post_weight[e];
                if constexpr (LAYER) u += post_bias[e];
            }
            if (live) sums[2][e] = fmaf(gu, u, sums[2][e]);
            gu *= gate[e];
            if constexpr (POST) {
                if (live) {
                    sums[3][e] = fmaf(gu, f[e], sums[3][e]);
                    if (LAYER) sums[4][e] += gu;
                }
                gu *= post_weight[e];
                back[0] = fmaf(gu, f[e], back[0]);
                back[1] += gu;
            }
            g[e] = gu;
        }
        if (live) s.store(a.gx, here, v);
        if constexpr (POST) {
            row_sums<WPR, 2>(back, lds, step++);
            back[0] *= inv_d;
            back[1] = LAYER ? back[1] * inv_d : 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) g[e] = post_inverse * (g[e] - f[e] * back[0] - back[1]);
        }
        if (a.gf != nullptr && live) s.store(a.gf, here, g);
    }
#pragma unroll
    for (int q = 0; q < kNormGrads; ++q) {
        const bool wanted = q == 0 || (q == 1 && LAYER) || (q == 2 && a.gate != nullptr) || (q == 3 && POST) || (q == 4 && POST && LAYER);
        if (!wanted) continue;
        float* out = a.partials + (static_cast<uint64_t>(q) * gridDim.x + blockIdx.x) * width;
        if constexpr (ROWS == 1) {
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (s.at(c) < a.d)
#pragma unroll
                    for (int k = 0; k < V; ++k) out[s.at(c) + k] = sums[q][c * V + k];
        } else {
            __syncthreads();  // the last gradient's rows are added up
            float* mine = rows_lds + threadIdx.x / LANES * a.d;
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (s.at(c) < a.d)
#pragma unroll
                    for (int k = 0; k < V; ++k) mine[s.at(c) + k] = sums[q][c * V + k];
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < a.d; i += THREADS) {
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < ROWS; ++w) sum += rows_lds[w * a.d + i];
                out[i] = sum;
            }
        }
    }
}

// out[q][i] = the sum over the blocks of partials[q][block][i], in a fixed order: 64 columns a block, four a thread, 64
// threads over the partial rows.
constexpr uint32_t kColumns = 64, kColumnThreads = 1024, kColumnRows = kColumnThreads / (kColumns / 4);
__global__ __launch_bounds__(kColumnThreads) void column_sums_kernel(const float* __restrict__ partials, NormGradients out, uint32_t rows, uint32_t d,
                                                                    uint32_t width) {
    __shared__ float4 lds[kColumnRows][kColumns / 4];
    float* const to = out.grad[blockIdx.y];
    if (to == nullptr) return;
    const uint32_t quad = threadIdx.x % (kColumns / 4), first = threadIdx.x / (kColumns / 4), column = blockIdx.x * kColumns + 4 * quad;
    const float* from = partials + static_cast<uint64_t>(blockIdx.y) * rows * width + column;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const auto add = [](float4 a, float4 b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); };
    if (column < width)
#pragma unroll 4
        for (uint32_t row = first; row < rows; row += kColumnRows) sum = add(sum, *reinterpret_cast<const float4*>(from + static_cast<uint64_t>(row) * width));
    lds[first][quad] = sum;
    __syncthreads();
#pragma unroll
    for (uint32_t half = kColumnRows / 2; half > 0; half /= 2) {
        if (first < half) lds[first][quad] = add(lds[first][quad], lds[first + half][quad]);
        __syncthreads();
    }
    if (threadIdx.x < kColumns && blockIdx.x * kColumns + threadIdx.x < d)
        to[blockIdx.x * kColumns + threadIdx.x] = reinterpret_cast<const float*>(&lds[0][0])[threadIdx.x];
}

constexpr uint32_t kBackBlocks = 256, kForwardBlocks = 1024;
// Waves that share a row: 8 entries a lane, 16 beyond 8192. Rows that start anywhere (one entry a load) take the next of
// 2, 8 and 16 waves.
uint32_t norm_waves(uint32_t d, bool whole) {
    if (!whole) return d <= 1024 ? 2 : d <= 4096 ? 8 : 16;
    return d <= 512 ? 1 : d <= 1024 ? 2 : d <= 2048 ? 4 : d <= 4096 ? 8 : 16;
}
uint32_t norm_rows(uint32_t d, bool whole) {  // a block's rows at a time
    const uint32_t waves = norm_waves(d, whole);
    return waves < 8 ? 8 / waves : 1;
}
uint32_t norm_width(uint32_t d) { return (d + 3) / 4 * 4; }

// Whether every row of these starts on a 16-byte boundary and holds whole 16-byte pieces.
bool whole_pieces(int vt, uint32_t d, std::initializer_list<const void*> rows, std::initializer_list<uint64_t> strides,
                  std::initializer_list<const float*> params) {
    const uint32_t per = vt == kBF16 ? 8 : 4;
    if (d % per != 0) return false;
    for (const void* p : rows)
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
    for (uint64_t s : strides)
        if (s % per != 0) return false;
    for (const float* p : params)
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
    return true;
}

template <typename T, int V, bool LAYER, bool POST>
hipError_t forward_widths(const NormForward& a, hipStream_t stream) {
    const uint32_t rows = norm_rows(a.d, V > 1), blocks = (a.n + rows - 1) / rows;
    const dim3 grid(blocks < kForwardBlocks ? blocks : kForwardBlocks);
#define HFFN_NORM(C, WPR, THREADS) hipLaunchKernelGGL((residual_norm_kernel<T, V, C, WPR, THREADS, LAYER, POST>), grid, dim3(THREADS), 0, stream, a)
    switch (norm_waves(a.d, V > 1)) {
        case 1: if constexpr (V > 1) HFFN_NORM(8 / V, 1, 512); break;
        case 2: HFFN_NORM(8 / V, 2, 512); break;
        case 4: if constexpr (V > 1) HFFN_NORM(8 / V, 4, 512); break;
        case 8: HFFN_NORM(8 / V, 8, 512); break;
        default: HFFN_NORM(16 / V, 16, 1024); break;
    }
#undef HFFN_NORM
    return hipGetLastError();
}

template <typename T, int V, bool LAYER, bool POST>
hipError_t backward_widths(const NormBackward& a, uint32_t blocks, hipStream_t stream) {
    const dim3 grid(blocks);
    const uint32_t width = norm_width(a.d);
#define HFFN_NORM(C, WPR, THREADS) hipLaunchKernelGGL((residual_norm_back_kernel<T, V, C, WPR, THREADS, LAYER, POST>), grid, dim3(THREADS), 0, stream, a, width)
    switch (norm_waves(a.d, V > 1)) {
        case 1: if constexpr (V > 1) HFFN_NORM(8 / V, 1, 512); break;
        case 2: HFFN_NORM(8 / V, 2, 512); break;
        case 4: if constexpr (V > 1) HFFN_NORM(8 / V, 4, 512); break;
        case 8: HFFN_NORM(8 / V, 8, 512); break;
        default: HFFN_NORM(16 / V, 16, 1024); break;
    }
#undef HFFN_NORM
    return hipGetLastError();
}

template <typename T, int V>
hipError_t forward_kinds(const NormForward& a, hipStream_t stream) {
    const bool post = a.post_weight != nullptr;
    if (a.layer) return post ? forward_widths<T, V, true, true>(a, stream) : forward_widths<T, V, true, false>(a, stream);
    return post ? forward_widths<T, V, false, true>(a, stream) : forward_widths<T, V, false, false>(a, stream);
}

template <typename T, int V>
hipError_t backward_kinds(const NormBackward& a, uint32_t blocks, hipStream_t stream) {
    const bool post = a.post_weight != nullptr;
    if (a.layer) return post ? backward_widths<T, V, true, true>(a, blocks, stream) : backward_widths<T, V, true, false>(a, blocks, stream);
    return post ? backward_widths<T, V, false, true>(a, blocks, stream) : backward_widths<T, V, false, false>(a, blocks, stream);
}

uint32_t back_blocks(uint32_t n, uint32_t d, bool whole) {
    const uint32_t rows = norm_rows(d, whole), blocks = (n + rows - 1) / rows;
    return blocks < kBackBlocks ? blocks : kBackBlocks;
}

}  // namespace

uint64_t norm_back_workspace(uint32_t n, uint32_t d) {  // one row a block gives the most blocks
    return static_cast<uint64_t>(kNormGrads) * (n < kBackBlocks ? n : kBackBlocks) * norm_width(d) * sizeof(float);
}

hipError_t launch_residual_norm(int vt, const NormForward& a, hipStream_t stream) {
    const bool whole = whole_pieces(vt, a.d, {a.x, a.f, a.r, a.h}, {a.x_stride, a.f_stride}, {a.weight, a.bias, a.gate, a.post_weight, a.post_bias});
    if (vt == kBF16) return whole ? forward_kinds<uint16_t, 8>(a, stream) : forward_kinds<uint16_t, 1>(a, stream);
    return whole ? forward_kinds<float, 4>(a, stream) : forward_kinds<float, 1>(a, stream);
}

hipError_t launch_residual_norm_backward(int vt, const NormBackward& a, const NormGradients& grads, hipStream_t stream) {
    const bool whole = whole_pieces(vt, a.d, {a.r, a.f, a.gr, a.gh, a.gx, a.gf}, {a.r_stride, a.f_stride, a.gr_stride, a.gh_stride},
                                    {a.weight, a.gate, a.post_weight, a.post_bias});
    const uint32_t blocks = back_blocks(a.n, a.d, whole);
    hipError_t status;
    if (vt == kBF16) status = whole ? backward_kinds<uint16_t, 8>(a, blocks, stream) : backward_kinds<uint16_t, 1>(a, blocks, stream);
    else status = whole ? backward_kinds<float, 4>(a, blocks, stream) : backward_kinds<float, 1>(a, blocks, stream);
    if (status != hipSuccess) return status;
    hipLaunchKernelGGL(column_sums_kernel, dim3((a.d + kColumns - 1) / kColumns, kNormGrads), dim3(kColumnThreads), 0, stream, a.partials, grads,
                       blocks, a.d, norm_width(a.d));
    return hipGetLastError();
}

}  // namespace hffn
