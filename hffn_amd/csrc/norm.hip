// The boundary between two blocks of a residual stack, forward and backward, one pass over the rows each:
//   u = post_norm(f) (or f),  r = x + scale gate u,  h = norm(r)
// with layer norms (v - mean) / sqrt(var + eps) w + b or RMS norms v / sqrt(mean(v^2) + eps) w.
#include "common.hpp"
#include "launch.hpp"

namespace hffn {
namespace {

// V consecutive entries of a row, widened: V = 16 bytes' worth, or 1 where rows start anywhere.
template <typename T, int V>
__device__ __forceinline__ void load_row(const T* p, float (&out)[V]) {
    if constexpr (V == 1) {
        out[0] = widen(*p);
    } else if constexpr (sizeof(T) == 4) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        out[0] = v.x; out[1] = v.y; out[2] = v.z; out[3] = v.w;
    } else {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            out[2 * k] = __uint_as_float(words[k] << 16);
            out[2 * k + 1] = __uint_as_float(words[k] & 0xffff0000u);
        }
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_row(T* p, const float (&in)[V]) {
    if constexpr (sizeof(T) == 4) {
        if constexpr (V == 1) *p = in[0];
        else *reinterpret_cast<float4*>(p) = make_float4(in[0], in[1], in[2], in[3]);
    } else if constexpr (V == 1) {
        *p = bf16_bits(in[0]);
    } else {
        uint32_t words[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) words[k] = bf16_pair(in[2 * k], in[2 * k + 1]);
        *reinterpret_cast<uint4*>(p) = make_uint4(words[0], words[1], words[2], words[3]);
    }
}

// V entries of a float32 parameter vector (16-byte aligned where V > 1).
template <int V>
__device__ __forceinline__ void load_param(const float* p, float (&out)[V]) {
    load_vec<V>(p, out);
}

// Sums of K values over the WPR waves of a row; every thread receives the same totals (waves in order). `slot` alternates
// between consecutive rows of a block, `step` counts the sums of a row: a slot is written again only after a barrier that
// every reader of its last use has passed.
template <int WPR, int K>
__device__ __forceinline__ void row_sums(float (&v)[K], float (*lds)[2 * WPR], uint32_t step) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = wave_sum(v[k]);
    if constexpr (WPR > 1) {
        const uint32_t wave = threadIdx.x / kWave;
        if (threadIdx.x % kWave == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) lds[step][K * wave + k] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < WPR; ++w) sum += lds[step][K * w + k];
            v[k] = sum;
        }
    }
}

// A thread's share of a row: C chunks of V entries, LANES chunks apart.
template <int V, int C, int LANES>
struct Share {
    static constexpr int kEntries = V * C;
    __device__ static __forceinline__ uint32_t at(uint32_t lane, int c) { return (c * LANES + lane) * V; }
};

constexpr int kSteps = 4;  // row sums of one row at most

template <typename T, int V, int C, int WPR, int THREADS, bool LAYER, bool POST>
__global__ __launch_bounds__(THREADS) void residual_norm_kernel(NormForward a) {
    constexpr int LANES = kWave * WPR, ROWS = THREADS / LANES, E = V * C;
    using S = Share<V, C, LANES>;
    __shared__ float lds[2 * kSteps][2 * WPR];
    const uint32_t lane = threadIdx.x % LANES, d = a.d;
    const float inv_d = 1.0f / static_cast<float>(d);
    uint32_t parity = 0;
    for (uint32_t row = blockIdx.x * ROWS + threadIdx.x / LANES; row < a.n; row += gridDim.x * ROWS) {
        float r[E];
        const T* x = static_cast<const T*>(a.x) + static_cast<uint64_t>(row) * a.x_stride;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float v[V];
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = 0.0f;
            if (S::at(lane, c) < d) load_row<T, V>(x + S::at(lane, c), v);
#pragma unroll
            for (int k = 0; k < V; ++k) r[c * V + k] = v[k];
        }
        uint32_t step = parity * kSteps;
        if (a.f != nullptr) {
            float u[E];
            const T* f = static_cast<const T*>(a.f) + static_cast<uint64_t>(row) * a.f_stride;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float v[V];
#pragma unroll
                for (int k = 0; k < V; ++k) v[k] = 0.0f;
                if (S::at(lane, c) < d) load_row<T, V>(f + S::at(lane, c), v);
#pragma unroll
                for (int k = 0; k < V; ++k) u[c * V + k] = v[k];
            }
            float mean = 0.0f, inverse = 1.0f;
            if constexpr (POST) {
                if constexpr (LAYER) {
                    float s[1] = {0.0f};
#pragma unroll
                    for (int e = 0; e < E; ++e) s[0] += u[e];
                    row_sums<WPR, 1>(s, lds, step++);
                    mean = s[0] * inv_d;
                }
                float s[1] = {0.0f};
#pragma unroll
                for (int c = 0; c < C; ++c)
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const float z = S::at(lane, c) < d ? u[c * V + k] - mean : 0.0f;
                        s[0] = fmaf(z, z, s[0]);
                    }
                row_sums<WPR, 1>(s, lds, step++);
                inverse = rsqrtf(s[0] * inv_d + a.eps);
            }
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const uint32_t at = S::at(lane, c);
                if (at >= d) continue;
                float w[V], b[V], g[V];
                if constexpr (POST) {
                    load_param<V>(a.post_weight + at, w);
                    if (LAYER && a.post_bias != nullptr) load_param<V>(a.post_bias + at, b);
                }
                if (a.gate != nullptr) load_param<V>(a.gate + at, g);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    float v = u[c * V + k];
                    if constexpr (POST) {
                        v = (v - mean) * inverse * w[k];
                        if (LAYER && a.post_bias != nullptr) v += b[k];
                    }
                    if (a.gate != nullptr) v *= g[k];
                    r[c * V + k] = fmaf(a.scale, v, r[c * V + k]);
                }
            }
            T* out = static_cast<T*>(a.r) + static_cast<uint64_t>(row) * d;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float v[V];
#pragma unroll
                for (int k = 0; k < V; ++k) v[k] = r[c * V + k];
                if (S::at(lane, c) < d) store_row<T, V>(out + S::at(lane, c), v);
            }
        }
        float mean = 0.0f;
        if constexpr (LAYER) {
            float s[1] = {0.0f};
#pragma unroll
            for (int e = 0; e < E; ++e) s[0] += r[e];
            row_sums<WPR, 1>(s, lds, step++);
            mean = s[0] * inv_d;
        }
        float s[1] = {0.0f};
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float z = S::at(lane, c) < d ? r[c * V + k] - mean : 0.0f;
                s[0] = fmaf(z, z, s[0]);
            }
        row_sums<WPR, 1>(s, lds, step++);
        const float inverse = rsqrtf(s[0] * inv_d + a.eps);
        T* h = static_cast<T*>(a.h) + static_cast<uint64_t>(row) * d;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const uint32_t at = S::at(lane, c);
            if (at >= d) continue;
            float w[V], b[V], v[V];
            load_param<V>(a.weight + at, w);
            if (LAYER && a.bias != nullptr) load_param<V>(a.bias + at, b);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                v[k] = (r[c * V + k] - mean) * inverse * w[k];
                if (LAYER && a.bias != nullptr) v[k] += b[k];
            }
            store_row<T, V>(h + at, v);
        }
        parity ^= 1;
    }
}

// Column sums of a block's rows stay in its threads' registers and go out once per block, as rows of partials
// [kNormGrads][blocks][d] in the order weight, bias, gate, post_weight, post_bias; column_sums_kernel adds them.
template <typename T, int V, int C, int WPR, int THREADS, bool LAYER, bool POST, bool GATE>
__global__ __launch_bounds__(THREADS) void residual_norm_back_kernel(NormBackward a) {
    constexpr int LANES = kWave * WPR, ROWS = THREADS / LANES, E = V * C;
    using S = Share<V, C, LANES>;
    __shared__ float lds[2 * kSteps][2 * WPR];
    extern __shared__ float rows_lds[];  // [ROWS][d] where ROWS > 1
    const uint32_t lane = threadIdx.x % LANES, d = a.d;
    const float inv_d = 1.0f / static_cast<float>(d);
    float sums[kNormGrads][E];
#pragma unroll
    for (int g = 0; g < kNormGrads; ++g)
#pragma unroll
        for (int e = 0; e < E; ++e) sums[g][e] = 0.0f;
    uint32_t parity = 0;
    for (uint32_t row = blockIdx.x * ROWS + threadIdx.x / LANES; row < a.n; row += gridDim.x * ROWS) {
        float r[E], g[E], f[E];  // r, then its normalised entries; gh, then gx; f, then its normalised entries
        const auto fill = [&](const void* from, uint64_t stride, float (&to)[E]) {
            const T* p = static_cast<const T*>(from) + static_cast<uint64_t>(row) * stride;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float v[V];
#pragma unroll
                for (int k = 0; k < V; ++k) v[k] = 0.0f;
                if (S::at(lane, c) < d) load_row<T, V>(p + S::at(lane, c), v);
#pragma unroll
                for (int k = 0; k < V; ++k) to[c * V + k] = v[k];
            }
        };
        fill(a.r, a.r_stride, r);
        fill(a.gh, a.gh_stride, g);
        if (POST || GATE) fill(a.f, a.f_stride, f);
        uint32_t step = parity * kSteps;
        float mean[2] = {0.0f, 0.0f}, inverse[2];
        if constexpr (LAYER) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                mean[0] += r[e];
                if (POST) mean[1] += f[e];
            }
            row_sums<WPR, 2>(mean, lds, step++);
            mean[0] *= inv_d;
            mean[1] *= inv_d;
        }
        float square[2] = {0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const bool in = S::at(lane, c) < d;
                r[c * V + k] = in ? r[c * V + k] - mean[0] : 0.0f;
                square[0] = fmaf(r[c * V + k], r[c * V + k], square[0]);
                if (POST) {
                    f[c * V + k] = in ? f[c * V + k] - mean[1] : 0.0f;
                    square[1] = fmaf(f[c * V + k], f[c * V + k], square[1]);
                }
            }
        row_sums<WPR, 2>(square, lds, step++);
        inverse[0] = rsqrtf(square[0] * inv_d + a.eps);
        inverse[1] = POST ? rsqrtf(square[1] * inv_d + a.eps) : 1.0f;
        // through the norm of r: g = inverse (gh w - hat mean(gh w hat) [- mean(gh w)]), and gr
        float along[2] = {0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float w[V];
#pragma unroll
            for (int k = 0; k < V; ++k) w[k] = 0.0f;
            if (S::at(lane, c) < d) load_param<V>(a.weight + S::at(lane, c), w);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const int e = c * V + k;
                r[e] *= inverse[0];
                if (POST) f[e] *= inverse[1];
                sums[0][e] = fmaf(g[e], r[e], sums[0][e]);
                if (LAYER) sums[1][e] += g[e];
                g[e] *= w[k];
                along[0] = fmaf(g[e], r[e], along[0]);
                along[1] += g[e];
            }
        }
        row_sums<WPR, 2>(along, lds, step++);
        along[0] *= inv_d;
        along[1] = LAYER ? along[1] * inv_d : 0.0f;
        float back[2] = {0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const uint32_t at = S::at(lane, c);
            if (at >= d) continue;
            float v[V], w[V], b[V], m[V];
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = 0.0f;
            if (a.gr != nullptr) load_row<T, V>(static_cast<const T*>(a.gr) + static_cast<uint64_t>(row) * a.gr_stride + at, v);
            if constexpr (POST) load_param<V>(a.post_weight + at, w);
            if (POST && LAYER && GATE && a.post_bias != nullptr) load_param<V>(a.post_bias + at, b);
            if constexpr (GATE) load_param<V>(a.gate + at, m);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const int e = c * V + k;
                v[k] += inverse[0] * (g[e] - r[e] * along[0] - along[1]);
                float gu = a.scale * v[k];
                if constexpr (GATE) {
                    float u = f[e];
                    if constexpr (POST) {
                        u *= w[k];
                        if (LAYER && a.post_bias != nullptr) u += b[k];
                    }
                    sums[2][e] = fmaf(gu, u, sums[2][e]);
                    gu *= m[k];
                }
                if constexpr (POST) {
                    sums[3][e] = fmaf(gu, f[e], sums[3][e]);
                    if (LAYER) sums[4][e] += gu;
                    gu *= w[k];
                    back[0] = fmaf(gu, f[e], back[0]);
                    back[1] += gu;
                }
                g[e] = gu;
            }
            store_row<T, V>(static_cast<T*>(a.gx) + static_cast<uint64_t>(row) * d + at, v);
        }
        if (a.gf != nullptr) {
            if constexpr (POST) {
                row_sums<WPR, 2>(back, lds, step++);
                back[0] *= inv_d;
                back[1] = LAYER ? back[1] * inv_d : 0.0f;
            }
            T* gf = static_cast<T*>(a.gf) + static_cast<uint64_t>(row) * d;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const uint32_t at = S::at(lane, c);
                if (at >= d) continue;
                float v[V];
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const int e = c * V + k;
                    v[k] = POST ? inverse[1] * (g[e] - f[e] * back[0] - back[1]) : g[e];
                }
                store_row<T, V>(gf + at, v);
            }
        }
        parity ^= 1;
    }
#pragma unroll
    for (int q = 0; q < kNormGrads; ++q) {
        const bool wanted = q == 0 || (q == 1 && LAYER) || (q == 2 && GATE) || (q == 3 && POST) || (q == 4 && POST && LAYER);
        if (!wanted) continue;
        float* out = a.partials + (static_cast<uint64_t>(q) * gridDim.x + blockIdx.x) * d;
        if constexpr (ROWS == 1) {
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (S::at(lane, c) < d)
#pragma unroll
                    for (int k = 0; k < V; ++k) out[S::at(lane, c) + k] = sums[q][c * V + k];
        } else {
            __syncthreads();  // the last gradient's rows are added up
            float* mine = rows_lds + threadIdx.x / LANES * d;
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (S::at(lane, c) < d)
#pragma unroll
                    for (int k = 0; k < V; ++k) mine[S::at(lane, c) + k] = sums[q][c * V + k];
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < d; i += THREADS) {
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < ROWS; ++w) sum += rows_lds[w * d + i];
                out[i] = sum;
            }
        }
    }
}

// out[q][i] = the sum over the blocks of partials[q][block][i], in a fixed order: 64 columns a block, a wave per 1/16 of
// the partial rows, the waves' sums in order.
constexpr int kColumnWaves = 16;
__global__ __launch_bounds__(kWave* kColumnWaves) void column_sums_kernel(const float* __restrict__ partials, NormGradients out, uint32_t rows,
                                                                         uint32_t d) {
    __shared__ float lds[kColumnWaves][kWave];
    float* const to = out.grad[blockIdx.y];
    if (to == nullptr) return;
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, column = blockIdx.x * kWave + lane;
    const float* from = partials + static_cast<uint64_t>(blockIdx.y) * rows * d;
    float sum = 0.0f;
    if (column < d)
        for (uint32_t row = wave; row < rows; row += kColumnWaves) sum += from[static_cast<uint64_t>(row) * d + column];
    lds[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && column < d) {
        sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kColumnWaves; ++w) sum += lds[w][lane];
        to[column] = sum;
    }
}

constexpr uint32_t kBackBlocks = 512;
// Waves that share a row: up to 16 entries a lane.
uint32_t norm_waves(uint32_t d) { return d <= 1024 ? 1 : d <= 4096 ? 4 : 16; }
uint32_t norm_rows(uint32_t d) { return norm_waves(d) == 1 ? 4 : 1; }

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
    const uint32_t waves = norm_waves(a.d), rows = norm_rows(a.d);
    const uint32_t blocks = (a.n + rows - 1) / rows;
    const dim3 grid(blocks < 4096 ? blocks : 4096);
    if (waves == 1) hipLaunchKernelGGL((residual_norm_kernel<T, V, 16 / V, 1, 256, LAYER, POST>), grid, dim3(256), 0, stream, a);
    else if (waves == 4) hipLaunchKernelGGL((residual_norm_kernel<T, V, 16 / V, 4, 256, LAYER, POST>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((residual_norm_kernel<T, V, 16 / V, 16, 1024, LAYER, POST>), grid, dim3(1024), 0, stream, a);
    return hipGetLastError();
}

template <typename T, int V, bool LAYER, bool POST, bool GATE>
hipError_t backward_widths(const NormBackward& a, hipStream_t stream) {
    const uint32_t waves = norm_waves(a.d), rows = norm_rows(a.d);
    const dim3 grid(norm_back_blocks(a.n, a.d));
    if (waves == 1)
        hipLaunchKernelGGL((residual_norm_back_kernel<T, V, 16 / V, 1, 256, LAYER, POST, GATE>), grid, dim3(256), rows * a.d * sizeof(float),
                           stream, a);
    else if (waves == 4)
        hipLaunchKernelGGL((residual_norm_back_kernel<T, V, 16 / V, 4, 256, LAYER, POST, GATE>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((residual_norm_back_kernel<T, V, 16 / V, 16, 1024, LAYER, POST, GATE>), grid, dim3(1024), 0, stream, a);
    return hipGetLastError();
}

template <typename T, int V>
hipError_t forward_kinds(const NormForward& a, hipStream_t stream) {
    const bool post = a.post_weight != nullptr;
    if (a.layer) return post ? forward_widths<T, V, true, true>(a, stream) : forward_widths<T, V, true, false>(a, stream);
    return post ? forward_widths<T, V, false, true>(a, stream) : forward_widths<T, V, false, false>(a, stream);
}

template <typename T, int V, bool LAYER>
hipError_t backward_kinds(const NormBackward& a, hipStream_t stream) {
    const bool post = a.post_weight != nullptr, gate = a.gate != nullptr;
    if (post) return gate ? backward_widths<T, V, LAYER, true, true>(a, stream) : backward_widths<T, V, LAYER, true, false>(a, stream);
    return gate ? backward_widths<T, V, LAYER, false, true>(a, stream) : backward_widths<T, V, LAYER, false, false>(a, stream);
}

}  // namespace

uint32_t norm_back_blocks(uint32_t n, uint32_t d) {
    const uint32_t rows = norm_rows(d), blocks = (n + rows - 1) / rows;
    return blocks < kBackBlocks ? blocks : kBackBlocks;
}

hipError_t launch_residual_norm(int vt, const NormForward& a, hipStream_t stream) {
    const bool whole = whole_pieces(vt, a.d, {a.x, a.f, a.r, a.h}, {a.x_stride, a.f_stride}, {a.weight, a.bias, a.gate, a.post_weight, a.post_bias});
    if (vt == kBF16) return whole ? forward_kinds<uint16_t, 8>(a, stream) : forward_kinds<uint16_t, 1>(a, stream);
    return whole ? forward_kinds<float, 4>(a, stream) : forward_kinds<float, 1>(a, stream);
}

hipError_t launch_residual_norm_backward(int vt, const NormBackward& a, const NormGradients& grads, hipStream_t stream) {
    const bool whole = whole_pieces(vt, a.d, {a.r, a.f, a.gr, a.gh, a.gx, a.gf}, {a.r_stride, a.f_stride, a.gr_stride, a.gh_stride},
                                    {a.weight, a.gate, a.post_weight, a.post_bias});
    hipError_t status;
    if (vt == kBF16) {
        if (whole) status = a.layer ? backward_kinds<uint16_t, 8, true>(a, stream) : backward_kinds<uint16_t, 8, false>(a, stream);
        else status = a.layer ? backward_kinds<uint16_t, 1, true>(a, stream) : backward_kinds<uint16_t, 1, false>(a, stream);
    } else {
        if (whole) status = a.layer ? backward_kinds<float, 4, true>(a, stream) : backward_kinds<float, 4, false>(a, stream);
        else status = a.layer ? backward_kinds<float, 1, true>(a, stream) : backward_kinds<float, 1, false>(a, stream);
    }
    if (status != hipSuccess) return status;
    hipLaunchKernelGGL(column_sums_kernel, dim3((a.d + kWave - 1) / kWave, kNormGrads), dim3(kWave * kColumnWaves), 0, stream, a.partials, grads,
                       norm_back_blocks(a.n, a.d), a.d);
    return hipGetLastError();
}

}  // namespace hffn
