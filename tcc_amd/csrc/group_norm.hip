// Group norm over the node rows of each graph, with its activation, channels
// last (include/tcc_training.h).
//
//   mean, var over the rows of segment b and the channels of group g
//   z = ((x - mean) * rstd) * weight + bias,  rstd = 1 / sqrt(var + eps)
//   y = act(z)
//
// and with dz = dY act'(z), xh = (x - mean) rstd, M values in the group:
//   dBias_c = sum dz,  dWeight_c = sum dz xh
//   dx = rstd (w dz - (S1 + xh S2) / M),  S1 = sum w dz,  S2 = sum w dz xh
//
// The rows are cut into tiles of equal length whatever the segments, so that
// one graph of millions of nodes and thousands of small ones spread over the
// GPU alike.  Tile t and segment s that share rows hold slot t + s: walking
// tiles and segments in order, one of the two moves on at every step, so the
// slots of all pairs are distinct and those of a segment are consecutive.
#include <algorithm>

#include "../../include/tcc_swtcf.h"
#include "../../include/tcc_training.h"
#include "primitives.hpp"
#include "row_types.hpp"

namespace tcc {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr std::uint32_t kMaxChannels = 4096;

struct Segments {
    const void* offsets;
    std::uint64_t N, B, each;  // rows of every segment where offsets is NULL
    std::uint32_t wide;        // int64 offsets

    // The first row of segment s (N for s = B), never outside [0, N].
    __device__ __forceinline__ std::uint64_t start(std::uint64_t s) const {
        if (offsets == nullptr) return s * each;
        const std::int64_t v = wide ? load_global<std::int64_t>(static_cast<const std::int64_t*>(offsets) + s)
                                    : load_global<std::int32_t>(static_cast<const std::int32_t*>(offsets) + s);
        return static_cast<std::uint64_t>(v < 0 ? 0 : min<std::uint64_t>(static_cast<std::uint64_t>(v), N));
    }
    // The last segment that starts at or before `row`, for row < N.
    __device__ __forceinline__ std::uint64_t find(std::uint64_t row) const {
        if (offsets == nullptr) return row / each;
        std::uint64_t lo = 0, hi = B;
        while (hi - lo > 1) {
            const std::uint64_t m = (lo + hi) / 2;
            if (start(m) <= row) lo = m;
            else hi = m;
        }
        return lo;
    }
};

struct NormArgs {
    Segments seg;
    const void *x, *dy, *weight, *bias;
    void* out;  // y, or dx
    float *mean, *rstd;
    float2* part;      // [slots][G]: mean and squared deviations, or S1 and S2
    float2* sums;      // [B][G]: S1 / M and S2 / M
    float2* channel;   // [tiles][C]: dBias and dWeight
    std::uint64_t ldx, lddy, ldo, tileRows;
    std::uint32_t C, G, K, colsV, rowLanes;  // K = C / G; colsV vectors a row, rowLanes rows at once
    std::uint32_t paramBytes, paramType, act;
    float eps;
};

__device__ __forceinline__ float param_at(const void* p, std::uint32_t type, std::uint32_t c, float none) {
    if (p == nullptr) return none;
    if (type == TCC_F32) return static_cast<const float*>(p)[c];
    if (type == TCC_BF16) return static_cast<float>(static_cast<const bf16_t*>(p)[c]);
    return static_cast<float>(static_cast<const f16_t*>(p)[c]);
}

// z with a rounding after each operation, in the forward as in the gradient.
__device__ __forceinline__ float normalise(float x, float mean, float rstd) {
#pragma clang fp contract(off)
    return (x - mean) * rstd;
}
__device__ __forceinline__ float affine(float xh, float w, float b) {
#pragma clang fp contract(off)
    const float m = xh * w;
    return m + b;
}

__device__ __forceinline__ float activate(std::uint32_t act, float z) {
    if (act == TCC_ACT_NONE) return z;
    if (act == TCC_ACT_RELU) return z > 0.0f ? z : z * 0.0f;  // keeps NaN
    if (act == TCC_ACT_SILU) return z / (1.0f + expf(-z));
    return z * (0.5f * (1.0f + erff(z * 0.70710678f)));
}

__device__ __forceinline__ float slope(std::uint32_t act, float z) {
    if (act == TCC_ACT_NONE) return 1.0f;
    if (act == TCC_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
    if (act == TCC_ACT_SILU) {
        const float p = 1.0f / (1.0f + expf(-z));
        return p * (1.0f + z * (1.0f - p));
    }
    return 0.5f * (1.0f + erff(z * 0.70710678f)) + z * expf(-0.5f * z * z) * 0.39894228f;
}

// Rows a, a + rowLanes, ... below b that a row lane takes.
__device__ __forceinline__ std::uint32_t lane_rows(std::uint64_t a, std::uint64_t b, std::uint32_t rl,
                                                   std::uint32_t rowLanes) {
    return a + rl < b ? static_cast<std::uint32_t>((b - a - rl + rowLanes - 1) / rowLanes) : 0u;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, kWave);
    return v;
}

// ---------------------------------------------------------------- statistics

constexpr int kBatch = 4;  // rows whose deviations are taken from their own mean

// The mean and squared deviations of each segment's rows in a tile, group by
// group.  A lane takes a few rows at a time in registers and forms their mean
// and their deviations from it, then joins them with those before: no
// difference of large sums, whatever the mean.
template <typename T, int N>
__global__ void __launch_bounds__(kThreads) stats_kernel(NormArgs a) {
    extern __shared__ float lds[];
    float* ldsMean = lds;
    float* ldsDev = lds + a.rowLanes * a.C;
    const std::uint64_t t = blockIdx.x;
    const std::uint64_t lo = t * a.tileRows, hi = min(lo + a.tileRows, a.seg.N);
    const std::uint32_t rl = threadIdx.x / a.colsV;
    const std::uint32_t cv0 = a.colsV > kThreads ? threadIdx.x : threadIdx.x - rl * a.colsV;
    const bool active = a.colsV > kThreads || rl < a.rowLanes;
    const std::uint32_t row = a.colsV > kThreads ? 0u : rl;
    const T* x = static_cast<const T*>(a.x);
    for (std::uint64_t s = a.seg.find(lo); s < a.seg.B; ++s) {
        const std::uint64_t first = max(a.seg.start(s), lo), end = min(a.seg.start(s + 1), hi);
        if (a.seg.start(s) >= hi) break;
        if (first >= end) continue;
        if (active) {
            for (std::uint32_t cv = cv0; cv < a.colsV; cv += kThreads) {
                vec_t<float, N> mean(0.0f), dev(0.0f);
                float count = 0.0f;
                for (std::uint64_t r = first + row; r < end; r += kBatch * a.rowLanes) {
                    vec_t<float, N> v[kBatch];
                    int got = 0;
#pragma unroll
                    for (int u = 0; u < kBatch; ++u) {
                        const std::uint64_t q = r + static_cast<std::uint64_t>(u) * a.rowLanes;
                        v[u] = vec_t<float, N>(0.0f);
                        if (q < end) {
                            v[u] = load_row<T, N>(x + q * a.ldx + cv * N);
                            got = u + 1;
                        }
                    }
                    const float inv = 1.0f / static_cast<float>(got);
                    vec_t<float, N> m = v[0];
#pragma unroll
                    for (int u = 1; u < kBatch; ++u) m += v[u];
                    m *= inv;
                    vec_t<float, N> d(0.0f);
#pragma unroll
                    for (int u = 0; u < kBatch; ++u) {
                        const vec_t<float, N> e = u < got ? v[u] - m : vec_t<float, N>(0.0f);
                        d += e * e;
                    }
                    const float all = count + static_cast<float>(got);
                    const float share = static_cast<float>(got) / all;
                    const vec_t<float, N> gap = m - mean;
                    mean += gap * share;
                    dev += d + gap * gap * (count * share);
                    count = all;
                }
#pragma unroll
                for (int q = 0; q < N; ++q) {
                    ldsMean[row * a.C + cv * N + q] = mean[q];
                    ldsDev[row * a.C + cv * N + q] = dev[q];
                }
            }
        }
        __syncthreads();
        const float total = static_cast<float>(end - first) * static_cast<float>(a.K);
        for (std::uint32_t g = threadIdx.x / kWave; g < a.G; g += kWaves) {
            const std::uint32_t entries = a.rowLanes * a.K;
            float sum = 0.0f;
            for (std::uint32_t e = __lane_id(); e < entries; e += kWave) {
                const std::uint32_t r = e / a.K, c = g * a.K + (e - r * a.K);
                const std::uint32_t n = lane_rows(first, end, r, a.rowLanes);
                if (n > 0) sum += static_cast<float>(n) * ldsMean[r * a.C + c];
            }
            const float mean = wave_sum(sum) / total;
            float dev = 0.0f;
            for (std::uint32_t e = __lane_id(); e < entries; e += kWave) {
                const std::uint32_t r = e / a.K, c = g * a.K + (e - r * a.K);
                const std::uint32_t n = lane_rows(first, end, r, a.rowLanes);
                if (n > 0) {
                    const float gap = ldsMean[r * a.C + c] - mean;
                    dev += ldsDev[r * a.C + c] + static_cast<float>(n) * gap * gap;
                }
            }
            dev = wave_sum(dev);
            if (__lane_id() == 0) a.part[(t + s) * a.G + g] = float2{mean, dev};
        }
        __syncthreads();
    }
}

// The rows that slot p of segment s holds.
__device__ __forceinline__ float slot_rows(const NormArgs& a, std::uint64_t t, std::uint64_t first, std::uint64_t end) {
    const std::uint64_t lo = max(t * a.tileRows, first), hi = min((t + 1) * a.tileRows, end);
    return static_cast<float>(hi - lo);
}

// The sum of a workgroup's values, in the same order every time.
template <int W>
__device__ __forceinline__ float group_sum(float v, float* red) {
    v = wave_sum(v);
    if (W == 1) return v;
    if (__lane_id() == 0) red[threadIdx.x / kWave] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) s += red[w];
    __syncthreads();
    return s;
}

// mean and rstd of one segment's group from its slots.
template <int W>
__global__ void __launch_bounds__(kWave* W) stats_join_kernel(NormArgs a) {
    __shared__ float red[W];
    const std::uint64_t s = blockIdx.x / a.G;
    const std::uint32_t g = blockIdx.x - static_cast<std::uint32_t>(s * a.G);
    const std::uint64_t first = a.seg.start(s), end = a.seg.start(s + 1);
    float mean = 0.0f, var = 0.0f;
    if (first < end) {
        const std::uint64_t t0 = first / a.tileRows, t1 = (end - 1) / a.tileRows;
        const float rows = static_cast<float>(end - first);
        float sum = 0.0f;
        for (std::uint64_t t = t0 + threadIdx.x; t <= t1; t += kWave * W)
            sum += a.part[(t + s) * a.G + g].x * slot_rows(a, t, first, end);
        mean = group_sum<W>(sum, red) / rows;
        float dev = 0.0f;
        for (std::uint64_t t = t0 + threadIdx.x; t <= t1; t += kWave * W) {
            const float2 p = a.part[(t + s) * a.G + g];
            const float gap = p.x - mean;
            dev += p.y + gap * gap * slot_rows(a, t, first, end) * static_cast<float>(a.K);
        }
        var = group_sum<W>(dev, red) / (rows * static_cast<float>(a.K));
    }
    if (threadIdx.x == 0) {
        a.mean[s * a.G + g] = mean;
        a.rstd[s * a.G + g] = 1.0f / sqrtf(var + a.eps);
    }
}

// ---------------------------------------------------------------- output

template <typename T, int N>
__global__ void __launch_bounds__(kThreads) apply_kernel(NormArgs a) {
    const std::uint64_t lo = blockIdx.x * a.tileRows, hi = min(lo + a.tileRows, a.seg.N);
    const std::uint32_t rl = threadIdx.x / a.colsV;
    const std::uint32_t cv0 = a.colsV > kThreads ? threadIdx.x : threadIdx.x - rl * a.colsV;
    if (a.colsV <= kThreads && rl >= a.rowLanes) return;
    const std::uint32_t row = a.colsV > kThreads ? 0u : rl;
    const T* x = static_cast<const T*>(a.x);
    T* y = static_cast<T*>(a.out);
    const std::uint64_t s0 = a.seg.find(lo);
    for (std::uint32_t cv = cv0; cv < a.colsV; cv += kThreads) {
        float w[N], b[N];
        std::uint32_t g[N];
#pragma unroll
        for (int q = 0; q < N; ++q) {
            w[q] = param_at(a.weight, a.paramType, cv * N + q, 1.0f);
            b[q] = param_at(a.bias, a.paramType, cv * N + q, 0.0f);
            g[q] = (cv * N + q) / a.K;
        }
        for (std::uint64_t s = s0; s < a.seg.B; ++s) {
            const std::uint64_t first = max(a.seg.start(s), lo), end = min(a.seg.start(s + 1), hi);
            if (a.seg.start(s) >= hi) break;
            if (first >= end) continue;
            float mean[N], rstd[N];
#pragma unroll
            for (int q = 0; q < N; ++q) {
                mean[q] = a.mean[s * a.G + g[q]];
                rstd[q] = a.rstd[s * a.G + g[q]];
            }
#pragma unroll 4
            for (std::uint64_t r = first + row; r < end; r += a.rowLanes) {
                const vec_t<float, N> v = load_row<T, N>(x + r * a.ldx + cv * N);
                vec_t<float, N> o;
#pragma unroll
                for (int q = 0; q < N; ++q) o[q] = activate(a.act, affine(normalise(v[q], mean[q], rstd[q]), w[q], b[q]));
                store_row<T, N>(y + r * a.ldo + cv * N, o);
            }
        }
    }
}

// ---------------------------------------------------------------- gradient

// S1 and S2 of each segment's rows in a tile, and the tile's dBias and
// dWeight.  LDS: the segment's sums and the tile's, a place for each lane.
template <typename T, int N>
__global__ void __launch_bounds__(kThreads) grad_sums_kernel(NormArgs a) {
    extern __shared__ float lds[];
    const std::uint32_t plane = a.rowLanes * a.C;
    float *seg1 = lds, *seg2 = lds + plane, *all1 = lds + 2 * plane, *all2 = lds + 3 * plane;
    const std::uint64_t t = blockIdx.x;
    const std::uint64_t lo = t * a.tileRows, hi = min(lo + a.tileRows, a.seg.N);
    const std::uint32_t rl = threadIdx.x / a.colsV;
    const std::uint32_t cv0 = a.colsV > kThreads ? threadIdx.x : threadIdx.x - rl * a.colsV;
    const bool active = a.colsV > kThreads || rl < a.rowLanes;
    const std::uint32_t row = a.colsV > kThreads ? 0u : rl;
    const T* x = static_cast<const T*>(a.x);
    const T* dy = static_cast<const T*>(a.dy);
    for (std::uint32_t i = threadIdx.x; i < 2 * plane; i += kThreads) all1[i] = 0.0f;
    __syncthreads();
    for (std::uint64_t s = a.seg.find(lo); s < a.seg.B; ++s) {
        const std::uint64_t first = max(a.seg.start(s), lo), end = min(a.seg.start(s + 1), hi);
        if (a.seg.start(s) >= hi) break;
        if (first >= end) continue;
        if (active) {
            for (std::uint32_t cv = cv0; cv < a.colsV; cv += kThreads) {
                float w[N], b[N], mean[N], rstd[N];
                vec_t<float, N> s1(0.0f), s2(0.0f);
#pragma unroll
                for (int q = 0; q < N; ++q) {
                    const std::uint32_t c = cv * N + q;
                    w[q] = param_at(a.weight, a.paramType, c, 1.0f);
                    b[q] = param_at(a.bias, a.paramType, c, 0.0f);
                    mean[q] = a.mean[s * a.G + c / a.K];
                    rstd[q] = a.rstd[s * a.G + c / a.K];
                }
#pragma unroll 4
                for (std::uint64_t r = first + row; r < end; r += a.rowLanes) {
                    const vec_t<float, N> v = load_row<T, N>(x + r * a.ldx + cv * N);
                    const vec_t<float, N> d = load_row<T, N>(dy + r * a.lddy + cv * N);
#pragma unroll
                    for (int q = 0; q < N; ++q) {
                        const float xh = normalise(v[q], mean[q], rstd[q]);
                        const float dz = d[q] * slope(a.act, affine(xh, w[q], b[q]));
                        s1[q] += dz;
                        s2[q] += dz * xh;
                    }
                }
#pragma unroll
                for (int q = 0; q < N; ++q) {
                    const std::uint32_t at = row * a.C + cv * N + q;
                    all1[at] += s1[q];
                    all2[at] += s2[q];
                    seg1[at] = s1[q] * w[q];
                    seg2[at] = s2[q] * w[q];
                }
            }
        }
        __syncthreads();
        for (std::uint32_t g = threadIdx.x / kWave; g < a.G; g += kWaves) {
            float s1 = 0.0f, s2 = 0.0f;
            for (std::uint32_t e = __lane_id(); e < a.rowLanes * a.K; e += kWave) {
                const std::uint32_t r = e / a.K, c = g * a.K + (e - r * a.K);
                s1 += seg1[r * a.C + c];
                s2 += seg2[r * a.C + c];
            }
            s1 = wave_sum(s1);
            s2 = wave_sum(s2);
            if (__lane_id() == 0) a.part[(t + s) * a.G + g] = float2{s1, s2};
        }
        __syncthreads();
    }
    for (std::uint32_t c = threadIdx.x; c < a.C; c += kThreads) {
        float s1 = 0.0f, s2 = 0.0f;
        for (std::uint32_t r = 0; r < a.rowLanes; ++r) {
            s1 += all1[r * a.C + c];
            s2 += all2[r * a.C + c];
        }
        a.channel[t * a.C + c] = float2{s1, s2};
    }
}

// S1 / M and S2 / M of one segment's group from its slots.
template <int W>
__global__ void __launch_bounds__(kWave* W) grad_join_kernel(NormArgs a) {
    __shared__ float red[W];
    const std::uint64_t s = blockIdx.x / a.G;
    const std::uint32_t g = blockIdx.x - static_cast<std::uint32_t>(s * a.G);
    const std::uint64_t first = a.seg.start(s), end = a.seg.start(s + 1);
    if (first >= end) return;
    const std::uint64_t t0 = first / a.tileRows, t1 = (end - 1) / a.tileRows;
    float s1 = 0.0f, s2 = 0.0f;
    for (std::uint64_t t = t0 + threadIdx.x; t <= t1; t += kWave * W) {
        const float2 p = a.part[(t + s) * a.G + g];
        s1 += p.x;
        s2 += p.y;
    }
    s1 = group_sum<W>(s1, red);
    s2 = group_sum<W>(s2, red);
    const float size = static_cast<float>(end - first) * static_cast<float>(a.K);
    if (threadIdx.x == 0) a.sums[s * a.G + g] = float2{s1 / size, s2 / size};
}

// dBias and dWeight from the tiles' sums: 16 columns a workgroup, 16 threads
// a column.
constexpr std::uint32_t kParamCols = 16;
__global__ void __launch_bounds__(kThreads) param_grad_kernel(const float2* channel, std::uint64_t tiles, std::uint32_t C,
                                                             float* dWeight, float* dBias) {
    __shared__ float2 red[kThreads];
    const std::uint32_t c = blockIdx.x * kParamCols + threadIdx.x % kParamCols;
    float2 s{0.0f, 0.0f};
    if (c < C) {
#pragma unroll 4
        for (std::uint64_t t = threadIdx.x / kParamCols; t < tiles; t += kThreads / kParamCols) {
            const float2 p = channel[t * C + c];
            s.x += p.x;
            s.y += p.y;
        }
    }
    red[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x < kParamCols && c < C) {
        for (std::uint32_t i = 1; i < kThreads / kParamCols; ++i) {
            s.x += red[i * kParamCols + threadIdx.x].x;
            s.y += red[i * kParamCols + threadIdx.x].y;
        }
        if (dBias != nullptr) dBias[c] = s.x;
        if (dWeight != nullptr) dWeight[c] = s.y;
    }
}

template <typename T, int N>
__global__ void __launch_bounds__(kThreads) grad_apply_kernel(NormArgs a) {
    const std::uint64_t lo = blockIdx.x * a.tileRows, hi = min(lo + a.tileRows, a.seg.N);
    const std::uint32_t rl = threadIdx.x / a.colsV;
    const std::uint32_t cv0 = a.colsV > kThreads ? threadIdx.x : threadIdx.x - rl * a.colsV;
    if (a.colsV <= kThreads && rl >= a.rowLanes) return;
    const std::uint32_t row = a.colsV > kThreads ? 0u : rl;
    const T* x = static_cast<const T*>(a.x);
    const T* dy = static_cast<const T*>(a.dy);
    T* dx = static_cast<T*>(a.out);
    const std::uint64_t s0 = a.seg.find(lo);
    for (std::uint32_t cv = cv0; cv < a.colsV; cv += kThreads) {
        float w[N], b[N];
        std::uint32_t g[N];
#pragma unroll
        for (int q = 0; q < N; ++q) {
            w[q] = param_at(a.weight, a.paramType, cv * N + q, 1.0f);
            b[q] = param_at(a.bias, a.paramType, cv * N + q, 0.0f);
            g[q] = (cv * N + q) / a.K;
        }
        for (std::uint64_t s = s0; s < a.seg.B; ++s) {
            const std::uint64_t first = max(a.seg.start(s), lo), end = min(a.seg.start(s + 1), hi);
            if (a.seg.start(s) >= hi) break;
            if (first >= end) continue;
            float mean[N], rstd[N];
            float2 m[N];
#pragma unroll
            for (int q = 0; q < N; ++q) {
                mean[q] = a.mean[s * a.G + g[q]];
                rstd[q] = a.rstd[s * a.G + g[q]];
                m[q] = a.sums[s * a.G + g[q]];
            }
#pragma unroll 4
            for (std::uint64_t r = first + row; r < end; r += a.rowLanes) {
                const vec_t<float, N> v = load_row<T, N>(x + r * a.ldx + cv * N);
                const vec_t<float, N> d = load_row<T, N>(dy + r * a.lddy + cv * N);
                vec_t<float, N> o;
#pragma unroll
                for (int q = 0; q < N; ++q) {
                    const float xh = normalise(v[q], mean[q], rstd[q]);
                    const float dz = d[q] * slope(a.act, affine(xh, w[q], b[q]));
                    o[q] = (dz * w[q] - m[q].x - xh * m[q].y) * rstd[q];
                }
                store_row<T, N>(dx + r * a.ldo + cv * N, o);
            }
        }
    }
}

// ---------------------------------------------------------------- host side

constexpr std::size_t align16(std::size_t b) { return (b + 15) & ~std::size_t(15); }

// Tiles of at most this many, so that the tiles' sums stay few.
constexpr std::uint64_t kTiles = 2048;

struct Layout {
    std::uint64_t tileRows, tiles;
    std::size_t part, sums, channel, bytes;
    Layout(const tcc_group_norm_shape& s, bool backward) {
        // at least 32 rows of a tile, however narrow the rows: a tile's own
        // reductions cost about as much
        tileRows = std::max<std::uint64_t>((s.N + kTiles - 1) / kTiles, 32);
        tiles = (s.N + tileRows - 1) / tileRows;
        part = 0;
        std::size_t at = align16((tiles + s.B) * s.G * sizeof(float2));
        sums = at;
        channel = at;
        if (backward) {
            at += align16(s.B * s.G * sizeof(float2));
            channel = at;
            at += align16(tiles * s.C * sizeof(float2));
        }
        bytes = at;
    }
};

int check_shape(const tcc_group_norm_shape* s) {
    TCC_REQUIRE(s != nullptr, TCC_ERR_INVALID_ARGUMENT, "group norm: no shape");
    TCC_REQUIRE(s->G >= 1 && s->C >= 1 && s->C % s->G == 0, TCC_ERR_INVALID_ARGUMENT,
                "group norm: the groups have to divide the channels");
    TCC_REQUIRE(s->C <= kMaxChannels, TCC_ERR_UNSUPPORTED, "group norm: at most 4096 channels");
    TCC_REQUIRE(dtype_bytes(s->dtype) != 0 && dtype_bytes(s->paramDtype) != 0, TCC_ERR_INVALID_ARGUMENT,
                "group norm tensors are fp32, bf16 or fp16");
    TCC_REQUIRE(s->activation <= TCC_ACT_GELU, TCC_ERR_INVALID_ARGUMENT, "group norm: unknown activation");
    TCC_REQUIRE(s->offsets == nullptr || s->offsetBytes == 4 || s->offsetBytes == 8, TCC_ERR_INVALID_ARGUMENT,
                "group norm offsets are int32 or int64");
    TCC_REQUIRE(s->offsets != nullptr || (s->B == 0 ? s->N == 0 : s->N % s->B == 0), TCC_ERR_INVALID_ARGUMENT,
                "group norm: segments without offsets have the same number of rows");
    TCC_REQUIRE(s->offsets == nullptr || s->B > 0 || s->N == 0, TCC_ERR_INVALID_ARGUMENT,
                "group norm: rows without a segment");
    TCC_REQUIRE(s->eps >= 0.0f, TCC_ERR_INVALID_ARGUMENT, "group norm: eps is not negative");
    TCC_REQUIRE(s->N < (1ull << 40) && s->B <= 0x7FFFFFFFull / s->G, TCC_ERR_UNSUPPORTED, "group norm: too many rows");
    return TCC_OK;
}

template <typename T, int N>
int forward_launch(NormArgs a, const Layout& lay, std::uint64_t B, hipStream_t st) {
    a.colsV = a.C / N;
    a.rowLanes = std::max<std::uint32_t>(1, kThreads / a.colsV);
    const unsigned tiles = static_cast<unsigned>(lay.tiles);
    if (tiles > 0) {
        hipLaunchKernelGGL((stats_kernel<T, N>), dim3(tiles), dim3(kThreads), 2 * a.rowLanes * a.C * sizeof(float), st, a);
        TCC_LAUNCH_CHECK();
    }
    const unsigned groups = static_cast<unsigned>(B * a.G);
    if (lay.tiles > 64 * B) hipLaunchKernelGGL(stats_join_kernel<4>, dim3(groups), dim3(4 * kWave), 0, st, a);
    else hipLaunchKernelGGL(stats_join_kernel<1>, dim3(groups), dim3(kWave), 0, st, a);
    TCC_LAUNCH_CHECK();
    if (tiles > 0) {
        hipLaunchKernelGGL((apply_kernel<T, N>), dim3(tiles), dim3(kThreads), 0, st, a);
        TCC_LAUNCH_CHECK();
    }
    return TCC_OK;
}

template <typename T, int N>
int backward_launch(NormArgs a, const Layout& lay, std::uint64_t B, float* dWeight, float* dBias, hipStream_t st) {
    a.colsV = a.C / N;
    a.rowLanes = std::max<std::uint32_t>(1, kThreads / a.colsV);
    const unsigned tiles = static_cast<unsigned>(lay.tiles);
    if (tiles > 0) {
        hipLaunchKernelGGL((grad_sums_kernel<T, N>), dim3(tiles), dim3(kThreads), 4 * a.rowLanes * a.C * sizeof(float), st,
                           a);
        TCC_LAUNCH_CHECK();
        const unsigned groups = static_cast<unsigned>(B * a.G);
        if (lay.tiles > 64 * B) hipLaunchKernelGGL(grad_join_kernel<4>, dim3(groups), dim3(4 * kWave), 0, st, a);
        else hipLaunchKernelGGL(grad_join_kernel<1>, dim3(groups), dim3(kWave), 0, st, a);
        TCC_LAUNCH_CHECK();
    }
    if (dWeight != nullptr || dBias != nullptr) {
        hipLaunchKernelGGL(param_grad_kernel, dim3((a.C + kParamCols - 1) / kParamCols), dim3(kThreads), 0, st, a.channel,
                           lay.tiles, a.C, dWeight, dBias);
        TCC_LAUNCH_CHECK();
    }
    if (tiles > 0) {
        hipLaunchKernelGGL((grad_apply_kernel<T, N>), dim3(tiles), dim3(kThreads), 0, st, a);
        TCC_LAUNCH_CHECK();
    }
    return TCC_OK;
}

NormArgs base_args(const tcc_group_norm_shape& s, const Layout& lay, void* workspace) {
    NormArgs a{};
    a.seg = Segments{s.offsets, s.N, s.B, s.B > 0 ? s.N / s.B : 0, s.offsetBytes == 8};
    if (s.offsets == nullptr && a.seg.each == 0) a.seg.each = 1;  // no rows: never read
    char* ws = static_cast<char*>(workspace);
    a.part = reinterpret_cast<float2*>(ws + lay.part);
    a.sums = reinterpret_cast<float2*>(ws + lay.sums);
    a.channel = reinterpret_cast<float2*>(ws + lay.channel);
    a.tileRows = lay.tileRows;
    a.C = s.C;
    a.G = s.G;
    a.K = s.C / s.G;
    a.paramType = s.paramDtype;
    a.act = s.activation;
    a.eps = s.eps;
    return a;
}

#define TCC_BY_WIDTH(T, MAXN, width, CALL)            \
    do {                                              \
        if ((MAXN) >= 8 && (width) >= 8) {            \
            constexpr int N = (MAXN) >= 8 ? 8 : 1;    \
            return CALL(T, N);                        \
        }                                             \
        if ((width) >= 4) return CALL(T, 4);          \
        if ((width) >= 2) return CALL(T, 2);          \
        return CALL(T, 1);                            \
    } while (0)

}  // namespace
}  // namespace tcc

using namespace tcc;

extern "C" {

size_t tcc_group_norm_workspace_bytes(const tcc_group_norm_shape* s, int backward) {
    if (check_shape(s) != TCC_OK) return 0;
    return Layout(*s, backward != 0).bytes;
}

int tcc_group_norm(const tcc_group_norm_shape* s, const void* x, uint64_t ldx, const void* weight, const void* bias,
                   void* y, uint64_t ldy, float* mean, float* rstd, void* workspace, size_t workspaceBytes,
                   void* stream) {
    if (const int rc = check_shape(s)) return rc;
    const Layout lay(*s, false);
    TCC_REQUIRE((s->N == 0 || (x && y)) && ldx >= s->C && ldy >= s->C && (s->B == 0 || (mean && rstd)),
                TCC_ERR_INVALID_ARGUMENT, "invalid group norm arguments");
    TCC_REQUIRE((workspace || lay.bytes == 0) && workspaceBytes >= lay.bytes &&
                    reinterpret_cast<std::uintptr_t>(workspace) % 16 == 0,
                TCC_ERR_INVALID_ARGUMENT, "group norm workspace too small or unaligned (tcc_group_norm_workspace_bytes)");
    if (s->B == 0) return TCC_OK;
    NormArgs a = base_args(*s, lay, workspace);
    a.x = x;
    a.ldx = ldx;
    a.weight = weight;
    a.bias = bias;
    a.out = y;
    a.ldo = ldy;
    a.mean = mean;
    a.rstd = rstd;
    const std::uint32_t w = RowWidth(s->C, dtype_bytes(s->dtype)).with(x).with(y).stride(ldx).stride(ldy).elems();
    const hipStream_t st = as_stream(stream);
#define CALL(T, N) (forward_launch<T, N>(a, lay, s->B, st))
    if (s->dtype == TCC_F32) TCC_BY_WIDTH(float, 4, w, CALL);
    if (s->dtype == TCC_BF16) TCC_BY_WIDTH(bf16_t, 8, w, CALL);
    TCC_BY_WIDTH(f16_t, 8, w, CALL);
#undef CALL
}

int tcc_group_norm_grad(const tcc_group_norm_shape* s, const void* dY, uint64_t lddy, const void* x, uint64_t ldx,
                        const float* mean, const float* rstd, const void* weight, const void* bias, void* dX,
                        uint64_t lddx, float* dWeight, float* dBias, void* workspace, size_t workspaceBytes,
                        void* stream) {
    if (const int rc = check_shape(s)) return rc;
    const Layout lay(*s, true);
    TCC_REQUIRE((s->N == 0 || (dY && x && dX)) && lddy >= s->C && ldx >= s->C && lddx >= s->C &&
                    (s->B == 0 || (mean && rstd)),
                TCC_ERR_INVALID_ARGUMENT, "invalid group norm gradient arguments");
    TCC_REQUIRE((workspace || lay.bytes == 0) && workspaceBytes >= lay.bytes &&
                    reinterpret_cast<std::uintptr_t>(workspace) % 16 == 0,
                TCC_ERR_INVALID_ARGUMENT, "group norm workspace too small or unaligned (tcc_group_norm_workspace_bytes)");
    NormArgs a = base_args(*s, lay, workspace);
    a.x = x;
    a.ldx = ldx;
    a.dy = dY;
    a.lddy = lddy;
    a.weight = weight;
    a.bias = bias;
    a.out = dX;
    a.ldo = lddx;
    a.mean = const_cast<float*>(mean);
    a.rstd = const_cast<float*>(rstd);
    const std::uint32_t w = RowWidth(s->C, dtype_bytes(s->dtype)).with(dY).with(x).with(dX).stride(lddy).stride(ldx)
                                .stride(lddx).elems();
    const hipStream_t st = as_stream(stream);
#define CALL(T, N) (backward_launch<T, N>(a, lay, s->B, dWeight, dBias, st))
    if (s->dtype == TCC_F32) TCC_BY_WIDTH(float, 4, w, CALL);
    if (s->dtype == TCC_BF16) TCC_BY_WIDTH(bf16_t, 8, w, CALL);
    TCC_BY_WIDTH(f16_t, 8, w, CALL);
#undef CALL
}

}  // extern "C"
