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
// Segments that a workgroup can walk in good time go whole, statistics and
// output (or sums and dx) in one kernel whose second reading the caches mostly
// serve.  The rows of longer ones are cut into tiles of equal length, whatever
// the segments, so that they spread over the GPU, and their statistics, the
// joining of these and the output are kernels one after the other: memory is
// read twice, as a statistic of all rows comes before the first output.  Both
// kinds can be in one batch, which only the device knows: each kernel passes
// over the segments of the other kind, and the tiles' end at once where the
// whole segments' workgroups saw none of theirs.  Tile t and segment s that
// share rows hold slot t + s: walking tiles and segments in order, one of the
// two moves on at every step, so the slots of all pairs are distinct and those
// of a segment are consecutive.
//
// What bounds it: memory.  One segment of 2.45M x 256 fp32 rows takes 1,240 us
// forward (7.5 GB, 6.1 TB/s: the statistics 385, the output 852) and 2,000 us
// backward (12.5 GB, 6.2 TB/s: the sums 731, dx 1,292); bf16 rows 690 and 1,140
// (3.8 and 6.3 GB, 5.5 TB/s).  2,000 ragged graphs of 169,000 x 128 bf16 rows
// together, 130 MB, take 82 us backward with gelu: 61 in the whole segments'
// kernel, half of it vector instructions, 8 in dWeight's and 14 in three empty
// launches, which a caller who knows the longest graph is spared.
#include <algorithm>

#include "../../include/tcc_swtcf.h"
#include "../../include/tcc_training.h"
#include "activations.hpp"
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
    // The last segment that starts at or before `row` (0 if there is none),
    // for row < N (so that segments of one size have rows), by a whole wave:
    // 64 starts a round.
    __device__ __forceinline__ std::uint64_t find(std::uint64_t row) const {
        if (offsets == nullptr) return row / each;
        std::uint64_t lo = 0, hi = B;  // start(lo) <= row < start(hi), or lo = 0
        while (hi - lo > 1) {
            const std::uint64_t step = (hi - lo + kWave - 1) / kWave;
            const std::uint64_t m = lo + (__lane_id() + 1) * step;
            const std::uint64_t above = __ballot(m >= hi || start(m) > row);
            const std::uint64_t k = above == 0 ? kWave : __builtin_ctzll(above);
            hi = min(lo + (k + 1) * step, hi);
            lo += k * step;
        }
        return lo;
    }
    // Segments of more rows than this go tile by tile, the others whole.
    std::uint64_t longest;
    __device__ __forceinline__ bool whole(std::uint64_t s) const { return start(s + 1) - start(s) <= longest; }
};

struct NormArgs {
    Segments seg;
    const void *x, *dy, *weight, *bias;
    void* out;  // y, or dx
    float *mean, *rstd;
    float2* part;      // [slots][G]: mean and squared deviations, or S1 and S2
    float2* sums;      // [B][G]: S1 / M and S2 / M
    float2* channel;   // [wholeRows + tiles][C]: dBias and dWeight
    std::uint8_t* seen;  // [kWholeBlocks]: whether a whole segments' workgroup met one that goes by tiles
    std::uint32_t seenCount;  // those workgroups; 0: tiles alone
    std::uint64_t ldx, lddy, ldo, tileRows, outRows;  // rows of a tile of the sums, and of the output
    std::uint32_t C, G, K, colsV, rowLanes;  // K = C / G; colsV vectors a row, rowLanes rows at once
    std::uint32_t paramType, act;
    float eps;
};

// Rows a, a + rowLanes, ... below b that a row lane takes.
__device__ __forceinline__ std::uint32_t lane_rows(std::uint64_t a, std::uint64_t b, std::uint32_t rl,
                                                   std::uint32_t rowLanes) {
    return a + rl < b ? static_cast<std::uint32_t>((b - a - rl + rowLanes - 1) / rowLanes) : 0u;
}

// Whether the tiles have anything to do, for a whole workgroup.
__device__ __forceinline__ bool tiles_needed(const std::uint8_t* seen, std::uint32_t count) {
    if (count == 0) return true;
    std::uint32_t any = 0;
    for (std::uint32_t i = threadIdx.x * 16; i < count; i += blockDim.x * 16) {
        const vu4 v = load_global<vu4>(seen + i);
        any |= v[0] | v[1] | v[2] | v[3];
    }
    return __syncthreads_or(static_cast<int>(any)) != 0;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, kWave);
    return v;
}

// Rows of tiles are read past the caches' order: read as usual, 2.45M x 256 fp32
// rows took 479 us for the statistics instead of 400, and their gradient's
// sums 843 instead of 747.
template <typename T, int N>
__device__ __forceinline__ vec_t<float, N> load_once(const T* p) {
    using V = vec_t<T, N>;
    const auto* g = (const __attribute__((address_space(1))) V*)(reinterpret_cast<std::uintptr_t>(p));
    return __builtin_convertvector(__builtin_nontemporal_load(g), vec_t<float, N>);
}

// What the channels c .. c + N need of their groups' values: one of each where
// a vector lies in one group (N divides K), as it mostly does.
template <int N>
struct OfGroups {
    float mean[N], rstd[N];
    float2 sums[N];
    template <bool SUMS>
    __device__ __forceinline__ void load(const NormArgs& a, std::uint64_t s, std::uint32_t c) {
        const std::uint32_t g = c / a.K;
        const std::uint64_t at = s * a.G + g;
        const float m0 = a.mean[at], r0 = a.rstd[at];
        float2 s0{0.0f, 0.0f};
        if (SUMS) s0 = a.sums[at];
#pragma unroll
        for (int q = 0; q < N; ++q) {
            mean[q] = m0;
            rstd[q] = r0;
            sums[q] = s0;
        }
        if (N > 1 && a.K % N != 0) {
#pragma unroll
            for (int q = 1; q < N; ++q) {
                const std::uint64_t other = s * a.G + (c + q) / a.K;
                mean[q] = a.mean[other];
                rstd[q] = a.rstd[other];
                if (SUMS) sums[q] = a.sums[other];
            }
        }
    }
};

// ---------------------------------------------------------------- statistics

constexpr int kTileBatch = 8;
constexpr int kBatch = 4;  // rows loaded before the first is used

// Deviations: sums of what values exceed a value of their own size by (their
// shift, the mean of the first few), and of the squares of that, at two
// operations an element.  The square of the sum is taken from the squares' sum,
// which costs the digits that the shift's distance from the mean is worth: none
// to speak of, unless an outlier lies among the first values.  Where the squares
// hold more than kMostLost times what remains, the values are taken again from
// their mean; once is enough, as what is left is that mean's own rounding (a
// shift that only rounding parts from the mean stays).  A batch of rows is summed
// by itself first: beside an outlier the others' squares are one small value
// again and again, which a single sum would round the same way every time.
// Together a few 2^-24 of a standard deviation at any outlier, as a plain
// two-pass evaluation; 600,000 x 256 bf16 rows 190 us instead of 183, 2,000
// ragged graphs of 169,000 x 128 36.5 instead of 35.5, fp32 rows as before.
constexpr float kMostLost = 8.0f;
__device__ __forceinline__ bool shift_is_far(float count, float shift, float sum, float dev) {
    return sum * sum > kMostLost * count * dev && fabsf(sum) > count * fabsf(shift) * 0x1p-20f;
}

// The mean and squared deviations of each segment's rows in a tile, group by
// group, first channel by channel for a lane's rows; a mean of every batch,
// joined, instead of one shift, took 2.45M x 256 bf16 rows 394 us, not 217.
template <typename T, int N>
__global__ void __launch_bounds__(kThreads, 4) stats_kernel(NormArgs a) {
    if (!tiles_needed(a.seen, a.seenCount)) return;
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
        if (first >= end || a.seg.whole(s)) continue;
        if (active) {
            for (std::uint32_t cv = cv0; cv < a.colsV; cv += kThreads) {
                vec_t<float, N> shift(0.0f), sum, square, mean, dev;
                const std::uint32_t count = lane_rows(first, end, row, a.rowLanes);
                const float rows = static_cast<float>(max(count, 1u));
                for (bool again = false;; again = true) {
                    const T* p = x + (first + row) * a.ldx + cv * N;
                    sum = square = vec_t<float, N>(0.0f);
                    for (std::uint32_t done = 0; done < count; done += kTileBatch) {
                        const std::uint32_t got = min(count - done, static_cast<std::uint32_t>(kTileBatch));
                        vec_t<float, N> v[kTileBatch];
#pragma unroll
                        for (std::uint32_t u = 0; u < kTileBatch; ++u) {
                            v[u] = load_once<T, N>(p);
                            if (u + 1 < got) p += a.rowLanes * a.ldx;
                        }
                        p += a.rowLanes * a.ldx;
                        if (done == 0 && !again) {  // places past the last row repeat it
                            shift = v[0];
#pragma unroll
                            for (int u = 1; u < kTileBatch; ++u) shift += v[u];
                            shift *= 1.0f / kTileBatch;
                        }
                        vec_t<float, N> some(0.0f), squares(0.0f);
#pragma unroll
                        for (std::uint32_t u = 0; u < kTileBatch; ++u)
                            if (u < got) {
                                const vec_t<float, N> e = v[u] - shift;
                                some += e;
                                squares += e * e;
                            }
                        sum += some;
                        square += squares;
                    }
                    mean = shift + sum / rows;
                    dev = square - sum * sum / rows;
                    bool far = false;
#pragma unroll
                    for (int q = 0; q < N; ++q) far |= shift_is_far(rows, shift[q], sum[q], dev[q]);
                    if (again || !far) break;
                    shift = mean;
                }
#pragma unroll
                for (int q = 0; q < N; ++q) {
                    ldsMean[row * a.C + cv * N + q] = mean[q];
                    ldsDev[row * a.C + cv * N + q] = fmaxf(dev[q], 0.0f) + (dev[q] - dev[q]);  // NaN stays
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

// The groups of a segment's joins: with W > 1 a workgroup of W waves each
// (few segments of many slots), else a wave each.
template <int W>
struct JoinGroup {
    static constexpr int threads = W > 1 ? W * kWave : kThreads;
    // few workgroups, each with many segments: most have none to join
    static dim3 grid(std::uint64_t B, std::uint32_t G) {
        const std::uint32_t y = W > 1 ? G : (G + kWaves - 1) / kWaves;
        return dim3(static_cast<unsigned>(std::min<std::uint64_t>(B, std::max(1u, 2048 / y))), y);
    }
    __device__ __forceinline__ static std::uint32_t group() {
        return W > 1 ? blockIdx.y : blockIdx.y * kWaves + threadIdx.x / kWave;
    }
    __device__ __forceinline__ static std::uint32_t first() { return W > 1 ? threadIdx.x : __lane_id(); }
    // The sum of the group's threads' values, in the same order every time.
    __device__ __forceinline__ static float sum(float v, float* red) {
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
};

// mean and rstd of one segment's groups from its slots.
template <int W>
__global__ void __launch_bounds__(JoinGroup<W>::threads) stats_join_kernel(NormArgs a) {
    if (!tiles_needed(a.seen, a.seenCount)) return;
    using Join = JoinGroup<W>;
    __shared__ float red[W];
    const std::uint32_t g = Join::group();
    for (std::uint64_t s = blockIdx.x; s < a.seg.B; s += gridDim.x) {
        const std::uint64_t first = a.seg.start(s), end = a.seg.start(s + 1);
        if (g >= a.G || (first < end && a.seg.whole(s))) continue;
        float mean = 0.0f, var = 0.0f;
        if (first < end) {
            const std::uint64_t t0 = first / a.tileRows, t1 = (end - 1) / a.tileRows;
            const float rows = static_cast<float>(end - first);
            float sum = 0.0f;
            for (std::uint64_t t = t0 + Join::first(); t <= t1; t += kWave * W)
                sum += a.part[(t + s) * a.G + g].x * slot_rows(a, t, first, end);
            mean = Join::sum(sum, red) / rows;
            float dev = 0.0f;
            for (std::uint64_t t = t0 + Join::first(); t <= t1; t += kWave * W) {
                const float2 p = a.part[(t + s) * a.G + g];
                const float gap = p.x - mean;
                dev += p.y + gap * gap * slot_rows(a, t, first, end) * static_cast<float>(a.K);
            }
            var = Join::sum(dev, red) / (rows * static_cast<float>(a.K));
        }
        if (Join::first() == 0) {
            a.mean[s * a.G + g] = mean;
            a.rstd[s * a.G + g] = 1.0f / sqrtf(var + a.eps);
        }
    }
}

// ---------------------------------------------------------------- output

template <typename T, int N, std::uint32_t ACT>
__global__ void __launch_bounds__(kThreads) apply_kernel(NormArgs a) {
    if (!tiles_needed(a.seen, a.seenCount)) return;
    const std::uint64_t lo = blockIdx.x * a.outRows, hi = min(lo + a.outRows, a.seg.N);
    const std::uint32_t rl = threadIdx.x / a.colsV;
    const std::uint32_t cv0 = a.colsV > kThreads ? threadIdx.x : threadIdx.x - rl * a.colsV;
    const std::uint64_t s0 = a.seg.find(lo);
    if (a.colsV <= kThreads && rl >= a.rowLanes) return;
    const std::uint32_t row = a.colsV > kThreads ? 0u : rl;
    const T* x = static_cast<const T*>(a.x);
    T* y = static_cast<T*>(a.out);
    for (std::uint32_t cv = cv0; cv < a.colsV; cv += kThreads) {
        const vec_t<float, N> w = load_params<N>(a.weight, a.paramType, cv * N, 1.0f);
        const vec_t<float, N> b = load_params<N>(a.bias, a.paramType, cv * N, 0.0f);
        for (std::uint64_t s = s0; s < a.seg.B; ++s) {
            const std::uint64_t first = max(a.seg.start(s), lo), end = min(a.seg.start(s + 1), hi);
            if (a.seg.start(s) >= hi) break;
            if (first >= end || a.seg.whole(s)) continue;
            OfGroups<N> of;
            of.template load<false>(a, s, cv * N);
#pragma unroll 4
            for (std::uint64_t r = first + row; r < end; r += a.rowLanes) {
                const vec_t<float, N> v = load_once<T, N>(x + r * a.ldx + cv * N);
                vec_t<float, N> o;
#pragma unroll
                for (int q = 0; q < N; ++q) o[q] = activate<ACT, kFine<T>>(affine(normalise(v[q], of.mean[q], of.rstd[q]), w[q], b[q]));
                store_row<T, N>(y + r * a.ldo + cv * N, o);
            }
        }
    }
}

// ---------------------------------------------------------------- gradient

// S1 and S2 of each segment's rows in a tile, and the tile's dBias and
// dWeight.  LDS: the segment's sums and the tile's, a place for each lane.
template <typename T, int N, std::uint32_t ACT>
__global__ void __launch_bounds__(kThreads) grad_sums_kernel(NormArgs a) {
    if (!tiles_needed(a.seen, a.seenCount)) return;
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
        if (first >= end || a.seg.whole(s)) continue;
        if (active) {
            for (std::uint32_t cv = cv0; cv < a.colsV; cv += kThreads) {
                const vec_t<float, N> w = load_params<N>(a.weight, a.paramType, cv * N, 1.0f);
                const vec_t<float, N> b = load_params<N>(a.bias, a.paramType, cv * N, 0.0f);
                OfGroups<N> of;
                of.template load<false>(a, s, cv * N);
                vec_t<float, N> s1(0.0f), s2(0.0f);
#pragma unroll 4
                for (std::uint64_t r = first + row; r < end; r += a.rowLanes) {
                    const vec_t<float, N> v = load_once<T, N>(x + r * a.ldx + cv * N);
                    const vec_t<float, N> d = load_once<T, N>(dy + r * a.lddy + cv * N);
#pragma unroll
                    for (int q = 0; q < N; ++q) {
                        const float xh = normalise(v[q], of.mean[q], of.rstd[q]);
                        const float dz = through<ACT, kFine<T>>(d[q], affine(xh, w[q], b[q]));
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

// S1 / M and S2 / M of one segment's groups from its slots.
template <int W>
__global__ void __launch_bounds__(JoinGroup<W>::threads) grad_join_kernel(NormArgs a) {
    if (!tiles_needed(a.seen, a.seenCount)) return;
    using Join = JoinGroup<W>;
    __shared__ float red[W];
    const std::uint32_t g = Join::group();
    for (std::uint64_t s = blockIdx.x; s < a.seg.B; s += gridDim.x) {
        const std::uint64_t first = a.seg.start(s), end = a.seg.start(s + 1);
        if (g >= a.G || first >= end || a.seg.whole(s)) continue;
        const std::uint64_t t0 = first / a.tileRows, t1 = (end - 1) / a.tileRows;
        float s1 = 0.0f, s2 = 0.0f;
        for (std::uint64_t t = t0 + Join::first(); t <= t1; t += kWave * W) {
            const float2 p = a.part[(t + s) * a.G + g];
            s1 += p.x;
            s2 += p.y;
        }
        s1 = Join::sum(s1, red);
        s2 = Join::sum(s2, red);
        const float size = static_cast<float>(end - first) * static_cast<float>(a.K);
        if (Join::first() == 0) a.sums[s * a.G + g] = float2{s1 / size, s2 / size};
    }
}

// dBias and dWeight from `rows` rows of partial sums: 4 columns a workgroup,
// 256 threads a column; the tiles' rows come after the whole segments'.
constexpr std::uint32_t kParamCols = 4, kParamRows = 256;
__global__ void __launch_bounds__(kParamCols* kParamRows) param_grad_kernel(NormArgs a, std::uint64_t wholeRows,
                                                                           std::uint64_t tiles, float* dWeight,
                                                                           float* dBias) {
    __shared__ float2 red[kParamCols * kParamRows];
    const std::uint32_t c = blockIdx.x * kParamCols + threadIdx.x % kParamCols, C = a.C;
    const float2* channel = a.channel;
    const std::uint64_t rows = wholeRows + (tiles > 0 && tiles_needed(a.seen, a.seenCount) ? tiles : 0);
    float2 s{0.0f, 0.0f};
    if (c < C) {
#pragma unroll 8
        for (std::uint64_t t = threadIdx.x / kParamCols; t < rows; t += kParamRows) {
            const float2 p = channel[t * C + c];
            s.x += p.x;
            s.y += p.y;
        }
    }
    red[threadIdx.x] = s;
    __syncthreads();
    for (std::uint32_t half = kParamRows / 2; half > 0; half /= 2) {
        if (threadIdx.x < half * kParamCols) {
            red[threadIdx.x].x += red[threadIdx.x + half * kParamCols].x;
            red[threadIdx.x].y += red[threadIdx.x + half * kParamCols].y;
        }
        __syncthreads();
    }
    if (threadIdx.x < kParamCols && c < C) {
        if (dBias != nullptr) dBias[c] = red[threadIdx.x].x;
        if (dWeight != nullptr) dWeight[c] = red[threadIdx.x].y;
    }
}

template <typename T, int N, std::uint32_t ACT>
__global__ void __launch_bounds__(kThreads) grad_apply_kernel(NormArgs a) {
    if (!tiles_needed(a.seen, a.seenCount)) return;
    const std::uint64_t lo = blockIdx.x * a.outRows, hi = min(lo + a.outRows, a.seg.N);
    const std::uint32_t rl = threadIdx.x / a.colsV;
    const std::uint32_t cv0 = a.colsV > kThreads ? threadIdx.x : threadIdx.x - rl * a.colsV;
    const std::uint64_t s0 = a.seg.find(lo);
    if (a.colsV <= kThreads && rl >= a.rowLanes) return;
    const std::uint32_t row = a.colsV > kThreads ? 0u : rl;
    const T* x = static_cast<const T*>(a.x);
    const T* dy = static_cast<const T*>(a.dy);
    T* dx = static_cast<T*>(a.out);
    for (std::uint32_t cv = cv0; cv < a.colsV; cv += kThreads) {
        const vec_t<float, N> w = load_params<N>(a.weight, a.paramType, cv * N, 1.0f);
        const vec_t<float, N> b = load_params<N>(a.bias, a.paramType, cv * N, 0.0f);
        for (std::uint64_t s = s0; s < a.seg.B; ++s) {
            const std::uint64_t first = max(a.seg.start(s), lo), end = min(a.seg.start(s + 1), hi);
            if (a.seg.start(s) >= hi) break;
            if (first >= end || a.seg.whole(s)) continue;
            OfGroups<N> of;
            of.template load<true>(a, s, cv * N);
#pragma unroll 4
            for (std::uint64_t r = first + row; r < end; r += a.rowLanes) {
                const vec_t<float, N> v = load_once<T, N>(x + r * a.ldx + cv * N);
                const vec_t<float, N> d = load_once<T, N>(dy + r * a.lddy + cv * N);
                vec_t<float, N> o;
#pragma unroll
                for (int q = 0; q < N; ++q) {
                    const float xh = normalise(v[q], of.mean[q], of.rstd[q]);
                    const float dz = through<ACT, kFine<T>>(d[q], affine(xh, w[q], b[q]));
                    o[q] = (dz * w[q] - of.sums[q].x - xh * of.sums[q].y) * of.rstd[q];
                }
                store_row<T, N>(dx + r * a.ldo + cv * N, o);
            }
        }
    }
}

// ---------------------------------------------------------------- whole segments

// A workgroup takes a segment (a slice of whole groups of it) at a time: the
// statistics come from a first reading and the output from a second, which the
// caches mostly serve.  (Rows held in registers between the two left so few
// waves that waiting for the first reading took longer than the second one
// does.)  A vector of a lane lies in one group (N divides K).  What a short
// segment costs is the wait for its offsets, its rows and its sums, so the
// workgroup is a single wave where that holds the usual segment: as many of
// them as fit a CU wait at the same time.
constexpr int kWholeThreads = 256;  // at most; one wave where segments are short

struct WholeArgs {
    std::uint32_t blocks;     // workgroups of a slice: the segments a grid's step apart
    std::uint32_t slices;
    std::uint32_t threads;    // of a workgroup
    std::uint32_t groups;     // of a slice
    std::uint32_t cols;       // its vectors a row
    std::uint32_t laneBits;   // lanes of a row: a power of two that holds them, at most `threads`
    std::uint32_t groupCols;  // vectors of a group (1 where they straddle groups)
};

// Sums of a pair of values over the lanes of each group, each lane getting its
// own group's, in the same order every time.  `red` is not read by the call
// before the next one's first wait, so two places used in turn need one wait.
struct GroupSum {
    std::uint32_t threads, lanes, groupCols, cv, g0;  // g0: the group's first vector
    bool tree;                               // groups of a power of two of vectors

    __device__ __forceinline__ float2 operator()(float2 v, float2* red) const {
        for (std::uint32_t d = lanes; d < kWave; d <<= 1) {
            v.x += __shfl_xor(v.x, d, kWave);
            v.y += __shfl_xor(v.y, d, kWave);
        }
        const std::uint32_t inWave = min(groupCols, static_cast<std::uint32_t>(kWave));
        if (tree)
            for (std::uint32_t d = 1; d < inWave; d <<= 1) {
                v.x += __shfl_xor(v.x, d, kWave);
                v.y += __shfl_xor(v.y, d, kWave);
            }
        if (tree && threads == kWave) return v;
        // rows of places: a wave's lanes' columns, or a row of lanes
        const std::uint32_t rows = lanes < kWave ? threads / kWave : threads / lanes;
        const std::uint32_t at = lanes < kWave ? threadIdx.x / kWave * lanes + cv : threadIdx.x;
        if (lanes >= kWave || __lane_id() < lanes) red[at] = v;
        __syncthreads();
        const std::uint32_t step = tree ? inWave : 1u;
        float2 s{0.0f, 0.0f};
        for (std::uint32_t r = 0; r < rows; ++r)
            for (std::uint32_t c = g0; c < g0 + groupCols; c += step) {
                const float2 p = red[r * lanes + c];
                s.x += p.x;
                s.y += p.y;
            }
        return s;
    }
};

// What a lane of a slice works on.
template <int N>
struct WholeLane {
    std::uint32_t cv, row, rowLanes, c;  // its vector of the slice, row lane, the rows at once, its first channel
    std::uint32_t g0, g;                 // the slice's first group; the lane's (where a vector lies in one)
    std::uint32_t block;                 // the first of its segments
    bool active;
    GroupSum sum;
    __device__ __forceinline__ WholeLane(const NormArgs& a, const WholeArgs& k) {
        // 8 segments' first slices, then their second ones: the slices of a
        // segment meet on one XCD (workgroups go to the 8 of them in turn),
        // whose L2 then holds the lines that they share
        const std::uint32_t turn = blockIdx.x / (8 * k.slices), place = blockIdx.x - turn * 8 * k.slices;
        const std::uint32_t slice = place / 8;
        block = turn * 8 + place % 8;
        const std::uint32_t lanes = 1u << k.laneBits;
        cv = threadIdx.x & (lanes - 1u);
        row = threadIdx.x >> k.laneBits;
        rowLanes = k.threads >> k.laneBits;
        active = cv < k.cols;
        g0 = slice * k.groups;
        c = (slice * k.cols + cv) * N;
        const std::uint32_t inSlice = cv / k.groupCols;
        g = g0 + inSlice;
        sum = GroupSum{k.threads, lanes, k.groupCols, cv, min(inSlice, k.groups - 1) * k.groupCols,
                       (k.groupCols & (k.groupCols - 1)) == 0};
    }
};

// Calls body(v..., place in the batch) for a lane's rows r, r + rowLanes, ... below
// `rows`, kBatch of them loaded before the first is used; p... go from row r on.  Past the end
// the last row is loaded again and not used: a loop for the remainder waited
// for each of its rows in turn.
template <typename T, int N, typename Body>
__device__ __forceinline__ void each_row(std::uint64_t r, std::uint64_t rows, std::uint32_t rowLanes, const T* p,
                                         std::uint64_t step, Body body) {
    for (; r < rows; r += kBatch * rowLanes) {
        const int more = static_cast<int>(min<std::uint64_t>(kBatch, (rows - r + rowLanes - 1) / rowLanes));
        vec_t<T, N> v[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            v[i] = load_global<vec_t<T, N>>(p);
            if (i + 1 < more) p += step;
        }
        p += step;
        body(v, more);
    }
}
template <typename T, int N, typename Body>
__device__ __forceinline__ void each_row(std::uint64_t r, std::uint64_t rows, std::uint32_t rowLanes, const T* p,
                                         std::uint64_t step, const T* q, std::uint64_t stepQ, Body body) {
    for (; r < rows; r += kBatch * rowLanes) {
        const int more = static_cast<int>(min<std::uint64_t>(kBatch, (rows - r + rowLanes - 1) / rowLanes));
        vec_t<T, N> v[kBatch], u[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            v[i] = load_global<vec_t<T, N>>(p);
            u[i] = load_global<vec_t<T, N>>(q);
            if (i + 1 < more) {
                p += step;
                q += stepQ;
            }
        }
        p += step;
        q += stepQ;
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (i < more) body(__builtin_convertvector(v[i], vec_t<float, N>), __builtin_convertvector(u[i], vec_t<float, N>), i);
    }
}

// What a workgroup saw, told by one of its segments' workgroups (`teller`).
__device__ __forceinline__ void tell_seen(const NormArgs& a, const WholeArgs& k, std::uint32_t block, bool teller,
                                          std::uint8_t anyLong) {
    if (!teller || a.seenCount == 0) return;
    if (block < k.blocks) a.seen[block] = anyLong;
    // places past `blocks` that the tiles' 16-byte loads take in
    if (block + 1 == k.blocks)
        for (std::uint32_t i = k.blocks; i % 16 != 0; ++i) a.seen[i] = 0;
}

// A lane's values: what they exceed their shift by, and the squares of that.
struct Deviations {
    float count;  // of all its values
    float shift = __builtin_nanf(""), sum = 0.0f, square = 0.0f;
    // the first `got` of R vectors
    template <int R, typename T, int N>
    __device__ __forceinline__ void add(const vec_t<T, N> (&v)[R], int got) {
        if (shift != shift) {  // none yet: from four values at least (vectors past the last repeat it)
            constexpr int kFirst = N < 4 ? 4 / N : 1;
            shift = 0.0f;
#pragma unroll
            for (int i = 0; i < kFirst; ++i) {
                const vec_t<float, N> f = __builtin_convertvector(v[i], vec_t<float, N>);
#pragma unroll
                for (int q = 0; q < N; ++q) shift += f[q];
            }
            shift *= 1.0f / (kFirst * N);
        }
        float some = 0.0f, squares = 0.0f;
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (i < got) {
                const vec_t<float, N> f = __builtin_convertvector(v[i], vec_t<float, N>);
#pragma unroll
                for (int q = 0; q < N; ++q) {
                    const float e = f[q] - shift;
                    some += e;
                    squares = fmaf(e, e, squares);
                }
            }
        sum += some;
        square += squares;
    }
    // whether the values are to be added again, from their mean
    __device__ __forceinline__ bool far() const { return shift_is_far(count, shift, sum, square - sum * (sum / count)); }
    __device__ __forceinline__ void restart() {
        shift += sum / count;
        sum = square = 0.0f;
    }
    __device__ __forceinline__ float total() const { return count == 0.0f ? 0.0f : fmaf(count, shift, sum); }
    // the squared deviations from `mean`
    __device__ __forceinline__ float around(float mean) const {
        if (count == 0.0f) return 0.0f;
        const float own = sum / count, gap = (shift - mean) + own;
        return (square - sum * own) + count * gap * gap;
    }
};

template <typename T, int N, std::uint32_t ACT>
__global__ void __launch_bounds__(kWholeThreads, 4) whole_kernel(NormArgs a, WholeArgs k) {
    extern __shared__ float2 places[];  // two of a GroupSum
    float2* const red[2] = {places, places + k.threads};
    const WholeLane<N> me(a, k);
    const std::uint32_t c = me.active ? me.c : 0u;
    const vec_t<float, N> w = load_params<N>(a.weight, a.paramType, c, 1.0f), b = load_params<N>(a.bias, a.paramType, c, 0.0f);
    std::uint8_t anyLong = 0;
    for (std::uint64_t s = me.block; s < a.seg.B; s += k.blocks) {
        const std::uint64_t first = a.seg.start(s), end = a.seg.start(s + 1);
        if (first < end && end - first > a.seg.longest) {
            anyLong = 1;
            continue;
        }
        const std::uint64_t rows = first < end ? end - first : 0;
        const T* x = static_cast<const T*>(a.x) + (first + me.row) * a.ldx + me.c;
        T* y = static_cast<T*>(a.out) + (first + me.row) * a.ldo + me.c;
        float gm = 0.0f, rs = 0.0f;
        // the group's mean and rstd from the lanes' deviations, kept for the gradient
        const auto settle = [&](const Deviations& mine) {
            const float size = static_cast<float>(rows) * static_cast<float>(a.K);
            if (rows > 0) {
                gm = me.sum(float2{mine.total(), 0.0f}, red[0]).x / size;
                rs = me.sum(float2{mine.around(gm), 0.0f}, red[1]).x / size;
                rs = rs < 0.0f ? 0.0f : rs;  // NaN stays
            }
            rs = 1.0f / sqrtf(rs + a.eps);
            if (me.active && me.row == 0 && me.cv == me.sum.g0) {
                a.mean[s * a.G + me.g] = gm;
                a.rstd[s * a.G + me.g] = rs;
            }
        };
        const auto apply = [&](vec_t<float, N> v, T* to) {
            vec_t<float, N> o;
#pragma unroll
            for (int q = 0; q < N; ++q) o[q] = activate<ACT, kFine<T>>(affine(normalise(v[q], gm, rs), w[q], b[q]));
            store_row<T, N>(to, o);
        };
        Deviations mine{static_cast<float>((me.active ? lane_rows(0, rows, me.row, me.rowLanes) : 0u) * N)};
        if (me.active)
            for (bool again = false;; again = true) {
                each_row<T, N>(me.row, rows, me.rowLanes, x, me.rowLanes * a.ldx,
                               [&](vec_t<T, N>(&v)[kBatch], int more) { mine.template add<kBatch, T, N>(v, more); });
                if (again || !mine.far()) break;
                mine.restart();
            }
        settle(mine);
        if (me.active)
            each_row<T, N>(me.row, rows, me.rowLanes, x, me.rowLanes * a.ldx, [&](vec_t<T, N>(&v)[kBatch], int more) {
#pragma unroll
                for (int i = 0; i < kBatch; ++i)
                    if (i < more) {
                        apply(__builtin_convertvector(v[i], vec_t<float, N>), y);
                        y += me.rowLanes * a.ldo;
                    }
            });
    }
    tell_seen(a, k, me.block, me.c == 0 && me.row == 0, anyLong);
}

// Whether the first batch's dz w stay in LDS between the two readings: where the
// slope costs more than the rest of the gradient (169,000 x 128 bf16 rows in
// 2,000 ragged graphs with gelu, 66 us instead of 73).
template <std::uint32_t ACT>
constexpr bool kKeep = ACT == TCC_ACT_SILU || ACT == TCC_ACT_GELU;

// Floats of LDS that a lane of the gradient has, for each of its N elements:
// the kept batch, or dBias and dWeight.
template <std::uint32_t ACT>
constexpr std::uint32_t kGradFloats = kKeep<ACT> ? kBatch : 2;

// `partial`: where this workgroup's dBias and dWeight go ([blocks][C]).
template <typename T, int N, std::uint32_t ACT>
__global__ void __launch_bounds__(kWholeThreads, 4) whole_grad_kernel(NormArgs a, WholeArgs k, float2* partial) {
    extern __shared__ float2 places[];  // two of a GroupSum, then the lanes' kept batches or dBias and dWeight
    float2* const all = places + 2 * k.threads;
    vec_t<float, N>* const kept = reinterpret_cast<vec_t<float, N>*>(all);
    const WholeLane<N> me(a, k);
    const std::uint32_t c = me.active ? me.c : 0u;
    const vec_t<float, N> w = load_params<N>(a.weight, a.paramType, c, 1.0f), b = load_params<N>(a.bias, a.paramType, c, 0.0f);
    vec_t<float, N> dw(0.0f), db(0.0f);
    std::uint32_t turn = 0;
    std::uint8_t anyLong = 0;
    for (std::uint64_t s = me.block; s < a.seg.B; s += k.blocks) {
        const std::uint64_t first = a.seg.start(s), end = a.seg.start(s + 1);
        if (first >= end) continue;
        if (end - first > a.seg.longest) {
            anyLong = 1;
            continue;
        }
        const std::uint64_t rows = end - first;
        const float mean = me.active ? a.mean[s * a.G + me.g] : 0.0f, rstd = me.active ? a.rstd[s * a.G + me.g] : 0.0f;
        const T* x = static_cast<const T*>(a.x) + (first + me.row) * a.ldx + me.c;
        const T* dy = static_cast<const T*>(a.dy) + (first + me.row) * a.lddy + me.c;
        T* dx = static_cast<T*>(a.out) + (first + me.row) * a.ldo + me.c;
        float2 part{0.0f, 0.0f}, m{0.0f, 0.0f};
        // dz, counted in the sums
        const auto gather = [&](vec_t<float, N> v, vec_t<float, N> d) {
#pragma unroll
            for (int q = 0; q < N; ++q) {
                const float xh = normalise(v[q], mean, rstd);
                d[q] = through<ACT, kFine<T>>(d[q], affine(xh, w[q], b[q]));
                db[q] += d[q];
                dw[q] = fmaf(d[q], xh, dw[q]);
                d[q] *= w[q];
                part.x += d[q];
                part.y = fmaf(d[q], xh, part.y);
            }
            return d;
        };
        const auto settle = [&] {
            const float size = static_cast<float>(rows) * static_cast<float>(a.K);
            m = me.sum(part, places + turn * k.threads);
            turn ^= 1u;
            m.x /= size;
            m.y /= size;
        };
        const auto apply = [&](vec_t<float, N> v, vec_t<float, N> dzw, T* to) {
            vec_t<float, N> o;
#pragma unroll
            for (int q = 0; q < N; ++q) o[q] = (dzw[q] - m.x - normalise(v[q], mean, rstd) * m.y) * rstd;
            store_row<T, N>(to, o);
        };
        const std::uint64_t stepX = me.rowLanes * a.ldx, stepD = me.rowLanes * a.lddy, stepO = me.rowLanes * a.ldo;
        const std::uint64_t after = kKeep<ACT> ? min(rows, static_cast<std::uint64_t>(kBatch * me.rowLanes)) : 0;
        const std::uint32_t skip = kKeep<ACT> ? kBatch : 0;
        if (me.active) {
            if (kKeep<ACT>)
                each_row<T, N>(me.row, after, me.rowLanes, x, stepX, dy, stepD,
                               [&](vec_t<float, N> v, vec_t<float, N> d, int i) {
                                   kept[i * k.threads + threadIdx.x] = gather(v, d);
                               });
            each_row<T, N>(me.row + skip * me.rowLanes, rows, me.rowLanes, x + skip * stepX, stepX, dy + skip * stepD, stepD,
                           [&](vec_t<float, N> v, vec_t<float, N> d, int) { gather(v, d); });
        }
        settle();
        if (me.active) {
            if (kKeep<ACT>)
                each_row<T, N>(me.row, after, me.rowLanes, x, stepX, [&](vec_t<T, N>(&v)[kBatch], int more) {
#pragma unroll
                    for (int i = 0; i < kBatch; ++i)
                        if (i < more)
                            apply(__builtin_convertvector(v[i], vec_t<float, N>), kept[i * k.threads + threadIdx.x],
                                  dx + i * stepO);
                });
            dx += skip * stepO;
            each_row<T, N>(me.row + skip * me.rowLanes, rows, me.rowLanes, x + skip * stepX, stepX, dy + skip * stepD, stepD,
                           [&](vec_t<float, N> v, vec_t<float, N> d, int) {
#pragma unroll
                               for (int q = 0; q < N; ++q)
                                   d[q] = through<ACT, kFine<T>>(d[q], affine(normalise(v[q], mean, rstd), w[q], b[q])) * w[q];
                               apply(v, d, dx);
                               dx += stepO;
                           });
        }
    }
    tell_seen(a, k, me.block, me.c == 0 && me.row == 0, anyLong);
    if (partial == nullptr || me.block >= k.blocks) return;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < N; ++q) all[threadIdx.x * N + q] = float2{db[q], dw[q]};
    __syncthreads();
    const std::uint32_t lanes = 1u << k.laneBits;
    for (std::uint32_t i = threadIdx.x; i < k.cols * N; i += k.threads) {
        float2 s{0.0f, 0.0f};
        for (std::uint32_t r = 0; r < me.rowLanes; ++r) {
            const float2 p = all[(r * lanes) * N + i];
            s.x += p.x;
            s.y += p.y;
        }
        partial[me.block * static_cast<std::uint64_t>(a.C) + (me.c - me.cv * N) + i] = s;
    }
}

// ---------------------------------------------------------------- groups of odd sizes

// Whole segments where a lane's vector straddles groups (C / G of 3 or 25, say):
// channels are summed apart and joined to groups in LDS.  Lanes as narrow as
// such groups allow, a channel each at worst, took 5 to 13 times the time that
// the bytes need.

// The lanes' pairs for each channel, summed over the rows of a workgroup: the
// places of `rows` partial sums of channel c of the slice are c, c + stride, ...
template <int N>
struct ChannelSums {
    float2* places;
    std::uint32_t rows, stride;
    __device__ __forceinline__ ChannelSums(const WholeArgs& k, float2* p) : places(p) {
        const std::uint32_t lanes = 1u << k.laneBits;
        rows = lanes < kWave ? k.threads / kWave : k.threads / lanes;
        stride = lanes * N;
    }
    __device__ __forceinline__ void put(const WholeArgs& k, vec_t<float, N> x, vec_t<float, N> y) const {
        const std::uint32_t lanes = 1u << k.laneBits;
        for (std::uint32_t d = lanes; d < kWave; d <<= 1)
#pragma unroll
            for (int q = 0; q < N; ++q) {
                x[q] += __shfl_xor(x[q], d, kWave);
                y[q] += __shfl_xor(y[q], d, kWave);
            }
        const std::uint32_t at = lanes < kWave ? threadIdx.x / kWave * lanes + __lane_id() : threadIdx.x;
        if (lanes >= kWave || __lane_id() < lanes)
#pragma unroll
            for (int q = 0; q < N; ++q) places[at * N + q] = float2{x[q], y[q]};
    }
    __device__ __forceinline__ float2 of(std::uint32_t c) const {
        float2 s{0.0f, 0.0f};
        for (std::uint32_t r = 0; r < rows; ++r) {
            const float2 p = places[r * stride + c];
            s.x += p.x;
            s.y += p.y;
        }
        return s;
    }
};

// The threads of a workgroup as teams, one for a group of the slice at a time.
struct GroupTeam {
    std::uint32_t size, first, step, lane;
    __device__ __forceinline__ explicit GroupTeam(const WholeArgs& k) {
        size = 1;
        while (size < kWave && 2 * size * k.groups <= k.threads) size *= 2;
        first = threadIdx.x / size;
        step = k.threads / size;
        lane = threadIdx.x % size;
    }
    __device__ __forceinline__ float sum(float v) const {
        for (std::uint32_t d = 1; d < size; d <<= 1) v += __shfl_xor(v, d, kWave);
        return v;
    }
};

// LDS: the channels' places, [lanes * N] floats of their shifts, a pair for each group.
template <int N>
std::uint32_t spread_lds(const WholeArgs& k) {
    return (k.threads * N + ((1u << k.laneBits) * N + 1) / 2 + k.groups) * static_cast<std::uint32_t>(sizeof(float2));
}

template <typename T, int N, std::uint32_t ACT>
__global__ void __launch_bounds__(kWholeThreads, 4) spread_kernel(NormArgs a, WholeArgs k) {
    extern __shared__ float2 places[];
    float* const shifts = reinterpret_cast<float*>(places + k.threads * N);
    float2* const groups = places + k.threads * N + ((1u << k.laneBits) * N + 1) / 2;
    const WholeLane<N> me(a, k);
    const ChannelSums<N> channels(k, places);
    const GroupTeam team(k);
    const std::uint32_t c = me.active ? me.c : 0u, own = me.cv * N;  // the channel in the slice
    const vec_t<float, N> w = load_params<N>(a.weight, a.paramType, c, 1.0f), b = load_params<N>(a.bias, a.paramType, c, 0.0f);
    std::uint8_t anyLong = 0;
    for (std::uint64_t s = me.block; s < a.seg.B; s += k.blocks) {
        const std::uint64_t first = a.seg.start(s), end = a.seg.start(s + 1);
        if (first < end && end - first > a.seg.longest) {
            anyLong = 1;
            continue;
        }
        const std::uint64_t rows = first < end ? end - first : 0;
        const T* x = static_cast<const T*>(a.x) + (first + me.row) * a.ldx + me.c;
        T* y = static_cast<T*>(a.out) + (first + me.row) * a.ldo + me.c;
        vec_t<float, N> shift(0.0f);
        if (me.active && rows > 0) {
            // the same for every lane of these channels: the mean of four rows
            const T* p = static_cast<const T*>(a.x) + first * a.ldx + me.c;
#pragma unroll
            for (int i = 0; i < 4; ++i) shift += load_row<T, N>(p + rows * i / 4 * a.ldx);
            shift *= 0.25f;
            if (me.row == 0)
#pragma unroll
                for (int q = 0; q < N; ++q) shifts[own + q] = shift[q];
        }
        const float n = static_cast<float>(rows), size = n * static_cast<float>(a.K);
        for (bool again = false;; again = true) {
            vec_t<float, N> sum(0.0f), square(0.0f);
            if (me.active)
                each_row<T, N>(me.row, rows, me.rowLanes, x, me.rowLanes * a.ldx, [&](vec_t<T, N>(&v)[kBatch], int more) {
                    vec_t<float, N> some(0.0f), squares(0.0f);
#pragma unroll
                    for (int i = 0; i < kBatch; ++i)
                        if (i < more) {
                            const vec_t<float, N> e = __builtin_convertvector(v[i], vec_t<float, N>) - shift;
                            some += e;
                            squares += e * e;
                        }
                    sum += some;
                    square += squares;
                });
            channels.put(k, sum, square);
            __syncthreads();
            bool far = false;
            for (std::uint32_t g = team.first; g < k.groups; g += team.step) {
                float mean = 0.0f, var = 0.0f;
                if (rows > 0) {
                    for (std::uint32_t e = g * a.K + team.lane; e < (g + 1) * a.K; e += team.size)
                        mean += shifts[e] + channels.of(e).x / n;
                    mean = team.sum(mean) / static_cast<float>(a.K);
                    for (std::uint32_t e = g * a.K + team.lane; e < (g + 1) * a.K; e += team.size) {
                        const float2 p = channels.of(e);
                        const float part = p.x / n, gap = (shifts[e] - mean) + part, dev = p.y - p.x * part;
                        var += dev + n * gap * gap;
                        far |= shift_is_far(n, shifts[e], p.x, dev);
                    }
                    var = team.sum(var) / size;
                    var = var < 0.0f ? 0.0f : var;  // NaN stays
                }
                if (team.lane == 0) {
                    const float rs = 1.0f / sqrtf(var + a.eps);
                    groups[g] = float2{mean, rs};
                    a.mean[s * a.G + me.g0 + g] = mean;
                    a.rstd[s * a.G + me.g0 + g] = rs;
                }
            }
            if (!__syncthreads_or(far) || again) break;
            for (std::uint32_t e = threadIdx.x; e < k.cols * N; e += k.threads) shifts[e] += channels.of(e).x / n;
            __syncthreads();
            if (me.active)
#pragma unroll
                for (int q = 0; q < N; ++q) shift[q] = shifts[own + q];
        }
        if (!me.active || rows == 0) continue;
        float2 of[N];
#pragma unroll
        for (int q = 0; q < N; ++q) of[q] = groups[(own + q) / a.K];
        each_row<T, N>(me.row, rows, me.rowLanes, x, me.rowLanes * a.ldx, [&](vec_t<T, N>(&v)[kBatch], int more) {
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
                if (i < more) {
                    const vec_t<float, N> f = __builtin_convertvector(v[i], vec_t<float, N>);
                    vec_t<float, N> o;
#pragma unroll
                    for (int q = 0; q < N; ++q) o[q] = activate<ACT, kFine<T>>(affine(normalise(f[q], of[q].x, of[q].y), w[q], b[q]));
                    store_row<T, N>(y, o);
                    y += me.rowLanes * a.ldo;
                }
        });
    }
    tell_seen(a, k, me.block, me.c == 0 && me.row == 0, anyLong);
}

// `partial` as in whole_grad_kernel.
template <typename T, int N, std::uint32_t ACT>
__global__ void __launch_bounds__(kWholeThreads, 4) spread_grad_kernel(NormArgs a, WholeArgs k, float2* partial) {
    extern __shared__ float2 places[];
    float2* const groups = places + k.threads * N + ((1u << k.laneBits) * N + 1) / 2;
    const WholeLane<N> me(a, k);
    const ChannelSums<N> channels(k, places);
    const GroupTeam team(k);
    const std::uint32_t c = me.active ? me.c : 0u, own = me.cv * N;
    const vec_t<float, N> w = load_params<N>(a.weight, a.paramType, c, 1.0f), b = load_params<N>(a.bias, a.paramType, c, 0.0f);
    vec_t<float, N> dw(0.0f), db(0.0f);
    std::uint8_t anyLong = 0;
    for (std::uint64_t s = me.block; s < a.seg.B; s += k.blocks) {
        const std::uint64_t first = a.seg.start(s), end = a.seg.start(s + 1);
        if (first >= end) continue;
        if (end - first > a.seg.longest) {
            anyLong = 1;
            continue;
        }
        const std::uint64_t rows = end - first;
        const T* x = static_cast<const T*>(a.x) + (first + me.row) * a.ldx + me.c;
        const T* dy = static_cast<const T*>(a.dy) + (first + me.row) * a.lddy + me.c;
        T* dx = static_cast<T*>(a.out) + (first + me.row) * a.ldo + me.c;
        const std::uint64_t stepX = me.rowLanes * a.ldx, stepD = me.rowLanes * a.lddy;
        float mean[N], rstd[N];
#pragma unroll
        for (int q = 0; q < N; ++q) {
            const std::uint64_t at = s * a.G + (me.active ? me.g0 + (own + q) / a.K : 0u);
            mean[q] = a.mean[at];
            rstd[q] = a.rstd[at];
        }
        vec_t<float, N> s1(0.0f), s2(0.0f);
        if (me.active)
            each_row<T, N>(me.row, rows, me.rowLanes, x, stepX, dy, stepD, [&](vec_t<float, N> v, vec_t<float, N> d, int) {
#pragma unroll
                for (int q = 0; q < N; ++q) {
                    const float xh = normalise(v[q], mean[q], rstd[q]);
                    const float z = through<ACT, kFine<T>>(d[q], affine(xh, w[q], b[q]));
                    s1[q] += z;
                    s2[q] = fmaf(z, xh, s2[q]);
                }
            });
        db += s1;
        dw += s2;
        channels.put(k, s1 * w, s2 * w);
        __syncthreads();
        const float size = static_cast<float>(rows) * static_cast<float>(a.K);
        for (std::uint32_t g = team.first; g < k.groups; g += team.step) {
            float2 m{0.0f, 0.0f};
            for (std::uint32_t e = g * a.K + team.lane; e < (g + 1) * a.K; e += team.size) {
                const float2 p = channels.of(e);
                m.x += p.x;
                m.y += p.y;
            }
            m.x = team.sum(m.x);
            m.y = team.sum(m.y);
            if (team.lane == 0) groups[g] = float2{m.x / size, m.y / size};
        }
        __syncthreads();
        if (!me.active) continue;
        float2 of[N];
#pragma unroll
        for (int q = 0; q < N; ++q) of[q] = groups[(own + q) / a.K];
        each_row<T, N>(me.row, rows, me.rowLanes, x, stepX, dy, stepD, [&](vec_t<float, N> v, vec_t<float, N> d, int) {
            vec_t<float, N> o;
#pragma unroll
            for (int q = 0; q < N; ++q) {
                const float xh = normalise(v[q], mean[q], rstd[q]);
                o[q] = (through<ACT, kFine<T>>(d[q], affine(xh, w[q], b[q])) * w[q] - of[q].x - xh * of[q].y) * rstd[q];
            }
            store_row<T, N>(dx, o);
            dx += me.rowLanes * a.ldo;
        });
    }
    tell_seen(a, k, me.block, me.c == 0 && me.row == 0, anyLong);
    if (partial == nullptr || me.block >= k.blocks) return;
    __syncthreads();
    channels.put(k, me.active ? db : vec_t<float, N>(0.0f), me.active ? dw : vec_t<float, N>(0.0f));
    __syncthreads();
    for (std::uint32_t i = threadIdx.x; i < k.cols * N; i += k.threads)
        partial[me.block * static_cast<std::uint64_t>(a.C) + me.g0 * a.K + i] = channels.of(i);
}

// ---------------------------------------------------------------- host side

constexpr std::size_t align16(std::size_t b) { return (b + 15) & ~std::size_t(15); }

// Tiles of at most this many, so that the tiles' sums stay few.
constexpr std::uint64_t kTiles = 2048;
// A segment that a workgroup walks in at most kWholeSteps steps goes whole (some
// 30 us; a longer one would end after all others), or in kManySteps where kMany
// segments and more take longer in all.  Where the longest is not known, it is
// taken for kUneven times the mean (kManyUneven with many, of which few go by
// tiles then): none goes whole if that is too long, as the kernels for both cost
// more than either.  Where no more than kSmallSteps could make one segment and
// the mean is half of what goes whole, all do, for the launches that this
// saves.  780 segments of 324,652 x 32 bf16 rows, gradient: 62 us with 128 steps,
// 89 with 64, 140 with 32; 70 of 17,559 x 42 rows (31 steps in the mean): 35 by
// tiles, 70 whole; 395 of 13,842 x 592 (9 steps): 71 by tiles, 49 mostly whole; 5
// of 665 x 96 rows: 12 whole, 39 by tiles.
constexpr std::uint64_t kWholeSteps = 64, kManySteps = 128, kMany = 512, kUneven = 5, kManyUneven = 4, kSmallSteps = 256;
// Workgroups of a slice of whole segments, each with its own dWeight and dBias.
constexpr std::uint64_t kWholeBlocks = 4096;

// Elements a lane takes in a whole segment, of `width` that the rows allow: a
// power of two that divides a group, or up to four that straddle groups where
// these have no such divisor.
struct WholeWidth {
    std::uint32_t n;
    bool spread;
    WholeWidth(std::uint32_t K, std::uint32_t width) : n(width), spread(false) {
        while (K % n != 0) n /= 2;
        const std::uint32_t wide = std::min(width, 4u);
        if (n < wide) {
            n = wide;
            spread = true;
        }
    }
};

// How whole segments are cut, for such lanes: into slices of whole groups (and
// lanes) of at least 128 bytes a row (64 where fewer than 1024 segments have to
// spread over the GPU), a wave for a slice where that takes the usual segment in
// two batches of loads, else four.  169,000 rows of 128 bf16 channels, forward and
// gradient together: in segments of 21 rows 97 us with one wave and 268 us with
// four, of 85 rows (four times as many) 224 us and 207 us; whole rows instead
// of slices cost 2 to 10% more.  No groups: a slice is wider than a workgroup.
WholeArgs whole_args(const tcc_group_norm_shape& s, const WholeWidth& width) {
    const std::uint32_t elem = dtype_bytes(s.dtype), K = s.C / s.G, n = width.n;
    WholeArgs k{};
    k.groupCols = width.spread ? 1 : K / n;
    for (std::uint32_t g = 1; g <= s.G; ++g) {
        if (s.G % g != 0 || g * K % n != 0) continue;
        if (g * K / n > kWholeThreads) break;
        k.groups = g;
        if (g * K * elem >= (s.B < 1024 ? 64 : 128)) break;
    }
    if (k.groups == 0) return k;
    k.slices = s.G / k.groups;
    k.cols = k.groups * K / n;
    while ((1u << k.laneBits) < k.cols) ++k.laneBits;
    const bool wave = s.B >= 1024 && k.cols <= kWave && s.N / s.B <= 2 * kBatch * (kWave >> k.laneBits);
    k.threads = wave ? kWave : kWholeThreads;
    return k;
}

// The width of aligned rows of C elements.
std::uint32_t full_width(std::uint32_t C, std::uint32_t elem) { return RowWidth(C, elem).elems(); }

// Which segments go whole and which tile by tile, from what the host knows.
struct Split {
    std::uint64_t longest;  // rows of a segment that goes whole
    bool whole, tiles;      // whether either kind may occur
    // `width`: elements a lane can take at once, by the rows' alignment
    Split(const tcc_group_norm_shape& s, std::uint32_t width) {
        const std::uint32_t K = s.C / s.G;
        const bool known = s.offsets == nullptr || s.maxRows > 0;
        const std::uint64_t each = s.B > 0 ? s.N / s.B : 0;
        const std::uint64_t most = s.offsets == nullptr ? each : known ? s.maxRows : s.N;
        const WholeArgs k = whole_args(s, WholeWidth(K, full_width(s.C, dtype_bytes(s.dtype))));
        if (k.groups == 0 || whole_args(s, WholeWidth(K, width)).groups == 0) {
            longest = 0;
        } else {
            const std::uint64_t rowLanes = k.threads >> k.laneBits;
            const bool many = s.B >= kMany;
            longest = (many ? kManySteps : kWholeSteps) * rowLanes;
            if (!known && s.N <= kSmallSteps * rowLanes && 2 * each <= longest) longest = s.N;
            else if (!known && (many ? kManyUneven : kUneven) * each > longest) longest = 0;
        }
        tiles = s.N > 0 && (most > longest || s.N > s.B * most);
        if (!tiles) longest = s.N;  // whatever maxRows says
        whole = longest > 0 && (s.offsets != nullptr || most <= longest);
    }
};

// Steps of rowLanes rows that a workgroup of the output takes.  Small workgroups
// move over memory as one front: with the sums' long tiles, a thousand fronts,
// 2.45M x 256 fp32 rows took 1,078 us forward instead of 835.  Lanes of 8
// elements have twice the weights to load before they begin: bf16 rows took
// 458 us with 16 steps and 570 with 4, their gradient 632 with 4 and 946 with 2
// (fp32 rows 940 and 835, 1,283 and 1,260).
// Narrower lanes take as many more steps.
template <typename T, int N>
constexpr std::uint32_t kOutSteps = (N == 8 ? 16 : 4) * (16 / (N * sizeof(T)));
template <typename T, int N>
constexpr std::uint32_t kGradSteps = (N == 8 ? 4 : 2) * (16 / (N * sizeof(T)));

struct Layout {
    std::uint64_t tileRows, tiles, wholeRows;
    std::size_t part, sums, channel, seen, bytes;
    Layout(const tcc_group_norm_shape& s, bool backward) {
        const Split split(s, full_width(s.C, dtype_bytes(s.dtype)));
        const bool unaligned = s.C / s.G > kWholeThreads;  // room for rows that cannot go whole
        // 16 rows of a tile at least and 64 where there are plenty, more where rows
        // are narrow: a tile's own reductions cost about as much (one segment of
        // 91,413 x 32 fp32 rows, gradient, 38 us with tiles of 128, 46 with 64)
        const std::uint64_t rowLanes = kThreads * full_width(s.C, dtype_bytes(s.dtype)) / s.C;
        tileRows = std::max<std::uint64_t>((s.N + kTiles - 1) / kTiles,
                                           std::clamp<std::uint64_t>(s.N / 512, 16, std::max<std::uint64_t>(64, 4 * rowLanes)));
        tiles = split.tiles || unaligned ? (s.N + tileRows - 1) / tileRows : 0;
        wholeRows = split.whole && backward ? std::min(s.B, kWholeBlocks) : 0;
        part = 0;
        std::size_t at = tiles > 0 ? align16((tiles + s.B) * s.G * sizeof(float2)) : 0;
        sums = at;
        channel = at;
        if (backward) {
            if (tiles > 0) at += align16(s.B * s.G * sizeof(float2));
            channel = at;
            at += align16((wholeRows + tiles) * s.C * sizeof(float2));
        }
        seen = at;
        bytes = at + kWholeBlocks;
    }
};

// The rows of a workgroup of the output, doubled until a launch has fewer
// than 2^32 threads (more, HIP takes for the remainder without an error).
std::uint64_t out_rows(std::uint64_t N, std::uint64_t rows) {
    while (N / rows >= (1ull << 32) / kThreads - 1) rows *= 2;
    return rows;
}

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
    TCC_REQUIRE(s->N < (1ull << 32) && s->B <= 0x7FFFFFFFull / s->G, TCC_ERR_UNSUPPORTED, "group norm: too many rows");
    return TCC_OK;
}

// A kernel's form for the activation.
#define TCC_BY_ACT(kernel, T, N, grid, threads, lds, st, ...)                                                   \
    do {                                                                                                        \
        auto* form = a.act == TCC_ACT_NONE   ? &kernel<T, N, TCC_ACT_NONE>                                      \
                     : a.act == TCC_ACT_RELU ? &kernel<T, N, TCC_ACT_RELU>                                      \
                     : a.act == TCC_ACT_SILU ? &kernel<T, N, TCC_ACT_SILU>                                      \
                                             : &kernel<T, N, TCC_ACT_GELU>;                                     \
        hipLaunchKernelGGL(form, grid, dim3(threads), lds, st, __VA_ARGS__);                                    \
    } while (0)

dim3 whole_grid(const WholeArgs& k) { return dim3((k.blocks + 7) / 8 * 8 * k.slices); }

template <typename T, int N>
int whole_launch(const NormArgs& a, WholeArgs k, bool spread, hipStream_t st) {
    if constexpr (N <= 4) {
        if (spread) {
            TCC_BY_ACT(spread_kernel, T, N, whole_grid(k), k.threads, spread_lds<N>(k), st, a, k);
            TCC_LAUNCH_CHECK();
            return TCC_OK;
        }
    }
    TCC_BY_ACT(whole_kernel, T, N, whole_grid(k), k.threads, 2 * k.threads * sizeof(float2), st, a, k);
    TCC_LAUNCH_CHECK();
    return TCC_OK;
}

template <int N>
std::uint32_t grad_lds(std::uint32_t act, std::uint32_t threads) {
    const bool keep = act == TCC_ACT_SILU || act == TCC_ACT_GELU;
    const std::uint32_t floats = keep ? kGradFloats<TCC_ACT_GELU> : kGradFloats<TCC_ACT_NONE>;
    return threads * static_cast<std::uint32_t>(2 * sizeof(float2) + N * floats * sizeof(float));
}

template <typename T, int N>
int whole_grad_launch(const NormArgs& a, WholeArgs k, bool spread, bool params, hipStream_t st) {
    if constexpr (N <= 4) {
        if (spread) {
            TCC_BY_ACT(spread_grad_kernel, T, N, whole_grid(k), k.threads, spread_lds<N>(k), st, a, k,
                       params ? a.channel : nullptr);
            TCC_LAUNCH_CHECK();
            return TCC_OK;
        }
    }
    TCC_BY_ACT(whole_grad_kernel, T, N, whole_grid(k), k.threads, grad_lds<N>(a.act, k.threads), st, a, k,
               params ? a.channel : nullptr);
    TCC_LAUNCH_CHECK();
    return TCC_OK;
}

int stats_join_launch(const NormArgs& a, const Layout& lay, std::uint64_t B, hipStream_t st) {
    if (lay.tiles > 64 * B)
        hipLaunchKernelGGL(stats_join_kernel<4>, JoinGroup<4>::grid(B, a.G),
                           dim3(JoinGroup<4>::threads), 0, st, a);
    else
        hipLaunchKernelGGL(stats_join_kernel<1>, JoinGroup<1>::grid(B, a.G),
                           dim3(JoinGroup<1>::threads), 0, st, a);
    TCC_LAUNCH_CHECK();
    return TCC_OK;
}

template <typename T, int N>
int tiles_launch(NormArgs a, const Layout& lay, std::uint64_t B, hipStream_t st) {
    a.colsV = a.C / N;
    a.rowLanes = std::max<std::uint32_t>(1, kThreads / a.colsV);
    const unsigned tiles = static_cast<unsigned>(lay.tiles);
    hipLaunchKernelGGL((stats_kernel<T, N>), dim3(tiles), dim3(kThreads), 2 * a.rowLanes * a.C * sizeof(float), st, a);
    TCC_LAUNCH_CHECK();
    if (const int rc = stats_join_launch(a, lay, B, st)) return rc;
    a.outRows = out_rows(a.seg.N, kOutSteps<T, N> * a.rowLanes);
    TCC_BY_ACT(apply_kernel, T, N, dim3(grid_for(a.seg.N, static_cast<unsigned>(a.outRows))), kThreads, 0, st, a);
    TCC_LAUNCH_CHECK();
    return TCC_OK;
}

template <typename T, int N>
int tiles_grad_launch(NormArgs a, const Layout& lay, std::uint64_t B, hipStream_t st) {
    a.colsV = a.C / N;
    a.rowLanes = std::max<std::uint32_t>(1, kThreads / a.colsV);
    const unsigned tiles = static_cast<unsigned>(lay.tiles);
    TCC_BY_ACT(grad_sums_kernel, T, N, dim3(tiles), kThreads, 4 * a.rowLanes * a.C * sizeof(float), st, a);
    TCC_LAUNCH_CHECK();
    if (lay.tiles > 64 * B)
        hipLaunchKernelGGL(grad_join_kernel<4>, JoinGroup<4>::grid(B, a.G),
                           dim3(JoinGroup<4>::threads), 0, st, a);
    else
        hipLaunchKernelGGL(grad_join_kernel<1>, JoinGroup<1>::grid(B, a.G),
                           dim3(JoinGroup<1>::threads), 0, st, a);
    TCC_LAUNCH_CHECK();
    a.outRows = out_rows(a.seg.N, kGradSteps<T, N> * a.rowLanes);
    TCC_BY_ACT(grad_apply_kernel, T, N, dim3(grid_for(a.seg.N, static_cast<unsigned>(a.outRows))), kThreads, 0, st, a);
    TCC_LAUNCH_CHECK();
    return TCC_OK;
}

NormArgs base_args(const tcc_group_norm_shape& s, const Layout& lay, const Split& split, void* workspace) {
    NormArgs a{};
    a.seg = Segments{s.offsets, s.N, s.B, s.B > 0 ? s.N / s.B : 0, s.offsetBytes == 8, split.longest};
    char* ws = static_cast<char*>(workspace);
    a.part = reinterpret_cast<float2*>(ws + lay.part);
    a.sums = reinterpret_cast<float2*>(ws + lay.sums);
    a.channel = reinterpret_cast<float2*>(ws + lay.channel);
    a.seen = reinterpret_cast<std::uint8_t*>(ws + lay.seen);
    a.tileRows = lay.tileRows;
    a.C = s.C;
    a.G = s.G;
    a.K = s.C / s.G;
    a.paramType = s.paramDtype;
    a.act = s.activation;
    a.eps = s.eps;
    return a;
}

// CALL(T, N) for an element type and a lane's elements.
#define TCC_BY_TYPE(dtype, n, CALL)                                                                      \
    ((dtype) == TCC_F32    ? ((n) >= 4 ? CALL(float, 4) : (n) >= 2 ? CALL(float, 2) : CALL(float, 1))    \
     : (dtype) == TCC_BF16 ? ((n) >= 8   ? CALL(bf16_t, 8)                                               \
                              : (n) >= 4 ? CALL(bf16_t, 4)                                               \
                              : (n) >= 2 ? CALL(bf16_t, 2)                                               \
                                         : CALL(bf16_t, 1))                                              \
                           : ((n) >= 8   ? CALL(f16_t, 8)                                                \
                              : (n) >= 4 ? CALL(f16_t, 4)                                                \
                              : (n) >= 2 ? CALL(f16_t, 2)                                                \
                                         : CALL(f16_t, 1)))

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
    const std::uint32_t w = RowWidth(s->C, dtype_bytes(s->dtype)).with(x).with(y).stride(ldx).stride(ldy).elems();
    const Split split(*s, w);
    NormArgs a = base_args(*s, lay, split, workspace);
    a.x = x;
    a.ldx = ldx;
    a.weight = weight;
    a.bias = bias;
    a.out = y;
    a.ldo = ldy;
    a.mean = mean;
    a.rstd = rstd;
    const hipStream_t st = as_stream(stream);
    if (split.whole) {
        const WholeWidth width(a.K, w);
        WholeArgs k = whole_args(*s, width);
        k.blocks = static_cast<std::uint32_t>(std::min(s->B, kWholeBlocks));
        if (split.tiles) a.seenCount = k.blocks;
#define CALL(T, N) (whole_launch<T, N>(a, k, width.spread, st))
        if (const int rc = TCC_BY_TYPE(s->dtype, width.n, CALL)) return rc;
#undef CALL
    }
    if (s->N == 0) return stats_join_launch(a, lay, s->B, st);  // segments without rows
    if (!split.tiles) return TCC_OK;
#define CALL(T, N) (tiles_launch<T, N>(a, lay, s->B, st))
    return TCC_BY_TYPE(s->dtype, w, CALL);
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
    const std::uint32_t w = RowWidth(s->C, dtype_bytes(s->dtype)).with(dY).with(x).with(dX).stride(lddy).stride(ldx)
                                .stride(lddx).elems();
    const Split split(*s, w);
    NormArgs a = base_args(*s, lay, split, workspace);
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
    const hipStream_t st = as_stream(stream);
    const bool params = dWeight != nullptr || dBias != nullptr;
    const std::uint64_t wholeRows = split.whole ? lay.wholeRows : 0, tileRows = split.tiles ? lay.tiles : 0;
    if (wholeRows > 0) {
        const WholeWidth width(a.K, w);
        WholeArgs k = whole_args(*s, width);
        k.blocks = static_cast<std::uint32_t>(wholeRows);
        if (split.tiles) a.seenCount = k.blocks;
#define CALL(T, N) (whole_grad_launch<T, N>(a, k, width.spread, params, st))
        if (const int rc = TCC_BY_TYPE(s->dtype, width.n, CALL)) return rc;
#undef CALL
    }
    if (tileRows > 0) {
        NormArgs at = a;
        at.channel += wholeRows * a.C;
#define CALL(T, N) (tiles_grad_launch<T, N>(at, lay, s->B, st))
        if (const int rc = TCC_BY_TYPE(s->dtype, w, CALL)) return rc;
#undef CALL
    }
    if (params) {
        hipLaunchKernelGGL(param_grad_kernel, dim3((a.C + kParamCols - 1) / kParamCols), dim3(kParamCols * kParamRows), 0,
                           st, a, wholeRows, tileRows, dWeight, dBias);
        TCC_LAUNCH_CHECK();
    }
    return TCC_OK;
}

}  // extern "C"
