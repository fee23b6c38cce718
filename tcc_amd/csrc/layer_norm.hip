// Layer norm of node rows with the sum before it and the activation after it
// (include/tcc_training.h).
//
//   h = x + residual (rounded to x's type), over the C channels of a row:
//   mean = sum h / C,  rstd = 1 / sqrt(sum (h - mean)^2 / C + eps)
//   z = ((h - mean) * rstd) * weight + bias,  y = act(z)
//
// and with dz = dY act'(z), xh = (h - mean) rstd, a = dz weight:
//   dBias = sum dz,  dWeight = sum dz xh  over the rows
//   dX = rstd (a - (sum a + xh sum a xh) / C) + dSum
//
// A team of lanes holds a row in registers, so that memory is read once: 16
// bytes a lane at a time, whatever the alignment (the last vector of a row that
// does not divide into them is moved back to end with it; what it shares with
// the one before counts once in every sum, and is written twice with the same
// value).  Teams are as small as 16 elements a lane allow, which saves
// reductions: four lanes of a wave to the 1,024 threads of a workgroup.
// A lane adds its elements in pairs, and the lanes' sums are added in 64 bits: the
// mean comes out rounded once for most rows.  The variance is the mean square of
// the differences from that, less the square of their mean, which is what rows
// far from zero have lost.
//
// The gradient's teams walk the rows in equal steps and keep the sums of dz and
// dz xh of their channels in registers, of a dozen rows at a time; a workgroup adds
// them in LDS in 64 bits, where rows of up to 8,192 channels have room for that (longer
// ones: up to four runs of rows, each written), and a second kernel adds what the
// workgroups wrote.
#include <algorithm>

#include "../../include/tcc_swtcf.h"
#include "../../include/tcc_training.h"
#include "activations.hpp"
#include "row_types.hpp"
#include "teams.hpp"

namespace tcc {
namespace {

constexpr std::uint32_t kMaxChannels = 16384;
constexpr int kTotalChannels = 8192;  // whose parameters' sums have room in LDS, 128 KB

struct Args {
    const void *x, *residual, *dy, *dSum, *weight, *bias;
    void *out, *sum;  // y or dx, h
    float *mean, *rstd;
    float* part;  // [runs][workgroups][2][C], dBias and dWeight
    std::uint64_t runRows;  // rows of a team in each of its runs
    std::uint64_t N, ldx, ldr, lddy, ldds, ldo, lds;
    std::uint32_t C, paramType, act, runs;
    float eps;
};

template <int TEAM>
constexpr int kThreads = TEAM > 256 ? TEAM : 256;
template <int TEAM>
constexpr int kTeams = kThreads<TEAM> / TEAM;  // of a workgroup

// The channels that a lane holds of every row: E vectors of V.
template <int V, int E, int TEAM>
struct Columns {
    std::uint32_t c[E];     // first channel
    std::uint32_t skip[E];  // elements that are another vector's (all: no vector)
    __device__ __forceinline__ explicit Columns(std::uint32_t C) {
        const std::uint32_t lane = threadIdx.x % TEAM;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const std::uint32_t at = (lane + e * TEAM) * V;
            c[e] = min(at, C - V);
            skip[e] = min(at - c[e], static_cast<std::uint32_t>(V));
        }
    }
    __device__ __forceinline__ bool any(int e) const { return skip[e] < V; }
    // v with 0 where another vector counts.
    __device__ __forceinline__ vec_t<float, V> own(int e, vec_t<float, V> v) const {
        if (skip[e] != 0) {
#pragma unroll
            for (int q = 0; q < V; ++q) v[q] = static_cast<std::uint32_t>(q) < skip[e] ? 0.0f : v[q];
        }
        return v;
    }
};

template <std::uint32_t ACT, bool FINE, int N>
__device__ __forceinline__ vec_t<float, N> activate_all(vec_t<float, N> z) {
#pragma unroll
    for (int q = 0; q < N; ++q) z[q] = activate<ACT, FINE>(z[q]);
    return z;
}
template <bool FINE, int N>
__device__ __forceinline__ vec_t<float, N> activate_by(std::uint32_t act, vec_t<float, N> z) {
    if (act == TCC_ACT_NONE) return z;
    if (act == TCC_ACT_RELU) return activate_all<TCC_ACT_RELU, FINE, N>(z);
    if (act == TCC_ACT_SILU) return activate_all<TCC_ACT_SILU, FINE, N>(z);
    return activate_all<TCC_ACT_GELU, FINE, N>(z);
}
template <std::uint32_t ACT, bool FINE, int N>
__device__ __forceinline__ vec_t<float, N> through_all(vec_t<float, N> d, vec_t<float, N> z) {
#pragma unroll
    for (int q = 0; q < N; ++q) d[q] = through<ACT, FINE>(d[q], z[q]);
    return d;
}
template <bool FINE, int N>
__device__ __forceinline__ vec_t<float, N> through_by(std::uint32_t act, vec_t<float, N> d, vec_t<float, N> z) {
    if (act == TCC_ACT_NONE) return d;
    if (act == TCC_ACT_RELU) return through_all<TCC_ACT_RELU, FINE, N>(d, z);
    if (act == TCC_ACT_SILU) return through_all<TCC_ACT_SILU, FINE, N>(d, z);
    return through_all<TCC_ACT_GELU, FINE, N>(d, z);
}

// The sum of N elements, pairs before pairs of pairs.
template <int N, typename A>
__device__ __forceinline__ float in_pairs(const A& v) {
    float s[N];
#pragma unroll
    for (int q = 0; q < N; ++q) s[q] = v[q];
#pragma unroll
    for (int d = 1; d < N; d <<= 1)
#pragma unroll
        for (int q = 0; q + d < N; q += 2 * d) s[q] += s[q + d];
    return s[0];
}

// Rounded to T, as memory holds it.
template <typename T, int N>
__device__ __forceinline__ vec_t<float, N> rounded(vec_t<float, N> v) {
    return __builtin_convertvector(__builtin_convertvector(v, vec_t<T, N>), vec_t<float, N>);
}

// A lane's elements of a row as memory holds them.
template <typename T, int V, int E, int TEAM, bool ONCE>
struct Raw {
    vec_t<T, V> v[E];
    __device__ __forceinline__ void load(const void* p, std::uint64_t at, const Columns<V, E, TEAM>& cols) {
        const T* row = static_cast<const T*>(p) + at;
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = cols.any(e) ? load_as<T, V, ONCE>(row + cols.c[e]) : vec_t<T, V>(static_cast<T>(0.0f));
    }
    __device__ __forceinline__ vec_t<float, V> operator[](int e) const { return __builtin_convertvector(v[e], vec_t<float, V>); }
};
// Whether there are registers for the next row's elements beside this one's: the
// gradient of 169,000 x 301 bf16 rows took 92 us with and 145 without.
template <typename T, int V, int E, int TEAM>
constexpr bool kAhead = E * V * sizeof(T) <= 32 && TEAM <= 256;

// Bound by memory: x and residual in, y and h out, once.  2.45M x 256 fp32 rows with
// a residual take 1,822 us (10.05 GB: 5.5 TB/s, where a copy of 4 GiB has 4.6),
// 16,384 x 4,096 bf16 rows with one 101 (537 MB: 5.3 TB/s).
template <typename T, int V, int E, int TEAM, bool ONCE>
__global__ void __launch_bounds__(kThreads<TEAM>) forward_kernel(Args a) {
    using F = vec_t<float, V>;
    __shared__ typename TeamSum<TEAM>::Shared shared;
    TeamSum<TEAM> sum(shared);
    const Columns<V, E, TEAM> cols(a.C);
    F w[E], b[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (!cols.any(e)) continue;
        w[e] = load_params<V>(a.weight, a.paramType, cols.c[e], 1.0f);
        b[e] = load_params<V>(a.bias, a.paramType, cols.c[e], 0.0f);
    }
    const double perC = 1.0 / a.C;
    const float inverse = static_cast<float>(perC);
    const std::uint64_t step = static_cast<std::uint64_t>(gridDim.x) * kTeams<TEAM>;
    std::uint64_t r = static_cast<std::uint64_t>(blockIdx.x) * kTeams<TEAM> + threadIdx.x / TEAM;
    Raw<T, V, E, TEAM, ONCE> x, res;
    const auto load = [&](std::uint64_t row) {
        if (row >= a.N) return;
        x.load(a.x, row * a.ldx, cols);
        if (a.residual != nullptr) res.load(a.residual, row * a.ldr, cols);
    };
    if constexpr (kAhead<T, V, E, TEAM>) load(r);
    for (; r < a.N; r += step) {
        if constexpr (!kAhead<T, V, E, TEAM>) load(r);
        F h[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            h[e] = x[e];
            if (a.residual != nullptr) h[e] = rounded<T, V>(h[e] + res[e]);
        }
        if constexpr (kAhead<T, V, E, TEAM>) load(r + step);
        float pairs[E];
#pragma unroll
        for (int e = 0; e < E; ++e) pairs[e] = in_pairs<V>(cols.own(e, h[e]));
        const double mean64 = sum(static_cast<double>(in_pairs<E>(pairs))) * perC;
        const float mean = static_cast<float>(mean64);
        float left = 0.0f, squares = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const F d = cols.own(e, h[e] - mean);
#pragma unroll
            for (int q = 0; q < V; ++q) {
                left += d[q];
                squares = fmaf(d[q], d[q], squares);
            }
        }
        const float2 both = sum(left, squares);
        const float off = both.x * inverse, var = fmaf(-off, off, both.y * inverse);
        const float rstd = 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + a.eps);  // keeps NaN
        T* y = static_cast<T*>(a.out) + r * a.ldo;
        T* s = static_cast<T*>(a.sum) + r * a.lds;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (!cols.any(e)) continue;
            if (a.sum != nullptr) store_any<T, V, ONCE>(s + cols.c[e], h[e]);
            F z;
#pragma unroll
            for (int q = 0; q < V; ++q) z[q] = affine(normalise(h[e][q], mean, rstd), w[e][q], b[e][q]);
            store_any<T, V, ONCE>(y + cols.c[e], activate_by<kFine<T>, V>(a.act, z));
        }
        if (threadIdx.x % TEAM == 0) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
    }
}

// The parameters' sums of a workgroup, in 64 bits: those of a wave's teams are added
// over its lanes, and each wave (or larger team) has a place of its own where these
// take 32 KB at most, else two waves have one.  A place has a pair, dBias and dWeight,
// for each element of the lanes' vectors (not for each channel).
template <int V, int E, int TEAM>
struct Totals {
    static constexpr bool used = TEAM * E * V <= kTotalChannels;
    static constexpr int group = TEAM < kWave ? kWave : TEAM, groups = kThreads<TEAM> / group;
    static constexpr int sums = used ? 2 * TEAM * E * V : 1;
    static constexpr int places = groups == 1 || groups * sums * sizeof(double) <= 32768 ? groups : groups / 2;
    struct Shared {
        double sum[places][sums] __attribute__((aligned(16)));
    };
    Shared& s;
    __device__ __forceinline__ explicit Totals(Shared& shared) : s(shared) {}

    // a and b of the lanes at distance D (16 or 32) and this one added: of a where bit D
    // of the lane is 0, of b where it is 1.
    template <int D>
    static __device__ __forceinline__ double halves(double a, double b) {
        const auto x = static_cast<std::uint64_t>(__double_as_longlong(a)), y = static_cast<std::uint64_t>(__double_as_longlong(b));
        std::uint32_t first[2], second[2];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const auto xs = static_cast<std::uint32_t>(x >> (32 * w)), ys = static_cast<std::uint32_t>(y >> (32 * w));
            if constexpr (D == 16) {
                const auto r = __builtin_amdgcn_permlane16_swap(xs, ys, false, false);
                first[w] = r[0], second[w] = r[1];
            } else {
                const auto r = __builtin_amdgcn_permlane32_swap(xs, ys, false, false);
                first[w] = r[0], second[w] = r[1];
            }
        }
        const auto whole = [](const std::uint32_t (&w)[2]) {
            return __longlong_as_double(static_cast<long long>(static_cast<std::uint64_t>(w[1]) << 32 | w[0]));
        };
        return whole(first) + whole(second);
    }
    template <int D>
    static __device__ __forceinline__ double with_other(double v) {
        return v + __longlong_as_double(static_cast<long long>(other<D>(static_cast<std::uint64_t>(__double_as_longlong(v)))));
    }

    // Takes in a lane's sums; the whole workgroup.
    __device__ __forceinline__ void add(bool first, const vec_t<float, V> (&db)[E], const vec_t<float, V> (&dw)[E]) {
        const int mine = threadIdx.x / group;
        const std::uint32_t lane = __lane_id();
        double* to = s.sum[mine % places] + threadIdx.x % TEAM * V * 2;
#pragma unroll 1
        for (int phase = 0; phase < groups / places; ++phase) {
            const auto put = [&](auto* p, auto v) { *p = first && phase == 0 ? v : v + *p; };
            if (mine / places == phase) {
                // pairs of elements, two at a time for their registers
#pragma unroll
                for (int i = 0; i < E * V; i += 2) {
                    constexpr int apart = V == 1 ? TEAM : 1;  // of the second element from the first
                    const int e0 = i / V, e1 = (i + 1) / V;
                    double* at = to + (e0 * TEAM * V + i % V) * 2;
                    const double b0 = db[e0][i % V], w0 = dw[e0][i % V], b1 = db[e1][(i + 1) % V], w1 = dw[e1][(i + 1) % V];
                    if constexpr (TEAM >= kWave) {
                        static_assert(V > 1);
                        put(reinterpret_cast<vec_t<double, 2>*>(at), vec_t<double, 2>{b0, w0});
                        put(reinterpret_cast<vec_t<double, 2>*>(at + 2), vec_t<double, 2>{b1, w1});
                    } else if constexpr (TEAM == 32) {
                        put(at + lane / 32, halves<32>(b0, w0));
                        put(at + lane / 32 + 2 * apart, halves<32>(b1, w1));
                    } else {  // each row of 16 lanes has one of the four
                        double v = halves<16>(halves<32>(b0, w0), halves<32>(b1, w1));
                        if constexpr (TEAM <= 4) v = with_other<4>(v);
                        if constexpr (TEAM <= 8) v = with_other<8>(v);
                        if (lane % 16 < TEAM) put(at + lane / 32 + (lane / 16 % 2) * 2 * apart, v);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if constexpr (places < groups) __syncthreads();
        }
    }
    // Writes dBias and dWeight of all C channels; the whole workgroup.
    __device__ __forceinline__ void write(float* to, std::uint32_t C) const {
        __syncthreads();
        const std::uint32_t body = C / V * V;
        for (std::uint32_t i = threadIdx.x; i < 2 * C; i += kThreads<TEAM>) {
            const std::uint32_t k = i < C ? 0 : 1, c = i - k * C, element = c < body ? c : c - C + V + body;
            double v = 0.0;
#pragma unroll
            for (int p = 0; p < places; ++p) v += s.sum[p][2 * element + k];
            to[i] = static_cast<float>(v);
        }
    }
};

// Bound by memory, and by vector instructions where 16-bit rows have an activation:
// 2.45M x 256 fp32 rows with d_sum and relu take 1,781 us (10.04 GB: 5.6 TB/s),
// 169,000 x 301 bf16 rows with gelu 84 (305 MB: 3.6 TB/s), both with the parameters'
// kernel.
template <typename T, int V, int E, int TEAM, bool ONCE>
__global__ void __launch_bounds__(kThreads<TEAM>) grad_kernel(Args a) {
    using F = vec_t<float, V>;
    __shared__ typename TeamSum<TEAM>::Shared shared;
    TeamSum<TEAM> sum(shared);
    __shared__ typename Totals<V, E, TEAM>::Shared sums;
    Totals<V, E, TEAM> totals(sums);
    const Columns<V, E, TEAM> cols(a.C);
    F w[E], b[E], dw[E], db[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        dw[e] = db[e] = F(0.0f);
        if (!cols.any(e)) continue;
        w[e] = load_params<V>(a.weight, a.paramType, cols.c[e], 1.0f);
        b[e] = load_params<V>(a.bias, a.paramType, cols.c[e], 0.0f);
    }
    const float perC = 1.0f / static_cast<float>(a.C);
    const std::uint64_t step = static_cast<std::uint64_t>(gridDim.x) * kTeams<TEAM>;
    std::uint64_t r = static_cast<std::uint64_t>(blockIdx.x) * kTeams<TEAM> + threadIdx.x / TEAM;
    Raw<T, V, E, TEAM, ONCE> x, dy;
    float mean = 0.0f, rstd = 0.0f;
    const auto load = [&](std::uint64_t row) {
        if (row >= a.N) return;
        x.load(a.x, row * a.ldx, cols);
        dy.load(a.dy, row * a.lddy, cols);
        mean = a.mean[row];
        rstd = a.rstd[row];
    };
    if constexpr (kAhead<T, V, E, TEAM>) load(r);
    for (std::uint32_t run = 0; run < a.runs; ++run) {
        for (std::uint64_t i = 0; i < a.runRows && r < a.N; ++i, r += step) {
            if constexpr (!kAhead<T, V, E, TEAM>) load(r);
            F xh[E], dz[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                xh[e] = x[e];
                dz[e] = dy[e];
            }
            const float m = mean, rs = rstd;
            if constexpr (kAhead<T, V, E, TEAM>) load(r + step);
            float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (!cols.any(e)) continue;
                F z;
#pragma unroll
                for (int q = 0; q < V; ++q) {
                    xh[e][q] = normalise(xh[e][q], m, rs);
                    z[q] = affine(xh[e][q], w[e][q], b[e][q]);
                }
                dz[e] = through_by<kFine<T>, V>(a.act, dz[e], z);
                const F d = cols.own(e, dz[e]);
                db[e] += d;
#pragma unroll
                for (int q = 0; q < V; ++q) {
                    const float dx = d[q] * xh[e][q];
                    dw[e][q] += dx;
                    s1 = fmaf(d[q], w[e][q], s1);
                    s2 = fmaf(dx, w[e][q], s2);
                }
            }
            const float2 both = sum(s1, s2);
            const float m1 = both.x * perC, m2 = both.y * perC;
            T* out = static_cast<T*>(a.out) + r * a.ldo;
            const T* add = static_cast<const T*>(a.dSum) + r * a.ldds;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (!cols.any(e)) continue;
                F v;
#pragma unroll
                for (int q = 0; q < V; ++q) v[q] = rs * (fmaf(dz[e][q], w[e][q], -m1) - xh[e][q] * m2);
                if (a.dSum != nullptr) v += load_any<T, V, ONCE>(add + cols.c[e]);
                store_any<T, V, ONCE>(out + cols.c[e], v);
            }
        }
        if (a.part == nullptr) continue;
        if constexpr (!Totals<V, E, TEAM>::used) {
            float* to = a.part + (static_cast<std::uint64_t>(run) * gridDim.x + blockIdx.x) * 2 * a.C;
#pragma unroll
            for (int e = 0; e < E; ++e)
#pragma unroll
                for (int q = 0; q < V; ++q)
                    if (static_cast<std::uint32_t>(q) >= cols.skip[e]) {
                        to[cols.c[e] + q] = db[e][q];
                        to[a.C + cols.c[e] + q] = dw[e][q];
                    }
        } else {
            totals.add(run == 0, db, dw);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) dw[e] = db[e] = F(0.0f);
    }
    if constexpr (Totals<V, E, TEAM>::used) {
        if (a.part != nullptr) totals.write(a.part + static_cast<std::uint64_t>(blockIdx.x) * 2 * a.C, a.C);
    }
}

// dBias and dWeight: the workgroups' sums added in 64 bits, kParamCols columns a
// workgroup (4 to 11 us).
constexpr std::uint32_t kParamCols = 8, kParamRows = 128;
__global__ void __launch_bounds__(kParamCols* kParamRows) params_kernel(const float* part, std::uint32_t parts,
                                                                        std::uint32_t C, float* dBias, float* dWeight) {
    const std::uint32_t i = blockIdx.x * kParamCols + threadIdx.x % kParamCols, first = threadIdx.x / kParamCols;
    double v = 0.0;
    if (i < 2 * C)
#pragma unroll 4
        for (std::uint32_t p = first; p < parts; p += kParamRows) v += part[static_cast<std::uint64_t>(p) * 2 * C + i];
    __shared__ double all[kParamRows][kParamCols];
    all[first][threadIdx.x % kParamCols] = v;
    __syncthreads();
    if (first != 0 || i >= 2 * C) return;
#pragma unroll 8
    for (std::uint32_t k = 1; k < kParamRows; ++k) v += all[k][threadIdx.x];
    float* to = i < C ? dBias : dWeight;
    if (to != nullptr) to[i < C ? i : i - C] = static_cast<float>(v);
}

// ---------------------------------------------------------------- launches

// The smallest team that holds rows of C elements; f is called with its <V, E,
// TEAM>.  Sixteen elements a lane at most.  Rows of 257 to 384 and of 513 to 768
// 16-bit elements, of which vectors of 16 bytes would leave up to half of a team's
// lanes without any, take 8 bytes a lane: the gradient of 169,000 x 301 bf16 rows with
// gelu, half of whose time is vector instructions, took 92 us instead of 104.
// (Others whose last vectors are few keep 16 bytes: 6.25M x 16 rows take 116 us,
// 66,666 x 1,500 ones 113, where a copy takes 98 and 87.)
template <typename T, typename F>
void with_team(std::uint32_t C, F f) {
    constexpr int V = kVec<T>;
    const auto fits = [&](std::uint64_t v, std::uint64_t e, std::uint64_t team) { return C <= team * e * v; };
    if (C < V) return f.template operator()<1, 2, 4>();
    if (fits(V, 1, 4)) return f.template operator()<V, 1, 4>();
    if (fits(V, 1, 8)) return f.template operator()<V, 1, 8>();
    if (fits(V, 1, 16)) return f.template operator()<V, 1, 16>();
    if (fits(V, 2, 16)) return f.template operator()<V, 2, 16>();
    if constexpr (V == 4) {
        if (fits(4, 3, 16)) return f.template operator()<4, 3, 16>();
        if (fits(4, 4, 16)) return f.template operator()<4, 4, 16>();
    }
    if (fits(4, 3, 32)) return f.template operator()<4, 3, 32>();
    if (fits(4, 2, 64)) return f.template operator()<V, 8 / V, 64>();
    if (fits(4, 3, 64)) return f.template operator()<4, 3, 64>();
    if (fits(4, 4, 64)) return f.template operator()<V, 16 / V, 64>();
    if (fits(4, 2, 256)) return f.template operator()<V, 8 / V, 256>();
    if (fits(4, 4, 256)) return f.template operator()<V, 16 / V, 256>();
    if (fits(4, 4, 512)) {  // the gradient has registers for two waves of 16 elements a lane on a SIMD, no more
        if constexpr (F::forward) return f.template operator()<V, 16 / V, 512>();
        else return f.template operator()<V, 8 / V, 1024>();
    }
    return f.template operator()<V, 16 / V, 1024>();
}

// Rows past what the caches hold are read and written past their order: 2.45M x
// 256 fp32 rows with a residual in 1,820 us instead of 1,870, their gradient in
// 4% less time than otherwise.
template <typename T>
bool once(const Args& a) { return a.N * a.C * sizeof(T) > kCacheBytes; }

template <typename T>
struct Forward {
    static constexpr bool forward = true;
    const Args& a;
    hipStream_t st;
    template <int V, int E, int TEAM>
    void operator()() const {
        // four rows a team where there are plenty, for one reading of the parameters
        const std::uint64_t all = (a.N + kTeams<TEAM> - 1) / kTeams<TEAM>;
        const std::uint64_t blocks = std::min<std::uint64_t>(std::min<std::uint64_t>(all, std::max<std::uint64_t>(all / 4, 2048)), 1u << 21);
        const dim3 grid(static_cast<unsigned>(blocks));
        if (once<T>(a)) hipLaunchKernelGGL((forward_kernel<T, V, E, TEAM, true>), grid, dim3(kThreads<TEAM>), 0, st, a);
        else hipLaunchKernelGGL((forward_kernel<T, V, E, TEAM, false>), grid, dim3(kThreads<TEAM>), 0, st, a);
    }
};

// The gradient's workgroups are as many as run at once, with equal shares of the
// rows (three or four times as many took 40 us more for 2.45M x 256 fp32 rows).  A
// team sums a run of its rows in 32 bits, which loses digits by the root of the run's
// length: dWeight of these is off by 0.8e-7 with runs of 8 rows, 1.0e-7 with 12 and
// 1.5e-7 with 50 (64-bit sums: 0.5e-7).  16-bit rows are read in half the time, of
// which runs of 8 take 1 to 4% more than those of 12.
constexpr std::uint64_t kMostRuns = 4;
template <typename T>
constexpr std::uint64_t kRun = sizeof(T) == 4 ? 8 : 12;
constexpr std::uint64_t kLongRun = 96;

// The most of them, for which the workspace is: no compute unit runs more of their
// size and registers at once.
std::uint64_t most_blocks(std::uint32_t C) { return (C <= 1024 ? 8ull : C <= 4096 ? 4ull : 1ull) * device_cus(); }
template <typename T>
struct Backward {
    static constexpr bool forward = false;
    const Args& a;
    hipStream_t st;
    std::uint64_t& parts;
    template <int V, int E, int TEAM, bool ONCE>
    void launch() const {
        static std::uint32_t perCu;
        const auto kernel = grad_kernel<T, V, E, TEAM, ONCE>;
        const std::uint64_t blocks = std::min<std::uint64_t>(
            {(a.N + kTeams<TEAM> - 1) / kTeams<TEAM>, resident_blocks(kernel, kThreads<TEAM>, perCu), most_blocks(a.C)});
        Args k = a;
        const std::uint64_t rows = (a.N + blocks * kTeams<TEAM> - 1) / (blocks * kTeams<TEAM>);
        constexpr bool totals = Totals<V, E, TEAM>::used;
        const std::uint64_t runs = totals ? rows / kRun<T> : std::min(rows / kLongRun, kMostRuns);
        k.runs = a.part == nullptr || runs == 0 ? 1u : static_cast<std::uint32_t>(runs);
        k.runRows = (rows + k.runs - 1) / k.runs;
        parts = totals ? blocks : blocks * k.runs;
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads<TEAM>), 0, st, k);
    }
    template <int V, int E, int TEAM>
    void operator()() const {
        if (once<T>(a)) launch<V, E, TEAM, true>();
        else launch<V, E, TEAM, false>();
    }
};

int check_shape(const tcc_layer_norm_shape* s) {
    TCC_REQUIRE(s != nullptr, TCC_ERR_INVALID_ARGUMENT, "layer norm: no shape");
    TCC_REQUIRE(s->C >= 1, TCC_ERR_INVALID_ARGUMENT, "layer norm: rows have channels");
    TCC_REQUIRE(dtype_bytes(s->dtype) != 0 && dtype_bytes(s->paramDtype) != 0, TCC_ERR_INVALID_ARGUMENT,
                "layer norm: unknown element type");
    TCC_REQUIRE(s->activation <= TCC_ACT_GELU, TCC_ERR_INVALID_ARGUMENT, "layer norm: unknown activation");
    TCC_REQUIRE(s->eps >= 0.0f, TCC_ERR_INVALID_ARGUMENT, "layer norm: eps is not negative");
    TCC_REQUIRE(s->C <= kMaxChannels, TCC_ERR_UNSUPPORTED, "layer norm: at most 16384 channels");
    TCC_REQUIRE(s->N < (1ull << 40), TCC_ERR_UNSUPPORTED, "layer norm: fewer than 2^40 rows");
    return TCC_OK;
}

Args args_of(const tcc_layer_norm_shape& s) {
    Args a{};
    a.N = s.N;
    a.C = s.C;
    a.paramType = s.paramDtype;
    a.act = s.activation;
    a.eps = s.eps;
    return a;
}

template <template <typename> class Launch, typename... More>
void launch_typed(std::uint32_t dtype, const Args& a, hipStream_t st, More&... more) {
    if (dtype == TCC_F32) with_team<float>(a.C, Launch<float>{a, st, more...});
    else if (dtype == TCC_BF16) with_team<bf16_t>(a.C, Launch<bf16_t>{a, st, more...});
    else with_team<f16_t>(a.C, Launch<f16_t>{a, st, more...});
}

}  // namespace
}  // namespace tcc

extern "C" int tcc_layer_norm(const tcc_layer_norm_shape* s, const void* x, uint64_t ldx, const void* residual,
                              uint64_t ldr, const void* weight, const void* bias, void* y, uint64_t ldy, void* sum,
                              uint64_t lds, float* mean, float* rstd, void* stream) {
    using namespace tcc;
    clear_last_error();
    if (const int rc = check_shape(s)) return rc;
    if (s->N == 0) return TCC_OK;
    TCC_REQUIRE(x != nullptr && y != nullptr && mean != nullptr && rstd != nullptr, TCC_ERR_INVALID_ARGUMENT,
                "layer norm: a null pointer");
    TCC_REQUIRE(ldx >= s->C && ldy >= s->C && (residual == nullptr || ldr >= s->C) && (sum == nullptr || lds >= s->C),
                TCC_ERR_INVALID_ARGUMENT, "layer norm: a row stride below the channels");
    Args a = args_of(*s);
    a.x = x;
    a.ldx = ldx;
    a.residual = residual;
    a.ldr = ldr;
    a.weight = weight;
    a.bias = bias;
    a.out = y;
    a.ldo = ldy;
    a.sum = sum;
    a.lds = lds;
    a.mean = mean;
    a.rstd = rstd;
    launch_typed<Forward>(s->dtype, a, as_stream(stream));
    TCC_LAUNCH_CHECK();
    return TCC_OK;
}

extern "C" size_t tcc_layer_norm_grad_workspace_bytes(const tcc_layer_norm_shape* s) {
    using namespace tcc;
    if (check_shape(s) != TCC_OK) return 0;
    // the most workgroups of any team, which has one row or more
    const std::uint64_t runs = s->C <= kTotalChannels ? 1 : kMostRuns;
    return std::min<std::uint64_t>(s->N, most_blocks(s->C)) * runs * 2 * s->C * sizeof(float);
}

extern "C" int tcc_layer_norm_grad(const tcc_layer_norm_shape* s, const void* dY, uint64_t lddy, const void* h,
                                   uint64_t ldh, const float* mean, const float* rstd, const void* weight,
                                   const void* bias, const void* dSum, uint64_t ldds, void* dX, uint64_t lddx,
                                   float* dWeight, float* dBias, void* workspace, size_t workspaceBytes, void* stream) {
    using namespace tcc;
    clear_last_error();
    if (const int rc = check_shape(s)) return rc;
    TCC_REQUIRE(s->N == 0 || (dY != nullptr && h != nullptr && dX != nullptr && mean != nullptr && rstd != nullptr),
                TCC_ERR_INVALID_ARGUMENT, "layer norm gradient: a null pointer");
    TCC_REQUIRE(lddy >= s->C && ldh >= s->C && lddx >= s->C && (dSum == nullptr || ldds >= s->C),
                TCC_ERR_INVALID_ARGUMENT, "layer norm gradient: a row stride below the channels");
    const bool params = dWeight != nullptr || dBias != nullptr;
    TCC_REQUIRE(!params || s->N == 0 ||
                    (workspace != nullptr && (reinterpret_cast<std::uintptr_t>(workspace) & 15) == 0 &&
                     workspaceBytes >= tcc_layer_norm_grad_workspace_bytes(s)),
                TCC_ERR_INVALID_ARGUMENT, "layer norm gradient: the workspace is too small or not 16-byte aligned");
    Args a = args_of(*s);
    a.dy = dY;
    a.lddy = lddy;
    a.x = h;
    a.ldx = ldh;
    a.mean = const_cast<float*>(mean);
    a.rstd = const_cast<float*>(rstd);
    a.weight = weight;
    a.bias = bias;
    a.dSum = dSum;
    a.ldds = ldds;
    a.out = dX;
    a.ldo = lddx;
    a.part = params ? static_cast<float*>(workspace) : nullptr;
    std::uint64_t parts = 0;
    if (s->N > 0) {
        launch_typed<Backward>(s->dtype, a, as_stream(stream), parts);
        TCC_LAUNCH_CHECK();
    }
    if (params) {
        hipLaunchKernelGGL(params_kernel, dim3(grid_for(2ull * s->C, kParamCols)), dim3(kParamCols * kParamRows), 0,
                           as_stream(stream), a.part, static_cast<std::uint32_t>(parts), s->C, dBias, dWeight);
        TCC_LAUNCH_CHECK();
    }
    return TCC_OK;
}
