// Distillation from a teacher's top logits: the loss and its gradient
// (include/tcc_training.h).
//
// A row has logits z of all C classes and K entries (value t_k, class id_k) of
// its teacher, with one more value r for all other classes where `rest` is
// given.  With temperature T, over the entries (and r) and over the classes
//   p = softmax(t / T),   q = softmax(z / T),   q_r = sum of q over the others
//   loss = w T^2 (sum_k p_k log(p_k / q_id_k) + p_r log(p_r / q_r))
//   dz_j = g w T (q_j - p_k)            for j = id_k
//          g w T (q_j - p_r q_j / q_r)  for the others (p_r = 0 without r)
//
// A team of lanes takes a row: 4, 16 or 64 of a wave, or a workgroup of 256.
// Each lane keeps the maximum of what it read and the sum of
// exp((z - maximum) / T), rescaled when the maximum rises, so that a row is
// read once.  Everything is in base 2 with one factor log2(e) / T, rounded
// once: the differences z - m are formed first, and p and q are those of a
// temperature that is the same for both.  What rest needs, the classes that are
// no id, is summed by itself (a difference of sums would lose what a
// confident student leaves them): one bit of a class in LDS says that it is an
// id, and their logits are taken out of the stream and added afterwards.
// The gradient's stream leaves out the ids in the same way, and the lanes that
// hold the entries write there.
#include <algorithm>

#include "../../include/tcc_spmm_cnic.h"
#include "../../include/tcc_swtcf.h"
#include "../../include/tcc_training.h"
#include "logits.hpp"
#include "teams.hpp"

namespace tcc {
namespace {

constexpr std::uint32_t kMaxEntries = 64;
constexpr int kThreads = 256;
constexpr int kBatch = 4;  // vectors that a lane loads before it uses the first

struct Args {
    const void *z, *values, *ids;
    const float *rest, *weight;
    float4* stats;
    float* loss;             // rows, where nothing is summed
    double2* part;           // [workgroups]: weighted losses, weights
    const float *dLoss, *total;
    void* dz;
    std::uint32_t* error;
    std::uint64_t n, ldz, ldv, ldi, ldd;
    std::uint32_t C, K, valueType, idBytes, reduction;
    float T, c;  // c = log2(e) / T
};

// Lanes of a team wait for each other's LDS.
template <int TEAM>
__device__ __forceinline__ void team_sync() {
    if constexpr (TEAM > kWave) {
        __syncthreads();
    } else {  // a wave's LDS operations run in order
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

template <int TEAM>
constexpr int kEntries = TEAM >= 64 ? 1 : 4;  // of a lane; TEAM * kEntries >= K

template <int TEAM>
constexpr int kTeams = kThreads / TEAM;

// Classes whose bits a team holds at once, a multiple of 32.
template <int TEAM>
constexpr std::uint32_t kWindow = TEAM == 4 ? 128 : TEAM == 16 ? 512 : TEAM == 64 ? 4096 : 1u << 17;

// LDS of the workgroup.
template <int TEAM>
struct Shared {
    std::uint32_t bits[kTeams<TEAM>][kWindow<TEAM> / 32 + 1];  // a word more, for the reads at the end
    float2 part[2][TEAM > kWave ? TEAM / kWave : 1];
    float2 one[2];
    double2 sums[kThreads / kWave];
};

// One team at its rows.
template <int TEAM>
struct Team {
    static constexpr int inWave = TEAM < kWave ? TEAM : kWave;
    Shared<TEAM>& lds;
    const Args& a;
    std::uint32_t* bits;
    std::uint32_t lane;
    int turn = 0, row = 0;  // places in LDS alternate, so that one barrier a use is enough
    __device__ __forceinline__ Team(Shared<TEAM>& shared, const Args& args)
        : lds(shared), a(args), bits(shared.bits[threadIdx.x / TEAM]), lane(threadIdx.x % TEAM) {}

    // The entries of a row: lane + e TEAM < K.  Only the first wave of a
    // workgroup holds any.
    std::int64_t id[kEntries<TEAM>];  // -1: no entry
    float t[kEntries<TEAM>], p[kEntries<TEAM>];
    float top, sum, pRest, rest;  // of the teacher's values
    bool twice;  // some id occurs again

    __device__ __forceinline__ std::int64_t id_at(std::uint64_t r, std::uint32_t k) const {
        const std::uint64_t at = r * a.ldi + k;
        return a.idBytes == 8 ? load_global<std::int64_t>(static_cast<const std::int64_t*>(a.ids) + at)
                              : load_global<std::int32_t>(static_cast<const std::int32_t*>(a.ids) + at);
    }
    __device__ __forceinline__ float value_at(std::uint64_t r, std::uint32_t k) const {
        const std::uint64_t at = r * a.ldv + k;
        if (a.valueType == TCC_F32) return load_global<float>(static_cast<const float*>(a.values) + at);
        if (a.valueType == TCC_BF16) return static_cast<float>(load_global<bf16_t>(static_cast<const bf16_t*>(a.values) + at));
        return static_cast<float>(load_global<f16_t>(static_cast<const f16_t*>(a.values) + at));
    }
    __device__ __forceinline__ bool is_class(std::int64_t i) const { return i >= 0 && i < static_cast<std::int64_t>(a.C); }

    // The maximum of a NaN is an infinity, so that its differences are NaN.
    static __device__ __forceinline__ float bound(float v) { return v != v ? -kNone : v; }

    // Loads the entries of row r and the teacher's probabilities; false where
    // the row has no target.
    __device__ __forceinline__ bool load(std::uint64_t r) {
        float m = kNone;
        bool bad = false;
#pragma unroll
        for (int e = 0; e < kEntries<TEAM>; ++e) {
            const std::uint32_t k = lane + e * TEAM;
            id[e] = -1;
            t[e] = kNone;
            if (k < a.K) {
                const std::int64_t i = id_at(r, k);
                if (is_class(i)) {
                    id[e] = i;
                    t[e] = value_at(r, k);
                } else if (i != -1) {
                    bad = true;
                }
            }
            m = fmaxf(m, bound(t[e]));
        }
        rest = a.rest == nullptr ? kNone : a.rest[r];
        m = fmaxf(wave_join<inWave>(m, Larger()), bound(rest));
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < kEntries<TEAM>; ++e) {
            p[e] = exp2_of((t[e] - base_of(m)) * a.c);
            s += p[e];
        }
        s = wave_join<inWave>(s, Add());
        s += exp2_of((rest - base_of(m)) * a.c);
        if (a.error != nullptr && bad) atomicOr(a.error, TCC_DEVERR_FEATURE_INDEX);
        if constexpr (TEAM > kWave) {  // from the first wave, which holds the entries, to the others
            if (threadIdx.x == 0) lds.one[row] = make_float2(m, s);
            __syncthreads();
            m = lds.one[row].x;
            s = lds.one[row].y;
            row ^= 1;
        }
        top = m;
        sum = s;
        const float per = 1.0f / s;
#pragma unroll
        for (int e = 0; e < kEntries<TEAM>; ++e) p[e] *= per;
        pRest = exp2_of((rest - base_of(m)) * a.c) * per;
        return m != kNone;
    }

    // Sets the bits of the ids from `first` on; the whole team.
    __device__ __forceinline__ void mark(std::uint32_t first) {
        team_sync<TEAM>();
        const std::uint32_t words = (min(a.C - first, kWindow<TEAM>) + 31) / 32;
        for (std::uint32_t i = lane; i < words; i += TEAM) bits[i] = 0;
        team_sync<TEAM>();
        bool again = false;
#pragma unroll
        for (int e = 0; e < kEntries<TEAM>; ++e) {
            if (!mine(e, first)) continue;
            const std::uint32_t at = static_cast<std::uint32_t>(id[e]) - first, bit = 1u << (at & 31);
            again |= (atomicOr(&bits[at / 32], bit) & bit) != 0;
        }
        twice = __ballot(again) != 0;
        team_sync<TEAM>();
    }
    __device__ __forceinline__ bool mine(int e, std::uint32_t first) const {
        return id[e] >= 0 && static_cast<std::uint32_t>(id[e]) - first < kWindow<TEAM>;
    }
    // Whether entry e is the first of its id, and the id's probability.
    __device__ __forceinline__ bool leads(int e, std::uint64_t r, float& all) const {
        all = p[e];
        if (!twice) return true;
        const std::uint32_t k = lane + e * TEAM;
        all = 0.0f;
        for (std::uint32_t o = 0; o < a.K; ++o) {
            if (id_at(r, o) != id[e]) continue;
            if (o < k) return false;
            all += exp2_of((value_at(r, o) - base_of(top)) * a.c) / sum;
        }
        return true;
    }
    // Bits of the N classes from `at` (of this window) on.
    template <int N>
    __device__ __forceinline__ std::uint32_t marked(std::uint32_t at) const {
        const std::uint32_t s = at & 31;
        std::uint32_t v = bits[at / 32] >> s;
        if (s + N > 32) v |= bits[at / 32 + 1] << (32 - s);
        return v & ((1u << N) - 1);
    }

    __device__ __forceinline__ Share join(Share v) {
        const float m = wave_join<inWave>(v.m, Larger());
        v.scale_to(m, a.c);
        v.s = wave_join<inWave>(v.s, Add());
        if constexpr (TEAM > kWave) {
            constexpr int waves = TEAM / kWave;
            if (__lane_id() == 0) lds.part[turn][threadIdx.x / kWave] = make_float2(v.m, v.s);
            __syncthreads();
            const float2 o = lds.part[turn][__lane_id() % waves];
            turn ^= 1;
            v = {o.x, o.y};
            const float all = wave_join<waves>(v.m, Larger());
            v.scale_to(all, a.c);
            v.s = wave_join<waves>(v.s, Add());
        }
        return v;
    }
};

template <typename T, int V, int TEAM, bool REST>
__global__ void __launch_bounds__(kThreads) loss_kernel(Args a) {
    using F = vec_t<float, V>;
    __shared__ Shared<TEAM> lds;
    Team<TEAM> team(lds, a);
    double lossSum = 0.0, weightSum = 0.0;
    const std::uint64_t step = static_cast<std::uint64_t>(gridDim.x) * kTeams<TEAM>;
    for (std::uint64_t r = static_cast<std::uint64_t>(blockIdx.x) * kTeams<TEAM> + threadIdx.x / TEAM; r < a.n; r += step) {
        const float w = a.weight == nullptr ? 1.0f : a.weight[r];
        weightSum += w;
        float loss = 0.0f;
        float4 stats = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (w != 0.0f && team.load(r)) {
            const T* z = static_cast<const T*>(a.z) + r * a.ldz;
            Share v, firsts;  // of the stream, and of the ids that are not in it
            for (std::uint32_t first = 0; first < a.C; first += kWindow<TEAM>) {
                if (REST) team.mark(first);
                const std::uint32_t end = min(a.C - first, kWindow<TEAM>) + first;
                for (std::uint32_t j = first / V + team.lane; static_cast<std::uint64_t>(j) * V < end; j += TEAM * kBatch) {
                    F x[kBatch];
                    float m = kNone;
#pragma unroll
                    for (int u = 0; u < kBatch; ++u) {
                        const Place<V> at(j + u * TEAM, a.C);
                        const bool here = at.any() && static_cast<std::uint64_t>(j + u * TEAM) * V < end;
                        x[u] = here ? load_any<T, V>(z + at.at) : F(kNone);
                        std::uint32_t out = here ? (1u << at.skip) - 1 : 0;
                        if (REST && here) out |= team.template marked<V>(at.at + at.skip - first) << at.skip;
                        if (out != 0) {
#pragma unroll
                            for (int q = 0; q < V; ++q) x[u][q] = (out >> q) & 1 ? kNone : x[u][q];
                        }
#pragma unroll
                        for (int q = 0; q < V; ++q) m = fmaxf(m, x[u][q]);
                    }
                    if (m > v.m) v.scale_to(m, a.c);
                    const float b = base_of(v.m);
#pragma unroll
                    for (int u = 0; u < kBatch; ++u)
#pragma unroll
                        for (int q = 0; q < V; ++q) v.s += exp2_of((x[u][q] - b) * a.c);
                }
                if (REST) {
#pragma unroll
                    for (int e = 0; e < kEntries<TEAM>; ++e) {
                        float unused;
                        if (team.mine(e, first) && team.leads(e, r, unused))
                            firsts = firsts.with({static_cast<float>(z[team.id[e]]), 1.0f}, a.c);
                    }
                }
            }
            const Share others = team.join(v);
            const Share all = REST ? others.with(team.join(firsts), a.c) : others;
            const Log2 logAll(all.s), logTop(team.sum);
            const float b = base_of(all.m), tb = base_of(team.top), sums = logAll.over(logTop);
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < kEntries<TEAM>; ++e) {
                if (team.id[e] < 0 || team.p[e] == 0.0f) continue;
                const float apart = (team.t[e] - tb) * a.c - (static_cast<float>(z[team.id[e]]) - b) * a.c;
                sum += team.p[e] * (apart + sums);
            }
            sum = wave_join<Team<TEAM>::inWave>(sum, Add());
            if (REST && team.pRest != 0.0f) {
                const float apart = (team.rest - tb) * a.c - (base_of(others.m) - b) * a.c;
                sum += team.pRest * (apart + (sums - Log2(others.s).over(Log2(1.0f))));
            }
            loss = w * (sum * (a.T * a.T * kLn2));
            stats = make_float4(b, all.s, REST ? base_of(others.m) : 0.0f, REST ? others.s : 0.0f);
        }
        if (team.lane == 0) {
            a.stats[r] = stats;
            if (a.loss != nullptr) a.loss[r] = loss;
            lossSum += loss;
        }
    }
    if (a.part == nullptr) return;
    // the first lanes' sums, in the order of the teams
    if (team.lane != 0) lossSum = weightSum = 0.0;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        lossSum += __shfl_xor(lossSum, d, kWave);
        weightSum += __shfl_xor(weightSum, d, kWave);
    }
    if (__lane_id() == 0) lds.sums[threadIdx.x / kWave] = make_double2(lossSum, weightSum);
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int k = 1; k < kThreads / kWave; ++k) {
        lossSum += lds.sums[k].x;
        weightSum += lds.sums[k].y;
    }
    a.part[blockIdx.x] = make_double2(lossSum, weightSum);
}

// The loss of all rows from the workgroups' sums.
__global__ void __launch_bounds__(kThreads) join_kernel(const double2* part, std::uint32_t parts, std::uint32_t mean,
                                                        float* loss, float* total) {
    double l = 0.0, w = 0.0;
    for (std::uint32_t i = threadIdx.x; i < parts; i += kThreads) {
        l += part[i].x;
        w += part[i].y;
    }
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        l += __shfl_xor(l, d, kWave);
        w += __shfl_xor(w, d, kWave);
    }
    __shared__ double2 sums[kThreads / kWave];
    if (__lane_id() == 0) sums[threadIdx.x / kWave] = make_double2(l, w);
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int k = 1; k < kThreads / kWave; ++k) {
        l += sums[k].x;
        w += sums[k].y;
    }
    *loss = static_cast<float>(mean ? (w == 0.0 ? 0.0 : l / w) : l);
    if (total != nullptr) *total = static_cast<float>(w);
}

template <typename T, int V, int TEAM, bool REST>
__global__ void __launch_bounds__(kThreads) grad_kernel(Args a) {
    using F = vec_t<float, V>;
    __shared__ Shared<TEAM> lds;
    Team<TEAM> team(lds, a);
    float each = a.T;
    if (a.reduction == TCC_REDUCE_MEAN) {
        const float count = a.total == nullptr ? static_cast<float>(a.n) : *a.total;
        each = count == 0.0f ? 0.0f : a.T / count;
    }
    if (a.reduction != TCC_REDUCE_NONE) each *= *a.dLoss;
    const std::uint64_t step = static_cast<std::uint64_t>(gridDim.x) * kTeams<TEAM>;
    for (std::uint64_t r = static_cast<std::uint64_t>(blockIdx.x) * kTeams<TEAM> + threadIdx.x / TEAM; r < a.n; r += step) {
        const float w = a.weight == nullptr ? 1.0f : a.weight[r];
        const T* z = static_cast<const T*>(a.z) + r * a.ldz;
        T* dz = static_cast<T*>(a.dz) + r * a.ldd;
        const bool target = w != 0.0f && team.load(r);
        const float4 stats = a.stats[r];
        float g = each * w, base = stats.x, factor;
        if (a.reduction == TCC_REDUCE_NONE) g *= a.dLoss[r];
        if (REST) {
            const float left = exp2_of((stats.z - stats.x) * a.c) * stats.w / stats.y - team.pRest;
            base = stats.z;
            factor = stats.w == 0.0f ? 0.0f : g * left / stats.w;
        } else {
            factor = g / stats.y;
        }
        for (std::uint32_t first = 0; first < a.C; first += kWindow<TEAM>) {
            if (target) team.mark(first);
            const std::uint32_t end = min(a.C - first, kWindow<TEAM>) + first;
            for (std::uint32_t j = first / V + team.lane; static_cast<std::uint64_t>(j) * V < end; j += TEAM * kBatch) {
                F x[kBatch];
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    const Place<V> at(j + u * TEAM, a.C);
                    const bool here = target && at.any() && static_cast<std::uint64_t>(j + u * TEAM) * V < end;
                    x[u] = here ? load_any<T, V>(z + at.at) : F(0.0f);
                }
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    const Place<V> at(j + u * TEAM, a.C);
                    if (!at.any() || static_cast<std::uint64_t>(j + u * TEAM) * V >= end) continue;
                    F d(0.0f);
                    std::uint32_t out = (1u << at.skip) - 1;
                    if (target) {
                        out |= team.template marked<V>(at.at + at.skip - first) << at.skip;
#pragma unroll
                        for (int q = 0; q < V; ++q) d[q] = factor * exp2_of((x[u][q] - base) * a.c);
                    }
                    if (out == 0) {
                        store_any<T, V>(dz + at.at, d);
                    } else {
#pragma unroll
                        for (int q = 0; q < V; ++q)
                            if (((out >> q) & 1) == 0) dz[at.at + q] = static_cast<T>(d[q]);
                    }
                }
            }
            if (!target) continue;
#pragma unroll
            for (int e = 0; e < kEntries<TEAM>; ++e) {
                float p;
                if (!team.mine(e, first) || !team.leads(e, r, p)) continue;
                const float q = exp2_of((static_cast<float>(z[team.id[e]]) - stats.x) * a.c) / stats.y;
                dz[team.id[e]] = static_cast<T>(g * (q - p));
            }
        }
    }
}

// ---------------------------------------------------------------- launches

// The team for rows of C classes and K entries; f is called with <V, TEAM>.
// A team's lanes take one batch of a row where it can be, and a wave up to
// 4,096 classes; they hold K / 4 lanes at least.
template <typename T, typename F>
void with_team(std::uint32_t C, std::uint32_t K, F f) {
    constexpr int V = kVec<T>;
    if (C < V) {
        if (K <= 16) return f.template operator()<1, 4>();
        return f.template operator()<1, 16>();
    }
    if (C <= 4 * kBatch * V && C <= kWindow<4> && K <= 16) return f.template operator()<V, 4>();
    if (C <= 16 * kBatch * V && C <= kWindow<16>) return f.template operator()<V, 16>();
    if (C <= 4096) return f.template operator()<V, 64>();
    return f.template operator()<V, 256>();
}

// Workgroups for n rows: eight a compute unit at most, each with as many rows.
std::uint64_t blocks_of(std::uint64_t n, std::uint64_t teams) {
    return std::min<std::uint64_t>((n + teams - 1) / teams, 8ull * device_cus());
}

template <typename T>
struct Loss {
    const Args& a;
    hipStream_t st;
    std::uint64_t& blocks;
    template <int V, int TEAM>
    void operator()() const {
        blocks = blocks_of(a.n, kTeams<TEAM>);
        const dim3 grid(static_cast<unsigned>(blocks));
        if (a.rest != nullptr) hipLaunchKernelGGL((loss_kernel<T, V, TEAM, true>), grid, dim3(kThreads), 0, st, a);
        else hipLaunchKernelGGL((loss_kernel<T, V, TEAM, false>), grid, dim3(kThreads), 0, st, a);
    }
};
template <typename T>
struct Grad {
    const Args& a;
    hipStream_t st;
    template <int V, int TEAM>
    void operator()() const {
        const dim3 grid(static_cast<unsigned>(blocks_of(a.n, kTeams<TEAM>)));
        if (a.rest != nullptr) hipLaunchKernelGGL((grad_kernel<T, V, TEAM, true>), grid, dim3(kThreads), 0, st, a);
        else hipLaunchKernelGGL((grad_kernel<T, V, TEAM, false>), grid, dim3(kThreads), 0, st, a);
    }
};

template <template <typename> class Launch, typename... More>
void launch_typed(std::uint32_t dtype, const Args& a, hipStream_t st, More&... more) {
    if (dtype == TCC_F32) with_team<float>(a.C, a.K, Launch<float>{a, st, more...});
    else if (dtype == TCC_BF16) with_team<bf16_t>(a.C, a.K, Launch<bf16_t>{a, st, more...});
    else with_team<f16_t>(a.C, a.K, Launch<f16_t>{a, st, more...});
}

int check_shape(const tcc_distill_shape* s) {
    TCC_REQUIRE(s != nullptr, TCC_ERR_INVALID_ARGUMENT, "distillation: no shape");
    TCC_REQUIRE(s->C >= 1 && s->K >= 1, TCC_ERR_INVALID_ARGUMENT, "distillation: rows have classes and entries");
    TCC_REQUIRE(dtype_bytes(s->dtype) != 0 && dtype_bytes(s->valueDtype) != 0, TCC_ERR_INVALID_ARGUMENT,
                "distillation: unknown element type");
    TCC_REQUIRE(s->idBytes == 4 || s->idBytes == 8, TCC_ERR_INVALID_ARGUMENT, "distillation: ids are int32 or int64");
    TCC_REQUIRE(s->reduction <= TCC_REDUCE_SUM, TCC_ERR_INVALID_ARGUMENT, "distillation: unknown reduction");
    TCC_REQUIRE(s->temperature > 0.0f && s->temperature < 1e18f, TCC_ERR_INVALID_ARGUMENT,
                "distillation: the temperature is positive");
    TCC_REQUIRE(s->K <= kMaxEntries, TCC_ERR_UNSUPPORTED, "distillation: at most 64 entries a row");
    TCC_REQUIRE(s->C <= 0x7FFFFFFFu, TCC_ERR_UNSUPPORTED, "distillation: fewer than 2^31 classes");
    TCC_REQUIRE(s->n < (1ull << 40), TCC_ERR_UNSUPPORTED, "distillation: fewer than 2^40 rows");
    return TCC_OK;
}

Args args_of(const tcc_distill_shape& s) {
    Args a{};
    a.n = s.n;
    a.C = s.C;
    a.K = s.K;
    a.valueType = s.valueDtype;
    a.idBytes = s.idBytes;
    a.reduction = s.reduction;
    a.T = s.temperature;
    a.c = static_cast<float>(1.4426950408889634 / static_cast<double>(s.temperature));
    return a;
}

bool aligned16(const void* p) { return (reinterpret_cast<std::uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace tcc

extern "C" size_t tcc_distill_loss_workspace_bytes(const tcc_distill_shape* s) {
    using namespace tcc;
    if (check_shape(s) != TCC_OK) return 0;
    return s->reduction == TCC_REDUCE_NONE ? 0 : 8 * device_cus() * sizeof(double2);
}

extern "C" int tcc_distill_loss(const tcc_distill_shape* s, const void* logits, uint64_t ldz, const void* values,
                                uint64_t ldv, const void* ids, uint64_t ldi, const float* rest, const float* weight,
                                float* loss, float* total, float* stats, uint32_t* deviceError, void* workspace,
                                size_t workspaceBytes, void* stream) {
    using namespace tcc;
    clear_last_error();
    if (const int rc = check_shape(s)) return rc;
    const bool summed = s->reduction != TCC_REDUCE_NONE;
    TCC_REQUIRE((s->n == 0 || (logits != nullptr && values != nullptr && ids != nullptr && stats != nullptr)) &&
                    (loss != nullptr || (s->n == 0 && !summed)),
                TCC_ERR_INVALID_ARGUMENT, "distillation: a null pointer");
    TCC_REQUIRE(ldz >= s->C && ldv >= s->K && ldi >= s->K, TCC_ERR_INVALID_ARGUMENT,
                "distillation: a row stride below the row's elements");
    TCC_REQUIRE(aligned16(stats), TCC_ERR_INVALID_ARGUMENT, "distillation: stats are 16-byte aligned");
    TCC_REQUIRE(!summed || s->n == 0 ||
                    (workspace != nullptr && aligned16(workspace) && workspaceBytes >= tcc_distill_loss_workspace_bytes(s)),
                TCC_ERR_INVALID_ARGUMENT, "distillation: the workspace is too small or not 16-byte aligned");
    Args a = args_of(*s);
    a.z = logits;
    a.ldz = ldz;
    a.values = values;
    a.ldv = ldv;
    a.ids = ids;
    a.ldi = ldi;
    a.rest = rest;
    a.weight = weight;
    a.stats = reinterpret_cast<float4*>(stats);
    a.error = deviceError;
    if (summed) a.part = static_cast<double2*>(workspace);
    else a.loss = loss;
    std::uint64_t blocks = 0;
    if (s->n > 0) {
        launch_typed<Loss>(s->dtype, a, as_stream(stream), blocks);
        TCC_LAUNCH_CHECK();
    }
    if (summed) {
        hipLaunchKernelGGL(join_kernel, dim3(1), dim3(kThreads), 0, as_stream(stream), a.part,
                           static_cast<std::uint32_t>(blocks), s->reduction == TCC_REDUCE_MEAN ? 1u : 0u, loss, total);
        TCC_LAUNCH_CHECK();
    }
    return TCC_OK;
}

extern "C" int tcc_distill_grad(const tcc_distill_shape* s, const float* dLoss, const void* logits, uint64_t ldz,
                                const void* values, uint64_t ldv, const void* ids, uint64_t ldi, const float* rest,
                                const float* weight, const float* total, const float* stats, void* dLogits, uint64_t ldd,
                                void* stream) {
    using namespace tcc;
    clear_last_error();
    if (const int rc = check_shape(s)) return rc;
    if (s->n == 0) return TCC_OK;
    TCC_REQUIRE(dLoss != nullptr && logits != nullptr && values != nullptr && ids != nullptr && stats != nullptr &&
                    dLogits != nullptr,
                TCC_ERR_INVALID_ARGUMENT, "distillation gradient: a null pointer");
    TCC_REQUIRE(ldz >= s->C && ldv >= s->K && ldi >= s->K && ldd >= s->C, TCC_ERR_INVALID_ARGUMENT,
                "distillation gradient: a row stride below the row's elements");
    TCC_REQUIRE(aligned16(stats), TCC_ERR_INVALID_ARGUMENT, "distillation gradient: stats are 16-byte aligned");
    TCC_REQUIRE(s->reduction != TCC_REDUCE_MEAN || (weight == nullptr) == (total == nullptr), TCC_ERR_INVALID_ARGUMENT,
                "distillation gradient: the weights' total goes with weights");
    Args a = args_of(*s);
    a.z = logits;
    a.ldz = ldz;
    a.values = values;
    a.ldv = ldv;
    a.ids = ids;
    a.ldi = ldi;
    a.rest = rest;
    a.weight = weight;
    a.total = total;
    a.dLoss = dLoss;
    a.stats = reinterpret_cast<float4*>(const_cast<float*>(stats));
    a.dz = dLogits;
    a.ldd = ldd;
    launch_typed<Grad>(s->dtype, a, as_stream(stream));
    TCC_LAUNCH_CHECK();
    return TCC_OK;
}
