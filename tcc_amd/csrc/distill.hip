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
// A team of lanes takes a row: 4, 16, 32 or 64 of a wave, or a workgroup of 256.
// Each lane keeps the maximum of what it read and the sum of
// exp((z - maximum) / T), rescaled when the maximum rises, so that a row is
// read once.  The batches of a long row are summed in 32 bits and added in 64: 2^20
// equal terms of exp(-1.25), added in 32 bits one after the other, are off by 0.9%.
// Everything is in base 2 with one factor log2(e) / T, rounded once: the
// differences z - m are formed first, and p and q are those of a temperature that
// is the same for both.  What rest needs, the classes that are no id, is summed by
// itself (a difference of sums would lose what a confident student leaves them):
// one bit of a class in LDS says that it is an id, and their logits are taken out
// of the stream and added afterwards.  The gradient's stream leaves out the ids in
// the same way, and the lanes that hold the entries write there; teams that hold a
// whole row in registers get the entries' gradients from a table of its classes in
// LDS instead.
#include <algorithm>
#include <type_traits>

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

using Share = ShareOf<false>;  // a row with an infinity has no softmax
using LongShare = LongShareOf<false>;

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
constexpr int kTeams = kThreads / TEAM;

// Classes whose bits a team holds at once, a multiple of 32.
template <int TEAM>
constexpr std::uint32_t kWindow = TEAM == 4 ? 128 : TEAM == 16 ? 512 : TEAM == 32 ? 1024 : TEAM == 64 ? 4096 : 1u << 17;

__device__ __forceinline__ float weight_of(const Args& a, std::uint64_t r) {
    return r >= a.n ? 0.0f : a.weight == nullptr ? 1.0f : a.weight[r];
}

// LDS of the workgroup.
template <int TEAM>
struct Shared {
    std::uint32_t bits[kTeams<TEAM>][kWindow<TEAM> / 32 + 1];  // a word more, for the reads at the end
    float2 part[2][TEAM > kWave ? TEAM / kWave : 1];
    float2 one[2];
    double2 sums[kThreads / kWave];
};

// One team at its rows; a lane holds E of their entries.
template <int TEAM, int E>
struct Team {
    static constexpr int inWave = TEAM < kWave ? TEAM : kWave;
    Shared<TEAM>& lds;
    const Args& a;
    std::uint32_t* bits;
    std::uint32_t lane;
    int turn = 0, odd = 0;  // places in LDS alternate, so that one barrier a use is enough
    __device__ __forceinline__ Team(Shared<TEAM>& shared, const Args& args)
        : lds(shared), a(args), bits(shared.bits[threadIdx.x / TEAM]), lane(threadIdx.x % TEAM) {}

    // The entries of a row: lane + e TEAM < K.  Only the first wave of a
    // workgroup holds any.
    std::int32_t id[E];  // -1: no entry
    float t[E], p[E], z[E];  // the teacher's value and probability, the student's logit
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

    // The entries of row r, as memory holds them.
    __device__ __forceinline__ void fetch(std::uint64_t r) {
        bad = false;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const std::uint32_t k = lane + e * TEAM;
            nextId[e] = -1;
            nextT[e] = kNone;
            if (k < a.K) {
                const std::int64_t i = id_at(r, k);
                nextId[e] = is_class(i) ? static_cast<std::int32_t>(i) : -1;
                bad |= nextId[e] < 0 && i != -1;
                nextT[e] = value_at(r, k);
            }
        }
        nextRest = a.rest == nullptr ? kNone : a.rest[r];
    }
    std::int32_t nextId[E];
    float nextT[E], nextRest;
    bool bad;

    // The fetched row, its logits at `row`, and the teacher's probabilities; false
    // where it has no target.
    template <typename T>
    __device__ __forceinline__ bool load(const T* row) {
        float m = kNone;
        rest = nextRest;
        if (a.error != nullptr && bad) atomicOr(a.error, TCC_DEVERR_FEATURE_INDEX);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            id[e] = nextId[e];
            t[e] = id[e] < 0 ? kNone : nextT[e];
            z[e] = id[e] < 0 ? kNone : static_cast<float>(row[id[e]]);
            m = fmaxf(m, bound(t[e]));
        }
        m = fmaxf(wave_join<inWave>(m, Larger()), bound(rest));
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            p[e] = exp2_of((t[e] - base_of(m)) * a.c);
            s += p[e];
        }
        s = wave_join<inWave>(s, Add());
        s += exp2_of((rest - base_of(m)) * a.c);
        if constexpr (TEAM > kWave) {  // from the first wave, which holds the entries, to the others
            if (threadIdx.x == 0) lds.one[odd] = make_float2(m, s);
            __syncthreads();
            m = lds.one[odd].x;
            s = lds.one[odd].y;
            odd ^= 1;
        }
        top = m;
        sum = s;
        const float per = inverse_of(s);
#pragma unroll
        for (int e = 0; e < E; ++e) p[e] *= per;
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
        for (int e = 0; e < E; ++e) {
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
            all += exp2_of((value_at(r, o) - base_of(top)) * a.c) * inverse_of(sum);
        }
        return true;
    }
    // Bits of the N classes from `at` (of this window) on; marked_here: of a
    // multiple of N.
    template <int N>
    __device__ __forceinline__ std::uint32_t marked_here(std::uint32_t at) const {
        return bits[at / 32] >> (at & 31) & ((1u << N) - 1);
    }
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

// A NaN that no operation gives: a class that no entry has.
constexpr std::uint32_t kNoEntry = 0x7FD00001u;

// A batch of a team: kBatch vectors a lane, from element `base` of the row on.
template <typename T, int V, int TEAM, bool WHOLE>
struct Batch {
    static constexpr std::uint32_t stride = TEAM * kBatch * V;
    static constexpr bool whole = WHOLE;  // rows are one batch
    vec_t<T, V> x[kBatch];

    static __device__ __forceinline__ Place<V> place(std::uint32_t base, int u, std::uint32_t lane, std::uint32_t C) {
        return Place<V>(base / V + u * TEAM + lane, C);
    }
    // Whether every lane has all of its vectors, whole ones.
    static __device__ __forceinline__ bool inside(std::uint32_t base, std::uint32_t C) { return base + stride <= C; }
    // Whether any lane has a vector u.
    static __device__ __forceinline__ bool any(std::uint32_t base, int u, std::uint32_t C) {
        return base + static_cast<std::uint32_t>(u * TEAM * V) < C;
    }
    __device__ __forceinline__ void load(const T* z, std::uint32_t base, std::uint32_t lane, std::uint32_t C) {
        if (!whole && inside(base, C)) {
            z += base + lane * V;
#pragma unroll
            for (int u = 0; u < kBatch; ++u) x[u] = load_as<T, V>(z + u * TEAM * V);
            return;
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            if (!any(base, u, C)) break;
            const Place<V> at = place(base, u, lane, C);
            if (at.any()) x[u] = load_as<T, V>(z + at.at);
        }
    }
    __device__ __forceinline__ vec_t<float, V> values(int u) const { return __builtin_convertvector(x[u], vec_t<float, V>); }
};

// A row that a team begins, and the next one where it holds whole rows: their
// logits and entries are on their way while this one is computed (the gradient of
// 2.45M x 100 fp32 rows: 420 us instead of 556), and the entries' logits
// come from `row` in LDS instead of memory.
template <typename T, int V, int TEAM, int E, bool WHOLE>
struct Front {
    using B = Batch<T, V, TEAM, WHOLE>;
    const Args& a;
    Team<TEAM, E>& team;
    std::uint64_t r, step;
    float w, nextW;
    B batch, after;

    __device__ __forceinline__ Front(const Args& args, Team<TEAM, E>& t) : a(args), team(t) {
        step = static_cast<std::uint64_t>(gridDim.x) * kTeams<TEAM>;
        r = static_cast<std::uint64_t>(blockIdx.x) * kTeams<TEAM> + threadIdx.x / TEAM;
        nextW = weight_of(a, r);
        if constexpr (B::whole) load(after, r, nextW);
    }
    __device__ __forceinline__ void load(B& to, std::uint64_t row, float weight) {
        if (weight == 0.0f) return;
        to.load(logits(row), 0, team.lane, a.C);
        team.fetch(row);
    }
    __device__ __forceinline__ const T* logits(std::uint64_t row) const { return static_cast<const T*>(a.z) + row * a.ldz; }

    // Takes up row r; true where it has a target.
    __device__ __forceinline__ bool begin(float* row) {
        w = nextW;
        nextW = weight_of(a, r + step);
        bool target = w != 0.0f;
        if constexpr (B::whole) {
            batch = after;
            if (target) {
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    if (!B::any(0, u, a.C)) break;
                    const Place<V> at = B::place(0, u, team.lane, a.C);
                    if (at.any()) *reinterpret_cast<any_vec_t<float, V>*>(row + at.at) = batch.values(u);
                }
                team_sync<TEAM>();
                target = team.load(row);
                team_sync<TEAM>();
            }
            load(after, r + step, nextW);
        } else {
            load(batch, r, w);
            target = target && team.load(logits(r));
        }
        return target;
    }
};

// Bound by the reading of the logits: 4,096 rows of 50,000 bf16 logits with 32
// entries and a rest take 89 us with the kernel that joins the sums (410 MB: 4.6 TB/s).
template <typename T, int V, int TEAM, int E, bool WHOLE, bool REST>
__global__ void __launch_bounds__(kThreads, WHOLE ? 1 : 4) loss_kernel(Args a) {
    using F = vec_t<float, V>;
    using B = Batch<T, V, TEAM, WHOLE>;
    static_assert(kWindow<TEAM> % B::stride == 0 || B::whole);
    __shared__ Shared<TEAM> lds;
    Team<TEAM, E> team(lds, a);
    double lossSum = 0.0, weightSum = 0.0;
    __shared__ __attribute__((aligned(16))) float table[B::whole ? kTeams<TEAM> : 1][B::whole ? B::stride : V];
    for (Front<T, V, TEAM, E, WHOLE> front(a, team); front.r < a.n; front.r += front.step) {
        const std::uint64_t r = front.r;
        const bool target = front.begin(B::whole ? table[threadIdx.x / TEAM] : nullptr);
        const T* z = front.logits(r);
        const float w = front.w;
        B& batch = front.batch;
        weightSum += w;
        float loss = 0.0f;
        float4 stats = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (target) {
            Share whole, firsts;  // of the stream, and of the ids that are not in it
            LongShare v;          // the stream's where rows have many batches
            for (std::uint32_t base = 0; base < a.C; base += B::stride) {
                const std::uint32_t first = base & ~(kWindow<TEAM> - 1);
                if (REST && first == base) {
                    team.mark(first);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        float unused;
                        if (team.mine(e, first) && team.leads(e, r, unused)) firsts = firsts.with({team.z[e], 1.0f}, a.c);
                    }
                }
                B after;
                if constexpr (!B::whole) after.load(z, base + B::stride, team.lane, a.C);
                const auto add = [&](auto inside) {
                    F x[kBatch];
                    float m = kNone;
#pragma unroll
                    for (int u = 0; u < kBatch; ++u) {
                        if (!inside && !B::any(base, u, a.C)) break;
                        x[u] = batch.values(u);
                        std::uint32_t out = 0;
                        if constexpr (inside) {
                            if (REST) out = team.template marked_here<V>(base + (u * TEAM + team.lane) * V - first);
                        } else {
                            const Place<V> at = B::place(base, u, team.lane, a.C);
                            out = (1u << at.skip) - 1;
                            if (REST && at.any()) out |= team.template marked<V>(at.at + at.skip - first) << at.skip;
                        }
                        if (out != 0) {
#pragma unroll
                            for (int q = 0; q < V; ++q) x[u][q] = (out >> q) & 1 ? kNone : x[u][q];
                        }
#pragma unroll
                        for (int q = 0; q < V; ++q) m = fmaxf(m, x[u][q]);
                    }
                    const float b = B::whole ? base_of(m) : v.raise(m, a.c);
                    float s = 0.0f;
#pragma unroll
                    for (int u = 0; u < kBatch; ++u) {
                        if (!inside && !B::any(base, u, a.C)) break;
#pragma unroll
                        for (int q = 0; q < V; ++q) s += exp2_of((x[u][q] - b) * a.c);
                    }
                    if constexpr (B::whole) whole = {m, s};
                    else v.s += s;
                };
                if (!B::whole && B::inside(base, a.C)) add(std::true_type());
                else add(std::false_type());
                if constexpr (B::whole) break;
                batch = after;
            }
            if constexpr (!B::whole) whole = v.share(a.c);
            const Share others = team.join(whole);
            const Share all = REST ? others.with(team.join(firsts), a.c) : others;
            const Log2 logAll(all.s), logTop(team.sum);
            const float b = base_of(all.m), tb = base_of(team.top), sums = logAll.over(logTop);
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (team.id[e] < 0 || team.p[e] == 0.0f) continue;
                const float apart = (team.t[e] - tb) * a.c - (team.z[e] - b) * a.c;
                sum += team.p[e] * (apart + sums);
            }
            sum = wave_join<Team<TEAM, E>::inWave>(sum, Add());
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

// Bound by memory, at a copy's rate: 2.45M x 100 fp32 rows with 8 entries take 420 us
// (2.05 GB: 4.9 TB/s), 4,096 x 50,001 bf16 rows with 32 and a rest 197 (820 MB: 4.2 TB/s).
template <typename T, int V, int TEAM, int E, bool WHOLE, bool REST>
__global__ void __launch_bounds__(kThreads) grad_kernel(Args a) {
    using F = vec_t<float, V>;
    using B = Batch<T, V, TEAM, WHOLE>;
    __shared__ Shared<TEAM> lds;
    __shared__ __attribute__((aligned(16))) float table[B::whole ? kTeams<TEAM> : 1][B::whole ? B::stride : V];
    Team<TEAM, E> team(lds, a);
    float each = a.T;
    if (a.reduction == TCC_REDUCE_MEAN) {
        const float count = a.total == nullptr ? static_cast<float>(a.n) : *a.total;
        each = count == 0.0f ? 0.0f : a.T / count;
    }
    if (a.reduction != TCC_REDUCE_NONE) each *= *a.dLoss;
    for (Front<T, V, TEAM, E, WHOLE> front(a, team); front.r < a.n; front.r += front.step) {
        const std::uint64_t r = front.r;
        const float4 stats = a.stats[r];
        float g = each;
        if (a.reduction == TCC_REDUCE_NONE) g *= a.dLoss[r];
        const bool target = front.begin(B::whole ? table[threadIdx.x / TEAM] : nullptr);
        g *= front.w;
        const T* z = front.logits(r);
        T* dz = static_cast<T*>(a.dz) + r * a.ldd;
        B& batch = front.batch;
        const float perAll = inverse_of(stats.y);
        float base2 = stats.x, factor;  // of the others: factor 2^((z - base2) c)
        if (REST) {
            const float left = exp2_of((stats.z - stats.x) * a.c) * stats.w * perAll - team.pRest;
            base2 = stats.z;
            factor = stats.w == 0.0f ? 0.0f : g * left * inverse_of(stats.w);
        } else {
            factor = g * perAll;
        }
        const auto entry = [&](float x, float p) { return g * (exp2_of((x - stats.x) * a.c) * perAll - p); };
        if constexpr (B::whole) {
            // the entries' gradients by their classes, so that every vector is stored once
            float* mine = table[threadIdx.x / TEAM];
            if (target) {
#pragma unroll
                for (int u = 0; u < kBatch; ++u)
                    if (B::any(0, u, a.C))
                        *reinterpret_cast<F*>(mine + (u * TEAM + team.lane) * V) = F(__uint_as_float(kNoEntry));
                team_sync<TEAM>();
                bool again = false;
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (team.id[e] >= 0)
                        again |= __float_as_uint(atomicExch(mine + team.id[e], entry(team.z[e], team.p[e]))) != kNoEntry;
                team.twice = __ballot(again) != 0;
                team_sync<TEAM>();
                if (team.twice) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        float p;
                        if (team.id[e] >= 0 && team.leads(e, r, p)) mine[team.id[e]] = entry(team.z[e], p);
                    }
                    team_sync<TEAM>();
                }
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                if (!B::any(0, u, a.C)) break;
                const Place<V> at = B::place(0, u, team.lane, a.C);
                if (!at.any()) continue;
                F d(0.0f);
                if (target) {
                    const F x = batch.values(u), known = *reinterpret_cast<const any_vec_t<float, V>*>(mine + at.at);
#pragma unroll
                    for (int q = 0; q < V; ++q)
                        d[q] = __float_as_uint(known[q]) == kNoEntry ? factor * exp2_of((x[q] - base2) * a.c) : known[q];
                }
                store_any<T, V>(dz + at.at, d);
            }
            team_sync<TEAM>();  // the next row's logits go there
        } else {
            for (std::uint32_t base = 0; base < a.C; base += B::stride) {
                const std::uint32_t first = base & ~(kWindow<TEAM> - 1);
                if (target && first == base) {
                    team.mark(first);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        float p;
                        if (!team.mine(e, first) || !team.leads(e, r, p)) continue;
                        dz[team.id[e]] = static_cast<T>(entry(team.z[e], p));
                    }
                }
                B after;
                if (target) after.load(z, base + B::stride, team.lane, a.C);
                const auto give = [&](auto inside) {
#pragma unroll
                    for (int u = 0; u < kBatch; ++u) {
                        if (!inside && !B::any(base, u, a.C)) break;
                        Place<V> at(0, V);
                        if constexpr (inside) {
                            at.at = base + (u * TEAM + team.lane) * V;
                        } else {
                            at = B::place(base, u, team.lane, a.C);
                            if (!at.any()) continue;
                        }
                        F d(0.0f);
                        std::uint32_t out = inside ? 0 : (1u << at.skip) - 1;
                        if (target) {
                            const F x = batch.values(u);
                            out |= inside ? team.template marked_here<V>(at.at - first)
                                          : team.template marked<V>(at.at + at.skip - first) << at.skip;
#pragma unroll
                            for (int q = 0; q < V; ++q) d[q] = factor * exp2_of((x[q] - base2) * a.c);
                        }
                        if (out == 0) {
                            store_any<T, V>(dz + at.at, d);
                        } else {
#pragma unroll
                            for (int q = 0; q < V; ++q)
                                if (((out >> q) & 1) == 0) dz[at.at + q] = static_cast<T>(d[q]);
                        }
                    }
                };
                if (B::inside(base, a.C)) give(std::true_type());
                else give(std::false_type());
                batch = after;
            }
        }
    }
}

// ---------------------------------------------------------------- launches

// The team for rows of C classes and K entries; f is called with <V, TEAM, E,
// WHOLE>.  A team takes whole rows where its lanes' batch holds them; a wave longer
// ones up to 4,096 classes, a workgroup above.
template <typename T, typename F>
void with_team(std::uint32_t C, std::uint32_t K, F f) {
    constexpr int V = kVec<T>;
    if (C < V) {
        if (K <= 4) return f.template operator()<1, 4, 1, true>();
        return f.template operator()<1, 16, 4, true>();
    }
    if (C <= 4 * kBatch * V && K <= 4) return f.template operator()<V, 4, 1, true>();
    if (C <= 16 * kBatch * V) {
        if (K <= 16) return f.template operator()<V, 16, 1, true>();
        if (K <= 32) return f.template operator()<V, 16, 2, true>();
        return f.template operator()<V, 16, 4, true>();
    }
    if (C <= 32 * kBatch * V) {
        if (K <= 32) return f.template operator()<V, 32, 1, true>();
        return f.template operator()<V, 32, 2, true>();
    }
    if (C <= 64 * kBatch * V) return f.template operator()<V, 64, 1, true>();
    if (C <= 4096) return f.template operator()<V, 64, 1, false>();
    return f.template operator()<V, 256, 1, false>();
}

// A grid of the workgroups that run at once, or those that n rows need.
template <typename Kernel>
std::uint64_t launch(Kernel kernel, std::uint32_t& perCu, const Args& a, std::uint64_t teams, hipStream_t st) {
    const std::uint64_t blocks = std::min<std::uint64_t>((a.n + teams - 1) / teams, resident_blocks(kernel, kThreads, perCu));
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, st, a);
    return blocks;
}

template <typename T>
struct Loss {
    const Args& a;
    hipStream_t st;
    std::uint64_t& blocks;
    template <int V, int TEAM, int E, bool WHOLE>
    void operator()() const {
        static std::uint32_t perCu[2];
        blocks = a.rest != nullptr ? launch(loss_kernel<T, V, TEAM, E, WHOLE, true>, perCu[1], a, kTeams<TEAM>, st)
                                   : launch(loss_kernel<T, V, TEAM, E, WHOLE, false>, perCu[0], a, kTeams<TEAM>, st);
    }
};
template <typename T>
struct Grad {
    const Args& a;
    hipStream_t st;
    template <int V, int TEAM, int E, bool WHOLE>
    void operator()() const {
        static std::uint32_t perCu[2];
        if (a.rest != nullptr) launch(grad_kernel<T, V, TEAM, E, WHOLE, true>, perCu[1], a, kTeams<TEAM>, st);
        else launch(grad_kernel<T, V, TEAM, E, WHOLE, false>, perCu[0], a, kTeams<TEAM>, st);
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
    TCC_REQUIRE(s->temperature >= 1e-18f && s->temperature <= 1e18f, TCC_ERR_INVALID_ARGUMENT,
                "distillation: the temperature lies between 1e-18 and 1e18");
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
