// The K largest logits of every row, and one logit for the rest
// (include/tcc_training.h).
//
//   ids: the K largest, the lowest index first among equals, NaN above all
//   rest = T log(sum of exp(z_j / T) over the other classes)
//
// A row is read once from memory.  From what the lanes have at first comes a bound
// that K elements reach; those that reach it, hardly more than K of a short row and
// a few hundred of a long one in random order, go to LDS as 64-bit keys (the value's
// order, then the index's), and each counts the larger ones, which is its place.
// What does not reach the bound, and what K others beat, is summed for the rest, a
// long row's batches in 64 bits: nothing is subtracted from a sum of all.  Rows of up
// to 1,024 classes are held in registers by 4, 16 or 64 lanes; longer ones are
// streamed, by a wave up to 4,096 classes and where there are many, by a workgroup
// else.  Rows with more at the bound than there is room for (that rise, or with many
// equal) go another way: the short ones take their K one after the other, the long
// ones are read again by a second kernel that keeps sorted lists.
#include <algorithm>

#include "../../include/tcc_swtcf.h"
#include "../../include/tcc_training.h"
#include "logits.hpp"
#include "teams.hpp"

namespace tcc {
namespace {

constexpr std::uint32_t kMostTop = 64;
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kBatch = 4;  // vectors that a lane loads before it uses the first
constexpr std::uint32_t kWaveClasses = 4096;

using Share = ShareOf<true>;  // a rest with an infinity is infinite
using LongShare = LongShareOf<true>;

struct Args {
    const void* z;
    void* values;
    std::int32_t* ids;
    float* rest;
    std::uint64_t n, ldz, ldv, ldi;
    std::uint32_t C, K;
    float T, c;  // c = log2(e) / T
};

using Key = std::uint64_t;

// Floats in the order of unsigned integers: -0 as 0, NaN above all.
__device__ __forceinline__ std::uint32_t order_of(float v) {
    if (v != v) return 0xFFFFFFFFu;
    const std::uint32_t b = __float_as_uint(v + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(std::uint32_t order) {
    return __uint_as_float(order & 0x80000000u ? order & 0x7FFFFFFFu : ~order);
}
// Larger for larger values, and for lower indices among equals; never 0, which
// stands for no element.
__device__ __forceinline__ Key key_of(float v, std::uint32_t index) {
    return static_cast<Key>(order_of(v)) << 32 | static_cast<std::uint32_t>(~index);
}
__device__ __forceinline__ std::uint32_t index_of(Key k) { return ~static_cast<std::uint32_t>(k); }

// The steps of a bitonic network from distance D on, in runs of SIZE lanes that
// alternate in direction: the larger first in the first run if DOWN.
template <int SIZE, bool DOWN, int D, typename K>
__device__ __forceinline__ K wave_steps(K v) {
    const unsigned l = lane_id();
    const K o = other<D>(v);
    const bool first = (l & D) == 0, forward = SIZE == kWave || (l & SIZE) == 0;
    v = (v > o) == ((first == forward) == DOWN) ? v : o;
    if constexpr (D > 1) return wave_steps<SIZE, DOWN, D / 2>(v);
    else return v;
}
// Sorted over the lanes.
template <bool DOWN, int SIZE = 2, typename K>
__device__ __forceinline__ K wave_sort(K v) {
    v = wave_steps<SIZE, DOWN, SIZE / 2>(v);
    if constexpr (SIZE < kWave) return wave_sort<DOWN, 2 * SIZE>(v);
    else return v;
}

// A wave's LDS operations run in order; the compiler keeps them so across this.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A batch of a wave: its lanes' vectors first + lane, and those step, 2 step, ...
// after them, of a row.
template <int V>
struct Range {
    std::uint32_t first, step, C;
    // Whether all of its vectors are whole ones, for the whole wave.
    __device__ __forceinline__ bool inside() const { return (first + kWave + (kBatch - 1) * step) * V <= C; }
    __device__ __forceinline__ Place<V> place(int u) const { return Place<V>(first + lane_id() + u * step, C); }
    // The first element of vector u.
    __device__ __forceinline__ std::uint32_t at(int u) const { return inside() ? (first + lane_id() + u * step) * V : place(u).at; }
};

template <typename T, int V>
struct Ahead {
    vec_t<T, V> x[kBatch];
    __device__ __forceinline__ void load(const T* z, Range<V> r) {
        if (r.inside()) {
            z += (r.first + lane_id()) * V;
#pragma unroll
            for (int u = 0; u < kBatch; ++u) x[u] = load_as<T, V>(z + u * r.step * V);
            return;
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const Place<V> at = r.place(u);
            if (at.any()) x[u] = load_as<T, V>(z + at.at);
        }
    }
};

// How many elements a bound is good for that K are wanted of: each of them is
// compared with all.
__device__ __forceinline__ std::uint32_t enough(std::uint32_t K) { return K + K / 2 + 8; }

// Its elements as floats, what is no element of it as -inf, and the largest of each
// vector, a NaN where it has one.
template <typename T, int V>
struct Elements {
    vec_t<float, V> x[kBatch];
    float most[kBatch];
    __device__ __forceinline__ Elements(const Ahead<T, V>& raw, Range<V> r) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) x[u] = __builtin_convertvector(raw.x[u], vec_t<float, V>);
        if (!r.inside()) {
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const std::uint32_t skip = r.place(u).skip;
#pragma unroll
                for (std::uint32_t q = 0; q < V; ++q) x[u][q] = q < skip ? kNone : x[u][q];
            }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            most[u] = x[u][0];
#pragma unroll
            for (int q = 1; q < V; ++q) most[u] = __builtin_elementwise_maximum(most[u], x[u][q]);
        }
    }
    // How many of the wave's elements reach b, which is above -inf.
    __device__ __forceinline__ std::uint32_t reaching(float b) const {
        std::uint32_t n = 0;
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
#pragma unroll
            for (int q = 0; q < V; ++q) n += __popcll(__ballot(!(x[u][q] < b)));
        return n;
    }
    // As `halved` of rows in registers.
    __device__ __forceinline__ float halved(float bound, std::uint32_t K) const {
        std::uint32_t lo = order_of(bound), hi = uniform(order_of(wave_join<kWave>(largest(kNone), Larger()))) + 1;
        while (hi - lo > 1) {
            const std::uint32_t mid = lo + (hi - lo) / 2, n = reaching(value_of(mid));
            if (n < K) {
                hi = mid;
            } else {
                lo = mid;
                if (n <= enough(K)) break;
            }
        }
        return value_of(lo);
    }
    // Takes what is not below (ABOVE: not up to) the bound from vector u, and says
    // what that is: element q is bit V - 1 - q.
    template <bool ABOVE>
    __device__ __forceinline__ std::uint32_t leave(int u, float bound, Range<V> r) {
        std::uint32_t out = 0;
#pragma unroll
        for (int q = 0; q < V; ++q) {
            const bool goes = ABOVE ? !(x[u][q] <= bound) : !(x[u][q] < bound);
            out += out + (goes ? 1u : 0u);
            x[u][q] = goes ? kNone : x[u][q];
        }
        most[u] = x[u][0];
#pragma unroll
        for (int q = 1; q < V; ++q) most[u] = fmaxf(most[u], x[u][q]);
        if (!r.inside()) out &= (1u << (V - r.place(u).skip)) - 1;
        return out;
    }
    // The larger of `own` and its elements of this lane.
    __device__ __forceinline__ float largest(float own) const {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) own = __builtin_elementwise_maximum(own, most[u]);
        return own;
    }
    __device__ __forceinline__ void add_to(LongShare& rest, float c) const {
        float m = kNone, s = 0.0f;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) m = fmaxf(m, most[u]);
        const float b = rest.raise(m, c);
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
#pragma unroll
            for (int q = 0; q < V; ++q) s += exp2_of((x[u][q] - b) * c);
        rest.s += s;
    }
};

__device__ __forceinline__ Share wave_join_share(Share v, float c) {
    const float m = wave_join<kWave>(v.m, Larger());
    v.scale_to(m, c);
    v.s = wave_join<kWave>(v.s, Add());
    return v;
}
// The K-th largest of the lanes' v, in the order of unsigned integers.
__device__ __forceinline__ std::uint32_t kth_lane(float v, std::uint32_t K) {
    return static_cast<std::uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(wave_sort<true>(order_of(v))), K - 1));
}
__device__ __forceinline__ float as_logit(const Args& a, Share rest) {
    return base_of<true>(rest.m) + a.T * kLn2 * log2_of(rest.s);
}

// ---------------------------------------------------------------- streamed rows

constexpr std::uint32_t kFound = 512;      // classes of a wave that have room in LDS
constexpr std::int32_t kToSort = -1;       // the first id of a row that had more
static_assert(kMostTop <= kWave);

// A row is read once by a wave, or by the four of a workgroup.  K elements at least
// reach the K-th largest of the lanes' maxima so far (of four waves: the least of
// their K/4-th); one wave raises that bound as it goes, four agree on one anew after
// half as many batches again as there were, and at the end.  The classes that reach
// it go to LDS: of rows in random order with K = 64 about 110 of 50,000 for a wave,
// 200 of a million, 370 of 2^27 (where one takes the row, with K = 32, 190, 340 and,
// of 2^24, 460).  Those that reach the last bound each count the larger ones among
// them, which is their place.  4,096 rows of 50,000 bf16 logits with K = 32 take 102
// us, with the kernel after it (5 us) that finds no row left to sort: 410 MB at 4.0
// TB/s, three instructions an element beside them.
template <typename T, int V, int WAVES>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 6 : 5) stream_kernel(Args a) {
    static_assert(WAVES == 1 || WAVES == kWaves);
    constexpr std::uint32_t teams = kWaves / WAVES, step = WAVES * kWave;
    __shared__ std::uint32_t classes[kWaves][kFound], counts[kWaves], kept[kWaves];
    __shared__ __attribute__((aligned(16))) Key keys[kWaves][kFound + 4];
    __shared__ float bounds[2][kWaves];
    __shared__ float2 rests[kWaves];
    const std::uint32_t w = uniform(threadIdx.x / kWave), first = WAVES == 1 ? 0 : w * kWave;
    // the least of the waves' bounds; the whole workgroup, and the places alternate,
    // so that one barrier a call is enough
    std::uint32_t turn = 0;
    const auto agreed = [&](float bound) {
        if (lane_id() == 0) bounds[turn][w] = bound;
        __syncthreads();
        const float mine = bounds[turn][lane_id() % WAVES];
        turn ^= 1;
        return wave_join<WAVES>(mine, Smaller());
    };
    const std::uint64_t rows = static_cast<std::uint64_t>(gridDim.x) * teams;
    for (std::uint64_t r = static_cast<std::uint64_t>(blockIdx.x) * teams + (WAVES == 1 ? w : 0); r < a.n; r += rows) {
        const T* z = static_cast<const T*>(a.z) + r * a.ldz;
        const std::uint32_t K = (a.K + WAVES - 1) / WAVES;
        LongShare rest;
        std::uint32_t count = 0;
        float bound = kNone, own = kNone;
        std::uint32_t batch = 0, next = 0;  // the batch before which they agree again
        Ahead<T, V> ahead;
        Range<V> range{first, step, a.C};
        ahead.load(z, range);
        for (; range.first * V < a.C; range.first += step * kBatch, ++batch) {  // of the wave's first lane
            Elements<T, V> e(ahead, range);
            ahead.load(z, {range.first + step * kBatch, step, a.C});
            own = e.largest(own);
            if constexpr (WAVES > 1) {
                // (every wave has this batch, or none agrees)
                if (batch == next && (range.first - first + step - kWave) * V < a.C) {
                    bound = fmaxf(bound, agreed(value_of(kth_lane(own, K))));
                    next = batch + 2 + batch / 2;
                }
            } else {
                if (K > 32) {  // the lanes' maxima are few for it: 2.5 times as many would reach the least of 64
                    if (batch == 0) bound = e.halved(value_of(kth_lane(own, K)), K);
                } else if (batch < 4 || batch % 4 == 0) {
                    bound = value_of(kth_lane(own, K));
                }
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                if (__ballot(!(e.most[u] < bound)) == 0) continue;
                std::uint32_t left = e.template leave<false>(u, bound, range);
                const std::uint32_t last = range.at(u) + V - 1;
                for (std::uint64_t more; (more = __ballot(left != 0)) != 0; left &= left - 1) {
                    const std::uint32_t to = count + __popcll(more & lanemask_lt());
                    if (left != 0 && to < kFound) classes[w][to] = last - __builtin_ctz(left);
                    count += __popcll(more);
                }
            }
            e.add_to(rest, a.c);
        }
        bound = fmaxf(bound, value_of(kth_lane(own, K)));
        bool fits = count <= kFound;
        if constexpr (WAVES > 1) {
            if (lane_id() == 0) counts[w] = count;
            bound = agreed(bound);
#pragma unroll
            for (int o = 0; o < WAVES; ++o) fits &= counts[o] <= kFound;
        }
        if (!fits) {
            if (lane_id() == 0 && (WAVES == 1 || w == 0)) a.ids[r * a.ldi] = kToSort;
            continue;
        }
        wave_sync();
        std::uint32_t all = 0;
        for (std::uint32_t i = lane_id(); i - lane_id() < count; i += kWave) {
            const std::uint32_t c = i < count ? classes[w][i] : 0u;
            const float x = static_cast<float>(z[c]);
            const bool keeps = i < count && !(x < bound);
            const std::uint64_t those = __ballot(keeps);
            if (keeps) keys[w][all + __popcll(those & lanemask_lt())] = key_of(x, c);
            else if (i < count) rest.add(x, a.c);
            all += __popcll(those);
        }
        if (lane_id() < 3) keys[w][all + lane_id()] = 0;  // for the reads of four
        if constexpr (WAVES > 1) {
            if (lane_id() == 0) kept[w] = all;
            __syncthreads();
        } else {
            wave_sync();
        }
        for (std::uint32_t i = lane_id(); i < all; i += kWave) {
            const Key k = keys[w][i];
            std::uint32_t at = 0;
#pragma unroll
            for (int t = 0; t < WAVES; ++t) {
                const Key* others = keys[WAVES == 1 ? w : t];
                const std::uint32_t n = WAVES == 1 ? all : kept[t];
                for (std::uint32_t o = 0; o < n; o += 4) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) at += others[o + q] > k ? 1u : 0u;
                }
            }
            if (at < a.K) {
                const std::uint32_t c = index_of(k);
                static_cast<T*>(a.values)[r * a.ldv + at] = z[c];
                a.ids[r * a.ldi + at] = static_cast<std::int32_t>(c);
            } else {
                rest.add(value_of(static_cast<std::uint32_t>(k >> 32)), a.c);
            }
        }
        Share sum = wave_join_share(rest.share(a.c), a.c);
        if constexpr (WAVES > 1) {
            if (lane_id() == 0) rests[w] = make_float2(sum.m, sum.s);
            __syncthreads();
            if (w == 0)
                for (int o = 1; o < WAVES; ++o) sum = sum.with({rests[o].x, rests[o].y}, a.c);
        } else {
            wave_sync();
        }
        if (a.rest != nullptr && lane_id() == 0 && (WAVES == 1 || w == 0)) a.rest[r] = as_logit(a, sum);
    }
}

// ---------------------------------------------------------------- rows by sorted lists

struct Buffer {
    Key k[2 * kWave];
};

// One wave at a row.
struct Top {
    const Args& a;
    Buffer& buffer;
    Key list = 0;             // sorted down over the lanes, 0 from K on
    std::uint32_t count = 0;  // waiting in the buffer, fewer than 64 between calls
    LongShare rest;
    float bound;  // what is not larger goes to the rest; NaN: nothing does

    __device__ __forceinline__ Top(const Args& args, Buffer& b) : a(args), buffer(b), bound(__builtin_nanf("")) {}

    __device__ __forceinline__ void drop(Key k) {
        if (k != 0) rest.add(value_of(static_cast<std::uint32_t>(k >> 32)), a.c);
    }
    // Takes in a list that is sorted up.
    __device__ __forceinline__ void take(Key up) {
        const Key low = list > up ? up : list;
        list = wave_steps<kWave, true, kWave / 2>(list > up ? list : up);
        drop(low);
        if (lane_id() >= a.K) {
            drop(list);
            list = 0;
        }
        const std::uint32_t last = static_cast<std::uint32_t>(__shfl(static_cast<int>(list >> 32), a.K - 1, kWave));
        if (last != 0) raise(last);
    }
    // Everything up to this order is known to be beaten by K others.
    // (0x7FFFFFFF would be -0, which is 0 and not below it.)
    __device__ __forceinline__ void raise(std::uint32_t order) {
        bound = value_of(order == 0x7FFFFFFFu ? 0x7FFFFFFEu : order);
    }

    __device__ __forceinline__ void flush() {
        if (count == 0) return;
        wave_sync();
        const Key mine = lane_id() < count ? buffer.k[lane_id()] : 0;
        take(wave_sort<false>(mine));
        count = 0;
    }
    __device__ __forceinline__ void push(bool mine, float v, std::uint32_t index) {
        const std::uint64_t all = __ballot(mine);
        if (all == 0) return;
        if (mine) buffer.k[count + __popcll(all & lanemask_lt())] = key_of(v, index);
        count += __popcll(all);
        if (count < kWave) return;
        wave_sync();
        take(wave_sort<false>(buffer.k[lane_id()]));
        const Key left = buffer.k[kWave + lane_id()];
        wave_sync();
        buffer.k[lane_id()] = left;
        count -= kWave;
        wave_sync();
    }
};

// The elements of vectors first, first + step, ... of a row.
template <typename T, int V>
__device__ __forceinline__ void scan(Top& top, const T* z, std::uint32_t first, std::uint32_t step) {
    const Args& a = top.a;
    bool begun = false;
    for (Range<V> range{first, step, a.C}; range.first * V < a.C; range.first += step * kBatch) {
        Ahead<T, V> raw;
        raw.load(z, range);
        Elements<T, V> e(raw, range);
        if (!begun) top.raise(kth_lane(e.largest(kNone), a.K) - 1);  // itself may be one of the K
        begun = true;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            // larger than the bound at the start of this vector: elements equal to a
            // bound from among these may come before it in the row
            const float bound = top.bound;
            if (__ballot(!(e.most[u] <= bound)) == 0) continue;
            const std::uint32_t last = range.at(u) + V - 1;
            for (std::uint32_t left = e.template leave<true>(u, bound, range); __ballot(left != 0) != 0; left &= left - 1) {
                const std::uint32_t c = left != 0 ? last - __builtin_ctz(left) : 0u;
                top.push(left != 0, static_cast<float>(z[c]), c);
            }
        }
        e.add_to(top.rest, a.c);
    }
    top.flush();
}

// By the wave that has the row's list and, in any lane, the sum of its rest.
template <typename T>
__device__ __forceinline__ void write(const Top& top, const T* z, std::uint64_t r, Share rest) {
    const Args& a = top.a;
    const std::uint32_t l = lane_id();
    if (l < a.K) {
        const std::uint32_t i = index_of(top.list);
        static_cast<T*>(a.values)[r * a.ldv + l] = z[i];
        a.ids[r * a.ldi + l] = static_cast<std::int32_t>(i);
    }
    if (a.rest != nullptr && l == 0) a.rest[r] = as_logit(a, rest);
}

// The rows that stream_kernel marked, a wave each: 4,096 x 50,000 bf16 rows whose
// every element beats those before it take 1,800 us.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) wave_kernel(Args a) {
    __shared__ Buffer buffers[kWaves];
    const std::uint32_t w = uniform(threadIdx.x / kWave);
    const std::uint64_t step = static_cast<std::uint64_t>(gridDim.x) * kWaves;
    for (std::uint64_t r = static_cast<std::uint64_t>(blockIdx.x) * kWaves + w; r < a.n; r += step) {
        if (a.ids[r * a.ldi] != kToSort) continue;
        const T* z = static_cast<const T*>(a.z) + r * a.ldz;
        Top top(a, buffers[w]);
        scan<T, V>(top, z, 0, kWave);
        write<T>(top, z, r, wave_join_share(top.rest.share(a.c), a.c));
    }
}

// The same, a workgroup each, whose waves take the vectors in turn.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) block_kernel(Args a) {
    __shared__ Buffer buffers[kWaves];
    __shared__ Key lists[kWaves][kWave];
    __shared__ float2 rests[kWaves];
    const std::uint32_t w = uniform(threadIdx.x / kWave);
    for (std::uint64_t r = blockIdx.x; r < a.n; r += gridDim.x) {
        if (a.ids[r * a.ldi] != kToSort) continue;
        const T* z = static_cast<const T*>(a.z) + r * a.ldz;
        Top top(a, buffers[w]);
        scan<T, V>(top, z, w * kWave, kThreads);
        if (w != 0) {
            lists[w][kWave - 1 - lane_id()] = top.list;
            const Share rest = wave_join_share(top.rest.share(a.c), a.c);
            if (lane_id() == 0) rests[w] = make_float2(rest.m, rest.s);
        }
        __syncthreads();
        if (w == 0) {
            for (int o = 1; o < kWaves; ++o) top.take(lists[o][lane_id()]);
            Share rest = wave_join_share(top.rest.share(a.c), a.c);
            for (int o = 1; o < kWaves; ++o) rest = rest.with({rests[o].x, rests[o].y}, a.c);
            write<T>(top, z, r, rest);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- rows in registers

// How many of the P values of the other lanes of a team, D and more lanes on, are
// larger than v.
template <int TEAM, int P, int D = 1>
__device__ __forceinline__ std::uint32_t larger_elsewhere(float v, const float (&t)[P]) {
    static_assert(TEAM == 4 || TEAM == 16);
    constexpr int turn = TEAM == 16 ? 0x120 + D : D == 1 ? 0x39 : D == 2 ? 0x4E : 0x93;  // row_ror:D, quad_perm turned by D
    std::uint32_t n = 0;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int i = static_cast<int>(__float_as_uint(t[p]));
        const float o = __uint_as_float(static_cast<std::uint32_t>(__builtin_amdgcn_update_dpp(i, i, turn, 0xF, 0xF, false)));
        n += o > v ? 1u : 0u;
    }
    if constexpr (D + 1 < TEAM) return n + larger_elsewhere<TEAM, P, D + 1>(v, t);
    else return n;
}

// A value that K elements of a team reach at least (-inf where none is known), in
// all its lanes: the K-th largest of the lanes' maxima, or, of 4 lanes, that of
// their four largest each.
template <int TEAM, int N>
__device__ __forceinline__ float reached(const float (&v)[N], std::uint32_t K) {
    constexpr int P = TEAM == 4 ? 4 : 1;
    if (K > TEAM * P) return kNone;
    float t[P];  // sorted down
#pragma unroll
    for (int p = 0; p < P; ++p) t[p] = kNone;
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int p = P - 1; p > 0; --p) t[p] = __builtin_amdgcn_fmed3f(t[p - 1], t[p], v[i]);
        t[0] = fmaxf(t[0], v[i]);
    }
    if constexpr (TEAM == kWave) {
        return value_of(kth_lane(t[0], K));
    } else {
        float least = -kNone;
#pragma unroll
        for (int p = 0; p < P; ++p)  // (p of the lane's own are before it, or equal)
            least = larger_elsewhere<TEAM>(t[p], t) + p < K ? t[p] : least;
        return wave_join<TEAM>(least, Smaller());
    }
}

// The sum of v over the lanes of a team up to this one.
template <int TEAM>
__device__ __forceinline__ std::uint32_t team_scan(std::uint32_t x) {
    int v = static_cast<int>(x);
    if constexpr (TEAM == 4) {  // a row of lanes has four teams
        const unsigned l = lane_id() % 4;
        const int one = __builtin_amdgcn_update_dpp(v, v, 0x90, 0xF, 0xF, false);  // quad_perm [0,0,1,2]
        v += l >= 1 ? one : 0;
        const int two = __builtin_amdgcn_update_dpp(v, v, 0x44, 0xF, 0xF, false);  // quad_perm [0,1,0,1]
        v += l >= 2 ? two : 0;
    } else {
        v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);  // row_shr:1
        v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
        v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
        v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    }
    if constexpr (TEAM == kWave) {
        v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
        v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
    }
    return static_cast<std::uint32_t>(v);
}

// Keys of a team that have room in LDS, a multiple of 4.
template <int TEAM>
constexpr std::uint32_t kRoom = TEAM == 4 ? 32 : TEAM == 16 ? 128 : 256;
// A bound that at least K elements reach and at most `most`, or the K-th largest,
// from one that more reach: by halves of the range up to the team's largest.
template <int TEAM, int N>
__device__ __forceinline__ float halved(const float (&v)[N], float bound, std::uint32_t K, std::uint32_t most) {
    float top = kNone;
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, v[i]);
    std::uint32_t lo = order_of(bound), hi = order_of(wave_join<TEAM>(top, Larger())) + 1;
    while (hi - lo > 1) {
        const std::uint32_t mid = lo + (hi - lo) / 2;
        const float b = value_of(mid);
        std::uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) n += v[i] < b ? 0u : 1u;
        n = wave_join<TEAM>(n, Add());
        if (n < K) {
            hi = mid;
        } else {
            lo = mid;
            if (n <= most) break;
        }
    }
    return value_of(lo);
}

// The keys of rows in registers: of 16-bit logits, whose values need the upper 19 bits
// of their order (fp16's 1 + 8 + 10 as fp32), 32 bits with a class of 10: 7M x 32 bf16
// rows take 866 us instead of 1,207 (K = 16).
template <typename T, bool SHORT = sizeof(T) == 2>
struct RowKey {
    using type = Key;
    static __device__ __forceinline__ type of(float v, std::uint32_t c) { return key_of(v, c); }
    static __device__ __forceinline__ std::uint32_t index(type k) { return index_of(k); }
    static __device__ __forceinline__ float value(type k) { return value_of(static_cast<std::uint32_t>(k >> 32)); }
};
template <typename T>
struct RowKey<T, true> {
    using type = std::uint32_t;
    static __device__ __forceinline__ type of(float v, std::uint32_t c) { return order_of(v) >> 13 << 10 | (1023 - c); }
    static __device__ __forceinline__ std::uint32_t index(type k) { return 1023 - (k & 1023); }
    static __device__ __forceinline__ float value(type k) {
        const std::uint32_t order = k >> 10 << 13;  // its lower bits are 0, or 1 of negative values
        return value_of(order & 0x80000000u ? order : order | 0x1FFFu);
    }
};

template <typename K>
__device__ __forceinline__ K larger_key(K a, K b) {
    return a > b ? a : b;
}
// The largest key of a team.
template <int TEAM, int D = 1, typename K>
__device__ __forceinline__ K team_top(K k) {
    if constexpr (D < TEAM) return team_top<TEAM, 2 * D>(larger_key(k, other<D>(k)));
    else return k;
}

// Whether a row of N elements a lane goes to LDS too, where what reaches the bound is
// read again: 7M x 32 fp32 rows take 457 us with it and 618 without (K = 8), 2.45M x
// 100 bf16 ones 328 and 363.  Larger rows leave too few workgroups room (2.45M x 100
// fp32 rows 433, and 423 without), and so do fp32 ones of 16 lanes, whose registers
// suffice for five (800,000 x 200: 230, and 203 without).
template <typename T, int N, int TEAM>
constexpr bool kNear = N * sizeof(T) <= 64 && (TEAM != 16 || sizeof(T) == 2);

// A team holds a row in registers, E vectors of V a lane.  What reaches a value
// that K elements reach, hardly more than K of them where these are few beside
// the row, goes to LDS, and each of those counts the larger ones among them, which
// is its place.  Rows with more of them than there is room for (equal ones, or
// mostly -inf) have their K taken one after the other.  Vector instructions bound it
// as much as memory: 2.45M x 100 fp32 rows take 420 us with K = 8 (1.15 GB: 250 at a
// copy's rate, and 176M vector instructions, 286 at 2.4 GHz), 1,850 if all their
// elements are equal.
template <typename T, int V, int E, int TEAM>
__global__ void __launch_bounds__(kThreads, TEAM > 4 && E * V == 16 ? 5 : 1) registers_kernel(Args a) {
    constexpr int teams = kThreads / TEAM, N = E * V;
    constexpr std::uint32_t room = kRoom<TEAM>;
    using Keys = RowKey<T>;
    using Key = typename Keys::type;
    __shared__ __attribute__((aligned(16))) Key found[teams][room];
    // the row by the lanes' vectors; 64 bytes more put other teams' into other banks
    constexpr bool near = kNear<T, N, TEAM>;
    __shared__ __attribute__((aligned(16))) T rows[near ? teams : 1][near ? TEAM * N + 64 / sizeof(T) : 1];
    Key* mine = found[threadIdx.x / TEAM];
    T* row = rows[near ? threadIdx.x / TEAM : 0];
    const std::uint32_t body = a.C / V * V;
    const auto class_at = [&](std::uint32_t slot) { return slot < body ? slot : slot - body + a.C - V; };
    const auto slot_of = [&](std::uint32_t c) { return c < body ? c : c + body + V - a.C; };
    const std::uint32_t lane = threadIdx.x % TEAM;
    const auto place = [&](int e) { return Place<V>(lane + e * TEAM, a.C); };
    // whether some lanes of the team have a vector e, and whether all have a whole one
    const auto some = [&](int e) { return static_cast<std::uint32_t>(e * TEAM * V) < a.C; };
    const auto whole = [&](int e) { return static_cast<std::uint32_t>((e + 1) * TEAM * V) <= a.C; };
    std::uint32_t valid = 0;  // element i is bit N - 1 - i
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const std::uint32_t skip = place(e).skip;
#pragma unroll
        for (std::uint32_t q = 0; q < V; ++q) valid += valid + (q >= skip ? 1u : 0u);
    }
    const std::uint64_t step = static_cast<std::uint64_t>(gridDim.x) * teams;
    std::uint64_t r = static_cast<std::uint64_t>(blockIdx.x) * teams + threadIdx.x / TEAM;
    vec_t<T, V> ahead[E];
    const auto load = [&](std::uint64_t row) {
        if (row >= a.n) return;
        const T* z = static_cast<const T*>(a.z) + row * a.ldz;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (!some(e)) break;
            const Place<V> at = place(e);
            if (at.any()) ahead[e] = load_as<T, V>(z + at.at);
        }
    };
    load(r);
    for (; r < a.n; r += step) {
        const T* z = static_cast<const T*>(a.z) + r * a.ldz;
        const auto element = [&](std::uint32_t c) {
            if constexpr (near) return row[slot_of(c)];
            else return z[c];
        };
        T* values = static_cast<T*>(a.values) + r * a.ldv;
        std::int32_t* ids = a.ids + r * a.ldi;
        float v[N];
#pragma unroll
        for (int e = 0; e < E; ++e) {
#pragma unroll
            for (int q = 0; q < V; ++q) v[e * V + q] = kNone;
            if (!some(e)) continue;
            const std::uint32_t skip = whole(e) ? 0 : place(e).skip;
#pragma unroll
            for (std::uint32_t q = 0; q < V; ++q) v[e * V + q] = q >= skip ? static_cast<float>(ahead[e][q]) : kNone;
            if constexpr (near) *reinterpret_cast<vec_t<T, V>*>(row + (lane + e * TEAM) * V) = ahead[e];
        }
        load(r + step);
        float bound = reached<TEAM>(v, a.K);
        std::uint32_t reach, own, to, all;
        for (bool again = false;; again = true) {
            reach = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) reach += reach + (v[i] < bound ? 0u : 1u);
            reach &= valid;
            own = __popc(reach);
            to = team_scan<TEAM>(own);
            all = static_cast<std::uint32_t>(__shfl(static_cast<int>(to), TEAM - 1, TEAM));
            if (again || all <= min(room, enough(a.K))) break;
            bound = halved<TEAM>(v, bound, a.K, min(room, enough(a.K)));
        }
        const auto slot = [&](std::uint32_t i) { return (lane + i / V * TEAM) * V + i % V; };
        Share rest;
        if (all <= room) {
            // their places first, then their keys: a register chosen at run time costs
            // two instructions for each that there is, and the row's lines are near
            using Slot = std::uint32_t __attribute__((may_alias));
            auto* slots = reinterpret_cast<Slot*>(mine);
            constexpr std::uint32_t apart = sizeof(Key) / sizeof(Slot);
            for (to -= own; reach != 0; reach &= reach - 1) slots[apart * to++] = slot(N - 1 - __builtin_ctz(reach));
            wave_sync();
#pragma unroll 4
            for (std::uint32_t i = lane; i < all; i += TEAM) {
                const std::uint32_t s = slots[apart * i];
                mine[i] = Keys::of(static_cast<float>(near ? row[s] : z[class_at(s)]), class_at(s));
            }
            if (lane < 3 && all + lane < room) mine[all + lane] = 0;  // for the reads of four
            wave_sync();
        } else {  // read again: the keys of all elements need more registers than all else
            wave_sync();
            Key last = ~Key(0);
            for (std::uint32_t k = 0; k < a.K; ++k) {
                Key best = 0;
#pragma unroll 4
                for (std::uint32_t c = lane; c < a.C; c += TEAM) {
                    const Key key = Keys::of(static_cast<float>(element(c)), c);
                    best = key < last ? larger_key(best, key) : best;
                }
                last = team_top<TEAM>(best);
                if (lane == 0) {
                    values[k] = element(Keys::index(last));
                    ids[k] = static_cast<std::int32_t>(Keys::index(last));
                }
            }
#pragma unroll 1
            for (std::uint32_t c = lane; c < a.C; c += TEAM) {
                const float x = static_cast<float>(element(c));
                if (Keys::of(x, c) < last) rest = rest.with({x, 1.0f}, a.c);
            }
        }
        const float below = all <= room ? bound : kNone;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = v[i] < below ? v[i] : kNone;
            rest.m = fmaxf(rest.m, v[i]);
        }
        const float b = base_of<true>(rest.m);
#pragma unroll
        for (int i = 0; i < N; ++i) rest.s += exp2_of((v[i] - b) * a.c);
        if (all <= room) {
            for (std::uint32_t i = lane; i < all; i += TEAM) {
                const Key k = mine[i];
                std::uint32_t at = 0;
                for (std::uint32_t o = 0; o < all; o += 4) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) at += mine[o + q] > k ? 1u : 0u;
                }
                if (at < a.K) {
                    const std::uint32_t c = Keys::index(k);
                    values[at] = element(c);
                    ids[at] = static_cast<std::int32_t>(c);
                } else {
                    rest = rest.with({Keys::value(k), 1.0f}, a.c);
                }
            }
        }
        wave_sync();
        if (a.rest == nullptr) continue;
        const float top = wave_join<TEAM>(rest.m, Larger());
        rest.scale_to(top, a.c);
        const float sum = wave_join<TEAM>(rest.s, Add());
        if (lane == 0) a.rest[r] = as_logit(a, {top, sum});
    }
}

// ---------------------------------------------------------------- launches

template <typename Kernel>
void launch_all(Kernel kernel, const Args& a, std::uint64_t rows, std::uint64_t most, hipStream_t st) {
    const std::uint64_t blocks = std::min<std::uint64_t>((a.n + rows - 1) / rows, most);
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, st, a);
}
template <typename T, int V, int E, int TEAM>
void in_registers(const Args& a, hipStream_t st) {
    static std::uint32_t perCu;
    const auto kernel = registers_kernel<T, V, E, TEAM>;
    launch_all(kernel, a, kThreads / TEAM, resident_blocks(kernel, kThreads, perCu), st);
}

// Rows of up to 1,024 classes are held in registers: by 4 lanes of a wave with up to
// 32 elements each where these have room for K, by 16 with as many, by a wave with
// 16.  Longer ones are streamed.
template <typename T>
void launch(const Args& a, hipStream_t st) {
    constexpr int V = kVec<T>;
    const std::uint32_t C = a.C;
    if (C < V) return in_registers<T, 1, 8, 4>(a, st);
    if (C <= 4 * V) return in_registers<T, V, 1, 4>(a, st);
    if (a.K <= 16) {
        if (C <= 8 * V) return in_registers<T, V, 2, 4>(a, st);
        if (C <= 64) return in_registers<T, V, 16 / V, 4>(a, st);
        if (C <= 128) return in_registers<T, V, 32 / V, 4>(a, st);
    }
    if (C <= 128) return in_registers<T, V, 8 / V, 16>(a, st);
    if (C <= 256) return in_registers<T, V, 16 / V, 16>(a, st);
    if (C <= 512) return in_registers<T, V, 32 / V, 16>(a, st);
    if (C <= 1024) return in_registers<T, V, 16 / V, 64>(a, st);
    // A wave a row where there are three for each SIMD (4,096 x 50,000 bf16, K = 32: 100 us
    // instead of 112 with a workgroup a row, of which an uneven number are left at the
    // end) and K leaves its bound room; a workgroup else.
    if (C <= kWaveClasses || (a.K <= 32 && a.n >= 12ull * device_cus())) {
        launch_all(stream_kernel<T, V, 1>, a, kWaves, 1u << 20, st);
        launch_all(wave_kernel<T, V>, a, kWaves, 2048, st);
    } else {
        launch_all(stream_kernel<T, V, kWaves>, a, 1, 1u << 20, st);
        launch_all(block_kernel<T, V>, a, 1, 2048, st);
    }
}

}  // namespace
}  // namespace tcc

extern "C" int tcc_top_logits(const void* logits, uint64_t ldz, uint32_t dtype, uint64_t n, uint32_t C, uint32_t K,
                              float temperature, void* values, uint64_t ldv, int32_t* ids, uint64_t ldi, float* rest,
                              void* stream) {
    using namespace tcc;
    clear_last_error();
    TCC_REQUIRE(dtype_bytes(dtype) != 0, TCC_ERR_INVALID_ARGUMENT, "top logits: unknown element type");
    TCC_REQUIRE(K >= 1 && K <= C, TCC_ERR_INVALID_ARGUMENT, "top logits: between one and all of a row's classes");
    TCC_REQUIRE(temperature >= 1e-18f && temperature <= 1e18f, TCC_ERR_INVALID_ARGUMENT,
                "top logits: the temperature lies between 1e-18 and 1e18");
    TCC_REQUIRE(K <= kMostTop, TCC_ERR_UNSUPPORTED, "top logits: at most 64 a row");
    TCC_REQUIRE(C <= 0x7FFFFFFFu, TCC_ERR_UNSUPPORTED, "top logits: fewer than 2^31 classes");
    TCC_REQUIRE(n < (1ull << 40), TCC_ERR_UNSUPPORTED, "top logits: fewer than 2^40 rows");
    if (n == 0) return TCC_OK;
    TCC_REQUIRE(logits != nullptr && values != nullptr && ids != nullptr, TCC_ERR_INVALID_ARGUMENT,
                "top logits: a null pointer");
    TCC_REQUIRE(ldz >= C && ldv >= K && ldi >= K, TCC_ERR_INVALID_ARGUMENT,
                "top logits: a row stride below the row's elements");
    Args a{};
    a.z = logits;
    a.ldz = ldz;
    a.n = n;
    a.C = C;
    a.K = K;
    a.T = temperature;
    a.c = static_cast<float>(1.4426950408889634 / static_cast<double>(temperature));
    a.values = values;
    a.ldv = ldv;
    a.ids = ids;
    a.ldi = ldi;
    a.rest = rest;
    if (dtype == TCC_F32) launch<float>(a, as_stream(stream));
    else if (dtype == TCC_BF16) launch<bf16_t>(a, as_stream(stream));
    else launch<f16_t>(a, as_stream(stream));
    TCC_LAUNCH_CHECK();
    return TCC_OK;
}
