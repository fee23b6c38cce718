// The K largest logits of every row, and one logit for the rest
// (include/tcc_training.h).
//
//   ids: the K largest, the lowest index first among equals, NaN above all
//   rest = T log(sum of exp(z_j / T) over the other classes)
//
// A row is read once.  A wave keeps the K largest so far sorted over its lanes,
// as 64-bit keys (the value's order, then the index's), and sends what is larger
// than the last of them into a buffer in LDS; 64 of these at a time are sorted
// and merged (the larger of each pair of a descending and an ascending list are
// the 64 largest of both).  What is not larger, and what a merge drops, goes to
// the sum of the rest, so that nothing is read or subtracted again.  The first
// bound is the K-th largest of the lanes' own maxima, which no more than K of
// the row's elements need exceed.  Rows of up to 4,096 classes have a wave each,
// longer ones a workgroup whose waves' lists are merged.
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

template <typename K>
__device__ __forceinline__ K pair_step(K v, int d, bool larger) {
    const K o = __shfl_xor(v, d, kWave);
    return (v > o) == larger ? v : o;
}
// Sorted over the lanes, a bitonic network: the larger first if `down`.
template <typename K>
__device__ __forceinline__ K wave_sort(K v, bool down) {
    const unsigned l = lane_id();
#pragma unroll
    for (int size = 2; size <= kWave; size <<= 1)
#pragma unroll
        for (int d = size / 2; d > 0; d >>= 1) {
            const bool first = (l & d) == 0, forward = size == kWave || (l & size) == 0;
            v = pair_step(v, d, (first == forward) == down);
        }
    return v;
}
// A bitonic sequence sorted down.
template <typename K>
__device__ __forceinline__ K wave_merge_down(K v) {
    const unsigned l = lane_id();
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) v = pair_step(v, d, (l & d) == 0);
    return v;
}

struct Buffer {
    Key k[2 * kWave];
};

// One wave at a row.
struct Top {
    const Args& a;
    Buffer& buffer;
    Key list = 0;             // sorted down over the lanes, 0 from K on
    std::uint32_t count = 0;  // waiting in the buffer, fewer than 64 between calls
    Share rest;
    float bound;  // what is not larger goes to the rest; NaN: nothing does

    __device__ __forceinline__ Top(const Args& args, Buffer& b) : a(args), buffer(b), bound(__builtin_nanf("")) {}

    __device__ __forceinline__ void drop(Key k) {
        if (k != 0) rest = rest.with({value_of(static_cast<std::uint32_t>(k >> 32)), 1.0f}, a.c);
    }
    // Takes in a list that is sorted up.
    __device__ __forceinline__ void take(Key up) {
        const Key low = list > up ? up : list;
        list = wave_merge_down(list > up ? list : up);
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
        sync();
        const Key mine = lane_id() < count ? buffer.k[lane_id()] : 0;
        take(wave_sort(mine, false));
        count = 0;
    }
    __device__ __forceinline__ void sync() const {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    __device__ __forceinline__ void push(bool mine, float v, std::uint32_t index) {
        const std::uint64_t all = __ballot(mine);
        if (all == 0) return;
        if (mine) buffer.k[count + __popcll(all & lanemask_lt())] = key_of(v, index);
        count += __popcll(all);
        if (count < kWave) return;
        sync();
        take(wave_sort(buffer.k[lane_id()], false));
        const Key left = buffer.k[kWave + lane_id()];
        sync();
        buffer.k[lane_id()] = left;
        count -= kWave;
        sync();
    }
};

// The elements of vectors first, first + step, ... of a row.
template <typename T, int V>
__device__ __forceinline__ void scan(Top& top, const T* z, std::uint32_t first, std::uint32_t step) {
    using F = vec_t<float, V>;
    const Args& a = top.a;
    bool begun = false;
    for (std::uint64_t j = first; j * V < a.C; j += static_cast<std::uint64_t>(step) * kBatch) {  // of the wave's first lane
        F x[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const Place<V> at(static_cast<std::uint32_t>(j + lane_id() + u * step), a.C);
            x[u] = at.any() ? load_any<T, V>(z + at.at) : F(kNone);
        }
        if (!begun) {  // a first bound
            begun = true;
            std::uint32_t own = 0;
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const Place<V> at(static_cast<std::uint32_t>(j + lane_id() + u * step), a.C);
#pragma unroll
                for (std::uint32_t q = 0; q < V; ++q) own = max(own, q >= at.skip ? order_of(x[u][q]) : 0u);
            }
            const std::uint32_t last = static_cast<std::uint32_t>(__shfl(static_cast<int>(wave_sort(own, true)), a.K - 1, kWave));
            if (last != 0) top.raise(last - 1);  // itself may be one of the K
        }
        float m = kNone;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const Place<V> at(static_cast<std::uint32_t>(j + lane_id() + u * step), a.C);
            // larger than the bound at the start of this vector: elements equal to a
            // bound from among these may come before it in the row
            const float bound = top.bound;
            std::uint32_t larger = 0;
#pragma unroll
            for (std::uint32_t q = 0; q < V; ++q) larger |= (q >= at.skip && !(x[u][q] <= bound) ? 1u : 0u) << q;
            if (__ballot(larger != 0) != 0) {
#pragma unroll
                for (std::uint32_t q = 0; q < V; ++q) top.push((larger >> q) & 1, x[u][q], at.at + q);
            }
            if (at.skip != 0) larger |= (1u << at.skip) - 1;
#pragma unroll
            for (int q = 0; q < V; ++q) {
                x[u][q] = (larger >> q) & 1 ? kNone : x[u][q];
                m = fmaxf(m, x[u][q]);
            }
        }
        if (m > top.rest.m) top.rest.scale_to(m, a.c);
        const float b = base_of(top.rest.m);
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
#pragma unroll
            for (int q = 0; q < V; ++q) top.rest.s += exp2_of((x[u][q] - b) * a.c);
    }
    top.flush();
}

__device__ __forceinline__ Share wave_join_share(Share v, float c) {
    const float m = wave_join<kWave>(v.m, Larger());
    v.scale_to(m, c);
    v.s = wave_join<kWave>(v.s, Add());
    return v;
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
    if (a.rest != nullptr && l == 0) a.rest[r] = rest.m == -kNone ? rest.m : base_of(rest.m) + a.T * kLn2 * log2_of(rest.s);
}

// A row a wave.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) wave_kernel(Args a) {
    __shared__ Buffer buffers[kWaves];
    const std::uint32_t w = uniform(threadIdx.x / kWave);
    const std::uint64_t step = static_cast<std::uint64_t>(gridDim.x) * kWaves;
    for (std::uint64_t r = static_cast<std::uint64_t>(blockIdx.x) * kWaves + w; r < a.n; r += step) {
        const T* z = static_cast<const T*>(a.z) + r * a.ldz;
        Top top(a, buffers[w]);
        scan<T, V>(top, z, 0, kWave);
        write<T>(top, z, r, wave_join_share(top.rest, a.c));
    }
}

// A row a workgroup: its waves take the vectors in turn.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) block_kernel(Args a) {
    __shared__ Buffer buffers[kWaves];
    __shared__ Key lists[kWaves][kWave];
    __shared__ float2 rests[kWaves];
    const std::uint32_t w = uniform(threadIdx.x / kWave);
    for (std::uint64_t r = blockIdx.x; r < a.n; r += gridDim.x) {
        const T* z = static_cast<const T*>(a.z) + r * a.ldz;
        Top top(a, buffers[w]);
        scan<T, V>(top, z, w * kWave, kThreads);
        if (w != 0) {
            lists[w][kWave - 1 - lane_id()] = top.list;
            const Share rest = wave_join_share(top.rest, a.c);
            if (lane_id() == 0) rests[w] = make_float2(rest.m, rest.s);
        }
        __syncthreads();
        if (w == 0) {
            for (int o = 1; o < kWaves; ++o) top.take(lists[o][lane_id()]);
            Share rest = wave_join_share(top.rest, a.c);
            for (int o = 1; o < kWaves; ++o) rest = rest.with({rests[o].x, rests[o].y}, a.c);
            write<T>(top, z, r, rest);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- launches

template <typename T>
void launch(const Args& a, hipStream_t st) {
    const bool wave = a.C <= kWaveClasses;
    const std::uint64_t blocks = std::min<std::uint64_t>(wave ? (a.n + kWaves - 1) / kWaves : a.n, 1u << 20);
    const dim3 grid(static_cast<unsigned>(blocks));
    if (a.C < kVec<T>) hipLaunchKernelGGL((wave_kernel<T, 1>), grid, dim3(kThreads), 0, st, a);
    else if (wave) hipLaunchKernelGGL((wave_kernel<T, kVec<T>>), grid, dim3(kThreads), 0, st, a);
    else hipLaunchKernelGGL((block_kernel<T, kVec<T>>), grid, dim3(kThreads), 0, st, a);
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
    TCC_REQUIRE(temperature > 0.0f && temperature < 1e18f, TCC_ERR_INVALID_ARGUMENT,
                "top logits: the temperature is positive");
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
