// Rows of an embedding table and their gradient (include/tcc_training.h).
//
//   lookup:   out[i]  = scale * table[ids[i]]
//   gradient: grad[v] = scale * sum over {i : ids[i] = v} of dOut[i]
//
// Both move bytes and compute next to nothing.  The lookup is bound by the
// lines of 128 bytes that its rows lie in: 2.45M rows of 100 bf16 from a table
// of as many take 243 us, 735 MB of ids, distinct rows and output (3.0 TB/s), or
// 1.17 GB past the L2 by the counters (4.8 TB/s).  A lane takes what the rows'
// alignment allows, so that odd widths go element by element: 101 columns take
// 539 us, 102 take 353 (fp32: 318 for 100 columns, 727 and 481), and their
// gradients 770 and 389 where 100 columns take 396 (fp32: 622, 951, 616).
//
// The gradient sorts the ids with their positions (stable, so that a row's
// terms have one order and the sums the same bits every time), then walks the
// sorted positions in chunks of equal length, whatever the ids' frequencies:
// a hub node with thousands of rows is spread over as many chunks as it needs,
// and its parts are joined afterwards in chunk order (by one workgroup for each
// hub: 2.45M rows of 100 fp32 take 665 us with a tenth of them in one, 950 with
// all of them).  Atomics on the rows
// would spare the sort, but add in no fixed order and round every partial sum
// of a bf16 row.  A few rows need no sort (few_grad_kernel), up to 65,536 one
// of a launch for each 11 bits of the rows (pass_kernel), the others passes of
// 8 bits and three launches: 2.45M rows of 100 fp32 into as many take 600 us,
// of which the sums are 486 (1.96 GB, 4.0 TB/s: rows of 400 bytes in the sorted
// order are read at random and share lines), the sort 95, the parts 20 and the
// windows' marks 5.
#include <algorithm>

#include "../../include/tcc_spmm_cnic.h"
#include "../../include/tcc_swtcf.h"
#include "../../include/tcc_training.h"
#include "primitives.hpp"
#include "row_types.hpp"

namespace tcc {
namespace {

constexpr int kThreads = 256;
constexpr std::uint32_t kNoRow = 0xFFFFFFFFu;

// The ids as the caller has them; row(i) is kNoRow for padding and for ids
// outside [0, V), which set `bad`.
struct Ids {
    const void* p;
    std::uint64_t V;
    std::int64_t padding;
    std::uint32_t wide;  // int64
    __device__ __forceinline__ std::uint32_t row(std::uint64_t i, bool& bad) const {
        return row_of(wide ? load_global<std::int64_t>(static_cast<const std::int64_t*>(p) + i)
                           : load_global<std::int32_t>(static_cast<const std::int32_t*>(p) + i),
                      bad);
    }
    __device__ __forceinline__ std::uint32_t row_of(std::int64_t id, bool& bad) const {
        const bool in = static_cast<std::uint64_t>(id) < V;
        bad |= !in;
        return in && id != padding ? static_cast<std::uint32_t>(id) : kNoRow;
    }
    // R ids, `step` apart from i on (the last id where they pass it), all
    // loaded before the first is looked at.
    template <int R>
    __device__ __forceinline__ void rows(std::uint64_t i, std::uint64_t step, std::uint64_t n, std::uint32_t (&v)[R],
                                         bool& bad) const {
        std::int64_t id[R];
        if (wide) {
#pragma unroll
            for (int r = 0; r < R; ++r)
                id[r] = load_global<std::int64_t>(static_cast<const std::int64_t*>(p) + min(i + r * step, n - 1));
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r)
                id[r] = load_global<std::int32_t>(static_cast<const std::int32_t*>(p) + min(i + r * step, n - 1));
        }
#pragma unroll
        for (int r = 0; r < R; ++r) v[r] = row_of(id[r], bad);
    }
};

__device__ __forceinline__ void report(std::uint32_t* err, bool bad) {
    if (err != nullptr && bad) *err = TCC_DEVERR_FEATURE_INDEX;
}

// ---------------------------------------------------------------- lookup

constexpr int kLookupUnroll = 4;

// The output as one run of n * colsV vectors, kThreads * kLookupUnroll of
// them a workgroup, so that no lane idles whatever the width.  Large outputs
// are written past the caches' order, which leaves those to rows that come
// again: 2.45M x 100 rows of bf16 248 us instead of 270, of fp32 323 instead
// of 359 (4 vectors a lane; with 2 of them 257 and 318, with 8 over 600).
// `from`: the launch's first vector.
template <typename T, int N, bool ONCE>
__global__ void __launch_bounds__(kThreads) lookup_kernel(const T* __restrict__ table, std::uint64_t ldt, Ids ids,
                                                         std::uint64_t n, std::uint32_t colsV, float scale,
                                                         T* __restrict__ out, std::uint64_t ldo, std::uint32_t* err,
                                                         std::uint64_t from) {
    const std::uint64_t first = from + static_cast<std::uint64_t>(blockIdx.x) * (kThreads * kLookupUnroll);
    const std::uint64_t row0 = first / colsV;
    const std::uint32_t col0 = static_cast<std::uint32_t>(first - row0 * colsV);
    std::uint64_t i[kLookupUnroll];
    std::uint32_t c[kLookupUnroll], v[kLookupUnroll];
    bool bad = false;
#pragma unroll
    for (int u = 0; u < kLookupUnroll; ++u) {
        const std::uint32_t at = col0 + u * kThreads + threadIdx.x;
        const std::uint32_t r = at / colsV;
        i[u] = row0 + r;
        c[u] = (at - r * colsV) * N;
        v[u] = kNoRow;
        if (i[u] < n) v[u] = ids.row(i[u], bad);
    }
    vec_t<float, N> x[kLookupUnroll];
#pragma unroll
    for (int u = 0; u < kLookupUnroll; ++u) {
        x[u] = vec_t<float, N>(0.0f);
        if (v[u] != kNoRow) x[u] = load_row<T, N>(table + v[u] * ldt + c[u]) * scale;
    }
#pragma unroll
    for (int u = 0; u < kLookupUnroll; ++u)
        if (i[u] < n) write_out<ONCE, T, N>(out + i[u] * ldo + c[u], x[u]);
    report(err, bad);
}

// ---------------------------------------------------------------- gradient

// Keys of the sort: row << 32 | position, kNoRow replaced by V so that the
// rows that do not count come last.
struct IdKeys {
    Ids ids;
    std::uint64_t n;
    std::uint32_t* err;
    __device__ __forceinline__ void load(std::uint64_t first, std::uint64_t (&k)[kPrimRounds], bool& bad) const {
        std::uint32_t v[kPrimRounds];
        ids.rows<kPrimRounds>(first, kWave, n, v, bad);
#pragma unroll
        for (int r = 0; r < kPrimRounds; ++r)
            k[r] = (v[r] == kNoRow ? ids.V : static_cast<std::uint64_t>(v[r])) << 32 |
                   min(first + static_cast<std::uint64_t>(r) * kWave, n - 1);
    }
    __device__ __forceinline__ void report(bool bad) const { tcc::report(err, bad); }
};

// A pass of the sort of up to kPassRows rows by a digit of up to kDigitBits
// bits, in one launch: every workgroup counts the digits of all keys, apart for
// those before its own, and so knows where each digit's run begins and its own
// keys' places in it.  The first pass also clears the windows' marks.  Counting
// costs a workgroup what its CU can read, so that it grows with n, while passes
// of three launches cost what these follow each other in: a gradient of rows of
// 32 fp32 into 1,500 takes (one pass) 18 us for 12,000 rows, 32 for 65,000 and
// 46 for 100,000, with passes of three launches 31, 41 and 45; into 70,000
// (two passes) 31, 50 and 75, with three launches 54, 59 and 67.
constexpr int kDigitBits = 11;
constexpr std::uint32_t kDigits = 1u << kDigitBits;
constexpr int kPassThreads = 1024, kPassWaves = kPassThreads / kWave, kPassUnroll = 8;
constexpr std::uint64_t kPassRows = 65536;

// The lanes of `mask` below this one.
__device__ __forceinline__ std::uint32_t rank_in(std::uint64_t mask) {
    return __builtin_popcountll(mask & ((1ull << __lane_id()) - 1ull));
}

struct SortedKeys {
    const std::uint64_t* keys;
    __device__ __forceinline__ std::uint64_t key(std::uint64_t i, bool&) const { return load_global<std::uint64_t>(keys + i); }
    template <int R>
    __device__ __forceinline__ void rows(std::uint64_t i, std::uint64_t step, std::uint64_t n, std::uint32_t (&v)[R],
                                         bool&) const {
#pragma unroll
        for (int r = 0; r < R; ++r)
            v[r] = static_cast<std::uint32_t>(load_global<std::uint64_t>(keys + min(i + r * step, n - 1)) >> 32);
    }
};

struct FirstKeys {
    Ids ids;
    __device__ __forceinline__ std::uint64_t key(std::uint64_t i, bool& bad) const {
        const std::uint32_t v = ids.row(i, bad);
        return (v == kNoRow ? ids.V : static_cast<std::uint64_t>(v)) << 32 | i;
    }
    template <int R>
    __device__ __forceinline__ void rows(std::uint64_t i, std::uint64_t step, std::uint64_t n, std::uint32_t (&v)[R],
                                         bool& bad) const {
        ids.rows<R>(i, step, n, v, bad);
#pragma unroll
        for (int r = 0; r < R; ++r) v[r] = v[r] == kNoRow ? static_cast<std::uint32_t>(ids.V) : v[r];
    }
};

template <typename Src>
__global__ void __launch_bounds__(kPassThreads) pass_kernel(Src src, std::uint32_t n, std::uint32_t shift,
                                                           std::uint32_t bits, std::uint64_t* __restrict__ out,
                                                           std::uint64_t* __restrict__ marks, std::uint64_t markWords,
                                                           std::uint32_t* err) {
    __shared__ std::uint32_t before[kDigits], rest[kDigits], waveSums[kPassWaves];
    const std::uint32_t t = threadIdx.x, first = blockIdx.x * kPassThreads, mask = (1u << bits) - 1u;
    for (std::uint64_t i = first + t; i < markWords; i += static_cast<std::uint64_t>(gridDim.x) * kPassThreads) marks[i] = 0;
    bool bad = false;
    const bool have = first + t < n;
    std::uint64_t key = 0;
    if (have) key = src.key(first + t, bad);
#pragma unroll
    for (std::uint32_t d = 0; d < kDigits; d += kPassThreads) before[d + t] = rest[d + t] = 0;
    __syncthreads();
    for (std::uint32_t i = t; i < n; i += kPassUnroll * kPassThreads) {
        std::uint32_t v[kPassUnroll];
        src.template rows<kPassUnroll>(i, kPassThreads, n, v, bad);
#pragma unroll
        for (int r = 0; r < kPassUnroll; ++r) {
            const std::uint32_t at = i + r * kPassThreads;  // a wave's are all before the workgroup's or none
            if (at >= n) continue;
            const std::uint32_t d = v[r] >> shift & mask;
            std::uint32_t* const c = at < first ? before : rest;
            const std::uint64_t active = __ballot(1);
            if (__ballot(d == uniform(d)) == active) {  // one digit for all, as a hub's are: not one after the other
                if (rank_in(active) == 0) atomicAdd(c + d, static_cast<std::uint32_t>(__builtin_popcountll(active)));
            } else {
                atomicAdd(c + d, 1u);
            }
        }
    }
    if (blockIdx.x == 0) report(err, bad);
    __syncthreads();
    // where each digit's run begins for this workgroup: the digits below, and its own before
    constexpr int E = kDigits / kPassThreads;
    std::uint32_t c[E], b[E], sum = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        b[e] = before[t * E + e];
        c[e] = b[e] + rest[t * E + e];
        sum += c[e];
    }
    const std::uint32_t inc = wave_inclusive_scan(sum);
    const std::uint32_t wave = uniform(t / kWave), lane = __lane_id();
    if (lane == kWave - 1) waveSums[wave] = inc;
    __syncthreads();
    std::uint32_t at = inc - sum;
    for (std::uint32_t w = 0; w < wave; ++w) at += waveSums[w];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        before[t * E + e] = at + b[e];
        at += c[e];
    }
    // keys of the same digit in a wave by lanes, the waves in turn
    const std::uint32_t digit = static_cast<std::uint32_t>(key >> 32) >> shift & mask;
    std::uint64_t same = __ballot(have);
    for (std::uint32_t k = 0; k < bits; ++k) {
        const bool one = digit >> k & 1u;
        const std::uint64_t ones = __ballot(one);
        same &= one ? ones : ~ones;
    }
    const std::uint32_t rank = rank_in(same);
    std::uint32_t place = 0;
    for (std::uint32_t w = 0; w < kPassWaves; ++w) {
        __syncthreads();
        if (w != wave || !have) continue;
        place = before[digit] + rank;
        if (rank == 0) before[digit] = place + __builtin_popcountll(same);
    }
    if (have) out[place] = key;
}

struct GradArgs {
    const std::uint64_t* keys;  // sorted
    const void* dOut;
    void* grad;
    float* parts;  // [2 * chunks][D]: sums of a chunk's first row (begun before it) and last row (going on after it)
    std::uint8_t* mark;  // [windows]: 1 where a row occurs
    std::uint64_t n, V, ldd, ldg;
    std::uint32_t D, chunk, chunks, laneBits, joinBlocks, zeroRows, waveWindows;
    float scale;
    int accumulate;
};

__device__ __forceinline__ std::uint32_t key_row(std::uint64_t k) { return static_cast<std::uint32_t>(k >> 32); }

template <typename T, int N>
__device__ __forceinline__ void write_sum(const GradArgs& a, std::uint32_t v, std::uint32_t c, vec_t<float, N> s) {
    T* p = static_cast<T*>(a.grad) + v * a.ldg + c;
    s *= a.scale;
    if (a.accumulate) s += load_row<T, N>(p);
    store_row<T, N>(p, s);
}

constexpr int kGradUnroll = 4;  // rows a lane has in flight

// Rows that do not occur are zeroed where they lie: those of a window of this
// many rows that holds others, by the teams that write these (a row's lines
// are then written whole, unless past the caches' order, which took 534 us for
// 2.45M x 100 rows instead of 488; zeroed apart from the sums, they took 577),
// those of empty windows by the join's launch.
constexpr std::uint32_t kWindow = 16;

// Zeros in the rows between q (kNoRow: none before) and r (V: none after)
// that share a window with either.
template <typename T, int N>
__device__ __forceinline__ void zero_between(const GradArgs& a, std::uint32_t q, std::uint32_t r, std::uint32_t c) {
    const std::uint32_t V = static_cast<std::uint32_t>(a.V);
    std::uint32_t v = q + 1;  // 0 where none is before
    const std::uint32_t endOfQ = q == kNoRow ? 0u : q + min(r - q, kWindow - q % kWindow);
    const std::uint32_t startOfR = r < V ? r / kWindow * kWindow : V;
    for (; v < r; ++v) {
        if (v >= endOfQ && v < startOfR) v = startOfR;  // an empty window begins
        if (v >= r) break;
        store_row<T, N>(static_cast<T*>(a.grad) + v * a.ldg + c, vec_t<float, N>(0.0f));
    }
}

// A team of 2^laneBits lanes sums one chunk of the sorted rows, the block's
// keys in LDS: 128 KB of them, one workgroup a CU, where a row is one vector and a
// chunk 64 rows (600,000 rows into 400,000 take 138 us with 4 fp32 columns, 111
// with 8 and 101 with 16).
template <typename T, int N>
__global__ void __launch_bounds__(kThreads) grad_kernel(GradArgs a) {
    extern __shared__ std::uint64_t ldsKeys[];
    const std::uint32_t teams = kThreads >> a.laneBits;
    const std::uint64_t base = static_cast<std::uint64_t>(blockIdx.x) * teams * a.chunk;
    const std::uint32_t here = static_cast<std::uint32_t>(min(a.n - base, static_cast<std::uint64_t>(teams * a.chunk)));
    for (std::uint32_t i = threadIdx.x; i < here; i += kThreads) ldsKeys[i] = a.keys[base + i];
    const std::uint32_t none = static_cast<std::uint32_t>(a.V);
    const std::uint32_t blockBefore = base > 0 ? key_row(a.keys[base - 1]) : kNoRow;
    const std::uint32_t blockAfter = base + here < a.n ? key_row(a.keys[base + here]) : kNoRow;
    __syncthreads();
    const std::uint32_t mine = threadIdx.x >> a.laneBits;
    const std::uint32_t lane = threadIdx.x & ((1u << a.laneBits) - 1u);
    const std::uint32_t lo = mine * a.chunk, hi = min(lo + a.chunk, here);
    if (lo >= hi) return;
    const std::uint64_t team = static_cast<std::uint64_t>(blockIdx.x) * teams + mine;
    const std::uint32_t before = lo > 0 ? key_row(ldsKeys[lo - 1]) : blockBefore;
    const std::uint32_t after = hi < here ? key_row(ldsKeys[hi]) : blockAfter;
    const T* dOut = static_cast<const T*>(a.dOut);
    float* headPart = a.parts + 2 * team * a.D;
    for (std::uint32_t c = lane * N; c < a.D; c += N << a.laneBits) {
        std::uint32_t cur = kNoRow;  // the row being summed; none: rows that do not count
        bool head = false;
        vec_t<float, N> s(0.0f);
        for (std::uint32_t i = lo; i < hi; i += kGradUnroll) {
            std::uint32_t v[kGradUnroll];
            vec_t<T, N> x[kGradUnroll];
#pragma unroll
            for (int u = 0; u < kGradUnroll; ++u) {
                const std::uint64_t k = ldsKeys[min(i + u, hi - 1)];
                v[u] = key_row(k);
                x[u] = vec_t<T, N>(T(0.0f));
                if (v[u] != none)  // rows that do not count are not read
                    x[u] = load_global<vec_t<T, N>>(dOut + (k & 0xFFFFFFFFu) * a.ldd + c);
            }
#pragma unroll
            for (int u = 0; u < kGradUnroll; ++u) {
                if (i + u >= hi) break;
                const vec_t<float, N> f = __builtin_convertvector(x[u], vec_t<float, N>);
                if (v[u] == cur) {
                    s += f;
                    continue;
                }
                if (cur < none) {
                    if (head) *reinterpret_cast<vec_t<float, N>*>(headPart + c) = s;
                    else write_sum<T, N>(a, cur, c, s);
                }
                const std::uint32_t last = i + u == lo ? before : cur;
                head = i + u == lo && v[u] == before;
                if (!head && !a.accumulate) {
                    zero_between<T, N>(a, last, v[u], c);
                    if (c == 0 && v[u] != none) a.mark[v[u] / kWindow] = 1;
                }
                cur = v[u];
                s = f;
            }
        }
        if (cur >= none) continue;
        if (base + hi == a.n && !a.accumulate) zero_between<T, N>(a, cur, none, c);
        if (head) *reinterpret_cast<vec_t<float, N>*>(headPart + c) = s;
        else if (cur == after) *reinterpret_cast<vec_t<float, N>*>(headPart + a.D + c) = s;
        else write_sum<T, N>(a, cur, c, s);
    }
}

// A workgroup's share of the empty windows: a wave zeroes one of its own after
// the other.
template <typename T, int N>
__device__ __forceinline__ void zero_windows(const GradArgs& a, std::uint32_t block) {
    const std::uint64_t wave = static_cast<std::uint64_t>(block) * (kThreads / kWave) + threadIdx.x / kWave;
    const std::uint64_t first = wave * a.waveWindows, windows = (a.V + kWindow - 1) / kWindow, w = first + __lane_id();
    const bool mine = __lane_id() < a.waveWindows && w < windows;
    std::uint64_t empty = __ballot(mine && a.mark[min(w, windows - 1)] == 0);
    while (empty != 0) {
        const std::uint64_t v0 = (first + __builtin_ctzll(empty)) * kWindow;
        empty &= empty - 1;
        const std::uint32_t cols = a.D / N, rows = static_cast<std::uint32_t>(min<std::uint64_t>(kWindow, a.V - v0));
        T* p = static_cast<T*>(a.grad) + v0 * a.ldg;
        if (a.ldg == a.D) {
            for (std::uint32_t i = __lane_id(); i < rows * cols; i += kWave)
                store_row<T, N>(p + static_cast<std::uint64_t>(i) * N, vec_t<float, N>(0.0f));
        } else {
            for (std::uint32_t i = __lane_id(); i < rows * cols; i += kWave) {
                const std::uint32_t r = i / cols;
                store_row<T, N>(p + r * a.ldg + (i - r * cols) * N, vec_t<float, N>(0.0f));
            }
        }
    }
}

// Adds the parts of the rows that go on after the chunk they begin in, a team
// for each such chunk, and zeroes the empty windows (blocks from joinBlocks
// on); a row of many parts (a hub's) is added by the whole
// workgroup, each of its teams taking every so many-th part.
constexpr std::uint32_t kLongRow = 16, kJoinUnroll = 8;
template <typename T, int N>
__global__ void __launch_bounds__(kThreads) join_kernel(GradArgs a) {
    __shared__ std::uint32_t rowOf[kThreads], partsOf[kThreads];
    __shared__ float sums[kThreads * N];
    if (blockIdx.x >= a.joinBlocks) {
        zero_windows<T, N>(a, blockIdx.x - a.joinBlocks);
        return;
    }
    const std::uint32_t teams = kThreads >> a.laneBits, mine = threadIdx.x >> a.laneBits;
    const std::uint32_t lane = threadIdx.x & ((1u << a.laneBits) - 1u);
    const std::uint32_t first = blockIdx.x * teams, team = first + mine;
    const std::uint32_t none = static_cast<std::uint32_t>(a.V);
    std::uint32_t v = none, count = 0;  // parts after the first
    if (team + 1 < a.chunks) {
        const std::uint64_t lo = static_cast<std::uint64_t>(team) * a.chunk, hi = lo + a.chunk;
        const std::uint32_t own = key_row(a.keys[hi - 1]), next = key_row(a.keys[hi]);
        const std::uint32_t before = lo > 0 ? key_row(a.keys[lo - 1]) : none;
        if (own != none && next == own && before != own) {
            v = own;
            // the last chunk that begins with the row: steps that double, then halve
            std::uint32_t last = team + 1, step = 1;
            const auto begins = [&](std::uint32_t k) {
                return k < a.chunks && key_row(a.keys[static_cast<std::uint64_t>(k) * a.chunk]) == v;
            };
            while (begins(last + step)) {
                last += step;
                step *= 2;
            }
            for (; step > 0; step /= 2)
                if (begins(last + step)) last += step;
            count = last - team;
        }
    }
    if (lane == 0) {
        rowOf[mine] = v;
        partsOf[mine] = count;
    }
    const auto part = [&](std::uint64_t k, std::uint32_t c) {
        return load_global<vec_t<float, N>>(a.parts + k * a.D + c);
    };
    // the first parts of the chunks t + k, t + k + step, ... up to t + last, kJoinUnroll
    // of them loaded before the first is added
    const auto add_parts = [&](vec_t<float, N>& s, std::uint32_t t, std::uint32_t k, std::uint32_t step, std::uint32_t last,
                               std::uint32_t c) {
        for (; k <= last; k += kJoinUnroll * step) {
            vec_t<float, N> x[kJoinUnroll];
#pragma unroll
            for (std::uint32_t u = 0; u < kJoinUnroll; ++u) x[u] = part(2ull * (t + min(k + u * step, last)), c);
#pragma unroll
            for (std::uint32_t u = 0; u < kJoinUnroll; ++u)
                if (k + u * step <= last) s += x[u];
        }
    };
    if (v != none && count <= kLongRow) {
        for (std::uint32_t c = lane * N; c < a.D; c += N << a.laneBits) {
            vec_t<float, N> s = part(2ull * team + 1, c);
            add_parts(s, team, 1, 1, count, c);
            write_sum<T, N>(a, v, c, s);
        }
    }
    __syncthreads();
    for (std::uint32_t t = 0; t < teams; ++t) {
        if (partsOf[t] <= kLongRow) continue;  // the same for the whole workgroup
        const std::uint32_t many = partsOf[t];
        for (std::uint32_t c0 = 0; c0 < a.D; c0 += N << a.laneBits) {
            const std::uint32_t c = c0 + lane * N;
            vec_t<float, N> s(0.0f);
            if (c < a.D) {
                if (mine == 0) s = part(2ull * (first + t) + 1, c);
                add_parts(s, first + t, 1 + mine, teams, many, c);
            }
            *reinterpret_cast<vec_t<float, N>*>(sums + threadIdx.x * N) = s;
            __syncthreads();
            if (mine == 0 && c < a.D) {
                for (std::uint32_t o = 1; o < teams; ++o)
                    s += *reinterpret_cast<const vec_t<float, N>*>(sums + ((o << a.laneBits) + lane) * N);
                write_sum<T, N>(a, rowOf[t], c, s);
            }
            __syncthreads();
        }
    }
}

// ---------------------------------------------------------------- few rows

// Without a sort, in one launch: every workgroup holds the ids, and the wave of
// the first position of each row looks for the others.  That is n^2 / 64
// comparisons, which a few thousand rows spread over the GPU need less time for
// than a sort's launches follow each other in: rows of 32 fp32 into 1,500 (and
// 70,000) take 6 us (7) for 1,000 of them, 14 (16) for 3,000 and 26 (27) for
// 4,000, sorted 15 (29) for any of these.  One wave adds all rows of an id here,
// column by column, so that a hub is not spread: 3,000 rows of one id take 38, 108
// and 1,573 us for 32, 128 and 602 fp32 columns (sorted 20, 22 and 85), where
// 1,500 ids take 14, 14 and 16 (sorted 15, 14 and 22).
constexpr std::uint64_t kFewRows = 3000;
constexpr std::uint64_t kFewTableRows = 1ull << 31;  // so that those that zero stay far below 2^32 threads
constexpr std::uint32_t kFewZeroRows = 256;  // rows of a workgroup that zeroes, at most

template <typename T, int N>
__global__ void __launch_bounds__(kThreads) few_grad_kernel(GradArgs a, Ids ids, std::uint32_t* err) {
    extern __shared__ std::uint32_t rowOf[];  // [n], then a list of n positions for each wave
    __shared__ std::uint32_t occurs[kFewZeroRows];
    const std::uint32_t n = static_cast<std::uint32_t>(a.n);
    bool bad = false;
    for (std::uint32_t i = threadIdx.x; i < n; i += 8 * kThreads) {
        std::uint32_t v[8];
        ids.rows<8>(i, kThreads, n, v, bad);
#pragma unroll
        for (std::uint32_t r = 0; r < 8; ++r)
            if (i + r * kThreads < n) rowOf[i + r * kThreads] = v[r];
    }
    if (blockIdx.x == 0) report(err, bad);
    if (blockIdx.x >= a.joinBlocks) {  // zeros in the rows that do not occur
        const std::uint64_t v0 = static_cast<std::uint64_t>(blockIdx.x - a.joinBlocks) * a.zeroRows;
        occurs[threadIdx.x] = 0;
        __syncthreads();
        for (std::uint32_t i = threadIdx.x; i < n; i += kThreads) {
            const std::uint64_t at = rowOf[i] - v0;  // past the rows for those before v0 too
            if (rowOf[i] != kNoRow && at < a.zeroRows) occurs[at] = 1;
        }
        __syncthreads();
        const std::uint32_t cols = a.D / N;
        const std::uint32_t rows = static_cast<std::uint32_t>(min<std::uint64_t>(a.zeroRows, a.V - v0));
        for (std::uint32_t i = threadIdx.x; i < rows * cols; i += kThreads) {
            const std::uint32_t r = i / cols;
            if (occurs[r] == 0)
                store_row<T, N>(static_cast<T*>(a.grad) + (v0 + r) * a.ldg + (i - r * cols) * N, vec_t<float, N>(0.0f));
        }
        return;
    }
    __syncthreads();
    constexpr std::uint32_t kWaves = kThreads / kWave;
    const std::uint32_t wave = threadIdx.x / kWave, lane = __lane_id();
    std::uint16_t* list = reinterpret_cast<std::uint16_t*>(rowOf + n) + wave * n;
    const std::uint32_t team = lane >> a.laneBits, teams = kWave >> a.laneBits;
    const std::uint32_t col = (lane & ((1u << a.laneBits) - 1u)) * N;
    const T* dOut = static_cast<const T*>(a.dOut);
    for (std::uint32_t i = blockIdx.x * kWaves + wave; i < n; i += a.joinBlocks * kWaves) {
        const std::uint32_t v = uniform(rowOf[i]);
        if (v == kNoRow) continue;
        std::uint32_t found = 0;
        bool first = true;
        for (std::uint32_t j0 = 0; j0 < n; j0 += kWave) {
            const std::uint32_t j = j0 + lane;
            const std::uint64_t same = __ballot(j < n && rowOf[min(j, n - 1)] == v);
            if (same == 0) continue;
            if (found == 0 && j0 + __builtin_ctzll(same) != i) {  // another position's
                first = false;
                break;
            }
            if (same >> lane & 1) list[found + __popcll(same & lanemask_lt())] = static_cast<std::uint16_t>(j);
            found += static_cast<std::uint32_t>(__popcll(same));
        }
        if (!first) continue;
        for (std::uint32_t c = col; c < a.D; c += N << a.laneBits) {
            vec_t<float, N> s(0.0f);
            for (std::uint32_t k = team; k < found; k += 4 * teams) {
                vec_t<T, N> x[4];
#pragma unroll
                for (std::uint32_t u = 0; u < 4; ++u)
                    x[u] = load_global<vec_t<T, N>>(dOut + list[min(k + u * teams, found - 1)] * a.ldd + c);
#pragma unroll
                for (std::uint32_t u = 0; u < 4; ++u)
                    if (k + u * teams < found) s += __builtin_convertvector(x[u], vec_t<float, N>);
            }
            for (std::uint32_t d = 1u << a.laneBits; d < kWave; d <<= 1)
#pragma unroll
                for (int q = 0; q < N; ++q) s[q] += __shfl_xor(s[q], d, kWave);
            if (team == 0) write_sum<T, N>(a, v, c, s);
        }
    }
}

// ---------------------------------------------------------------- host side

// The lanes of a team, as a power of two, for lanes of `width` elements.
unsigned team_bits(std::uint32_t D, std::uint32_t width) {
    unsigned bits = 0;
    while (bits < 6 && (width << bits) < D) ++bits;
    return bits;
}

// Rows a chunk: short ones give few rows enough teams, long ones keep the
// parts few.  12,000 rows of 32 into 70,000: the sums 12 us with chunks of 4, 19
// with 8, 32 with 16; 250,000 rows of 32 into 400,000 together 68 us with 8, 70
// with 16, 80 with 32, and 520,000 rows of 100 150, 143, 140.
std::uint32_t grad_chunk(std::uint64_t n) { return n < (1u << 15) ? 4u : n < (1u << 17) ? 8u : n < (1u << 19) ? 16u : 64u; }

unsigned id_bits(std::uint64_t V) {  // of the values 0 .. V
    unsigned b = 1;
    while (b < 64 && (V >> b) != 0) ++b;
    return b;
}

// Columns of a gradient: a window's elements are counted in 32 bits.
constexpr std::uint32_t kMaxGradCols = (1u << 28) - 1;
static_assert(kMaxGradCols <= 0xFFFFFFFFu / kWindow);

constexpr std::size_t align16(std::size_t b) { return (b + 15) & ~std::size_t(15); }

struct GradLayout {
    std::size_t keysA, keysB, hist, total, parts, mark, bytes;
    GradLayout(std::uint64_t n, std::uint64_t V, std::uint32_t D) {
        std::size_t at = 0;
        const auto take = [&at](std::size_t b) {
            const std::size_t r = at;
            at += align16(b);
            return r;
        };
        const std::uint64_t chunks = (n + grad_chunk(n) - 1) / grad_chunk(n);
        keysA = take(n * 8);
        keysB = take(n * 8);
        hist = take(partition_hist_elems(n) * 4);
        total = take(kRadixBins * 4);
        parts = take(2 * chunks * D * 4);
        mark = take((V + kWindow - 1) / kWindow + 8);
        bytes = at;
    }
};

template <typename T, int N>
int lookup_launch(const void* table, std::uint64_t ldt, const Ids& ids, std::uint64_t n, std::uint32_t D, float scale,
                  void* out, std::uint64_t ldo, std::uint32_t* err, hipStream_t st) {
    const std::uint32_t colsV = D / N;
    TCC_REQUIRE(colsV < kNoRow - kThreads * kLookupUnroll, TCC_ERR_UNSUPPORTED, "embedding rows too wide for a lookup");
    const std::uint64_t vecs = n * colsV;
    constexpr std::uint64_t kVecs = kThreads * kLookupUnroll, kMost = kVecs << 22;  // of a launch: 2^30 threads
    auto* form = n * D * sizeof(T) > kCacheBytes ? &lookup_kernel<T, N, true> : &lookup_kernel<T, N, false>;
    for (std::uint64_t from = 0; from < vecs; from += kMost) {
        const unsigned blocks = grid_for(std::min(vecs - from, kMost), kVecs);
        hipLaunchKernelGGL(form, dim3(blocks), dim3(kThreads), 0, st, static_cast<const T*>(table), ldt, ids, n, colsV, scale,
                           static_cast<T*>(out), ldo, err, from);
        TCC_LAUNCH_CHECK();
    }
    return TCC_OK;
}

template <typename T, int N>
int few_grad_launch(GradArgs a, const Ids& ids, std::uint32_t* err, hipStream_t st) {
    a.laneBits = team_bits(a.D, N);
    a.joinBlocks = grid_for(a.n, kThreads / kWave);
    a.zeroRows = static_cast<std::uint32_t>(std::clamp<std::uint64_t>(a.V / 1024, 4, kFewZeroRows));
    const unsigned zeroBlocks = a.accumulate ? 0u : grid_for(a.V, a.zeroRows);
    const std::size_t lds = a.n * (sizeof(std::uint32_t) + kThreads / kWave * sizeof(std::uint16_t));
    hipLaunchKernelGGL((few_grad_kernel<T, N>), dim3(a.joinBlocks + zeroBlocks), dim3(kThreads), lds, st, a, ids, err);
    TCC_LAUNCH_CHECK();
    return TCC_OK;
}

// Waves that the windows are spread over where there are as many (with 4,096 of
// them 2M rows of 100 take 176 us instead of 169 where nearly all are zero).
constexpr std::uint64_t kZeroWaves = 16384;

template <typename T, int N>
int grad_launch(GradArgs a, hipStream_t st) {
    a.laneBits = team_bits(a.D, N);
    const unsigned blocks = grid_for(static_cast<std::uint64_t>(a.chunks) << a.laneBits, kThreads);
    if (blocks > 0) {
        const std::uint32_t lds = (kThreads >> a.laneBits) * a.chunk * sizeof(std::uint64_t);
        hipLaunchKernelGGL((grad_kernel<T, N>), dim3(blocks), dim3(kThreads), lds, st, a);
        TCC_LAUNCH_CHECK();
    }
    a.joinBlocks = a.chunks > 1 ? blocks : 0u;
    const std::uint64_t windows = (a.V + kWindow - 1) / kWindow;
    a.waveWindows = static_cast<std::uint32_t>(std::clamp<std::uint64_t>(windows / kZeroWaves, 1, kWave));
    const unsigned zeroBlocks = a.accumulate ? 0u : grid_for(windows, a.waveWindows * (kThreads / kWave));
    if (a.joinBlocks + zeroBlocks > 0) {
        hipLaunchKernelGGL((join_kernel<T, N>), dim3(a.joinBlocks + zeroBlocks), dim3(kThreads), 0, st, a);
        TCC_LAUNCH_CHECK();
    }
    return TCC_OK;
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

int check_ids(const void* ids, std::uint32_t idBytes, std::uint64_t n, std::uint64_t V, std::uint32_t D,
              std::uint32_t dtype) {
    TCC_REQUIRE(dtype_bytes(dtype) != 0, TCC_ERR_INVALID_ARGUMENT, "embedding rows are fp32, bf16 or fp16");
    TCC_REQUIRE(idBytes == 4 || idBytes == 8, TCC_ERR_INVALID_ARGUMENT, "embedding ids are int32 or int64");
    TCC_REQUIRE(D >= 1 && (n == 0 || ids != nullptr), TCC_ERR_INVALID_ARGUMENT, "invalid embedding arguments");
    TCC_REQUIRE(n < kNoRow && V < kNoRow, TCC_ERR_UNSUPPORTED, "embedding ids and rows must be below 2^32 - 1");
    return TCC_OK;
}

}  // namespace
}  // namespace tcc

using namespace tcc;

extern "C" {

int tcc_embedding_lookup(const void* table, uint64_t ldt, uint32_t dtype, const void* ids, uint32_t idBytes, uint64_t n,
                         uint64_t V, uint32_t D, float scale, int64_t padding, void* out, uint64_t ldo,
                         uint32_t* deviceError, void* stream) {
    if (const int rc = check_ids(ids, idBytes, n, V, D, dtype)) return rc;
    TCC_REQUIRE(ldt >= D && ldo >= D && (table || V == 0) && (out || n == 0), TCC_ERR_INVALID_ARGUMENT,
                "invalid embedding lookup arguments");
    if (n == 0) return TCC_OK;
    const Ids rows{ids, V, padding, idBytes == 8};
    const std::uint32_t w = RowWidth(D, dtype_bytes(dtype)).with(table).with(out).stride(ldt).stride(ldo).elems();
#define CALL(T, N) (lookup_launch<T, N>(table, ldt, rows, n, D, scale, out, ldo, deviceError, as_stream(stream)))
    if (dtype == TCC_F32) TCC_BY_WIDTH(float, 4, w, CALL);
    if (dtype == TCC_BF16) TCC_BY_WIDTH(bf16_t, 8, w, CALL);
    TCC_BY_WIDTH(f16_t, 8, w, CALL);
#undef CALL
}

size_t tcc_embedding_grad_workspace_bytes(uint64_t n, uint64_t V, uint32_t D) { return GradLayout(n, V, D).bytes; }

int tcc_embedding_grad(const void* dOut, uint64_t ldd, uint32_t dtype, const void* ids, uint32_t idBytes, uint64_t n,
                       uint64_t V, uint32_t D, float scale, int64_t padding, void* grad, uint64_t ldg, int accumulate,
                       uint32_t* deviceError, void* workspace, size_t workspaceBytes, void* stream) {
    if (const int rc = check_ids(ids, idBytes, n, V, D, dtype)) return rc;
    TCC_REQUIRE(D <= kMaxGradCols, TCC_ERR_UNSUPPORTED, "embedding rows too wide for a gradient (2^28 - 1 elements at most)");
    const GradLayout lay(n, V, D);
    TCC_REQUIRE(ldd >= D && ldg >= D && (dOut || n == 0) && (grad || V == 0), TCC_ERR_INVALID_ARGUMENT,
                "invalid embedding gradient arguments");
    TCC_REQUIRE((workspace || lay.bytes == 0) && workspaceBytes >= lay.bytes, TCC_ERR_INVALID_ARGUMENT,
                "embedding gradient workspace too small (tcc_embedding_grad_workspace_bytes)");
    TCC_REQUIRE(reinterpret_cast<std::uintptr_t>(workspace) % 16 == 0, TCC_ERR_INVALID_ARGUMENT,
                "embedding gradient workspace must be 16-byte aligned");
    if (n == 0 && (accumulate || V == 0)) return TCC_OK;
    const hipStream_t st = as_stream(stream);
    char* ws = static_cast<char*>(workspace);
    const Ids rows{ids, V, padding, idBytes == 8};
    GradArgs a{};
    a.dOut = dOut;
    a.grad = grad;
    a.parts = reinterpret_cast<float*>(ws + lay.parts);
    a.mark = reinterpret_cast<std::uint8_t*>(ws + lay.mark);
    a.n = n;
    a.V = V;
    a.ldd = ldd;
    a.ldg = ldg;
    a.D = D;
    a.chunk = grad_chunk(n);
    a.chunks = static_cast<std::uint32_t>((n + a.chunk - 1) / a.chunk);
    a.scale = scale;
    a.accumulate = accumulate;
    const std::uint32_t w = RowWidth(D, dtype_bytes(dtype)).with(dOut).with(grad).stride(ldd).stride(ldg).elems();
    if (n > 0 && n <= kFewRows && V <= kFewTableRows) {
#define CALL(T, N) (few_grad_launch<T, N>(a, rows, deviceError, st))
        if (dtype == TCC_F32) TCC_BY_WIDTH(float, 4, w, CALL);
        if (dtype == TCC_BF16) TCC_BY_WIDTH(bf16_t, 8, w, CALL);
        TCC_BY_WIDTH(f16_t, 8, w, CALL);
#undef CALL
    }
    const std::uint64_t markWords = accumulate ? 0 : (V + 8 * kWindow - 1) / (8 * kWindow);
    std::uint64_t* const marks = reinterpret_cast<std::uint64_t*>(a.mark);
    std::uint64_t* const keys = reinterpret_cast<std::uint64_t*>(ws + lay.keysA);
    if (n > 0 && n <= kPassRows) {
        const std::uint32_t bits = id_bits(V), passes = (bits + kDigitBits - 1) / kDigitBits, digit = (bits + passes - 1) / passes;
        std::uint64_t* const other = reinterpret_cast<std::uint64_t*>(ws + lay.keysB);
        const dim3 grid(grid_for(n, kPassThreads)), block(kPassThreads);
        const std::uint32_t count = static_cast<std::uint32_t>(n);
        for (std::uint32_t p = 0; p < passes; ++p) {
            const std::uint32_t width = std::min(digit, bits - p * digit);
            std::uint64_t* const to = p % 2 == 0 ? keys : other;
            if (p == 0)
                hipLaunchKernelGGL(pass_kernel<FirstKeys>, grid, block, 0, st, FirstKeys{rows}, count, 0u, width, to, marks,
                                   markWords, deviceError);
            else
                hipLaunchKernelGGL(pass_kernel<SortedKeys>, grid, block, 0, st, SortedKeys{a.keys}, count, p * digit, width,
                                   to, marks, std::uint64_t(0), static_cast<std::uint32_t*>(nullptr));
            TCC_LAUNCH_CHECK();
            a.keys = to;
        }
    } else {
        if (n > 0) {
            std::uint64_t* sorted = nullptr;
            TCC_HIP_CHECK(partition_by(IdKeys{rows, n, deviceError}, keys,
                                       reinterpret_cast<std::uint64_t*>(ws + lay.keysB), n, 32, id_bits(V),
                                       reinterpret_cast<std::uint32_t*>(ws + lay.hist),
                                       reinterpret_cast<std::uint32_t*>(ws + lay.total), &sorted, st));
            a.keys = sorted;
        }
        TCC_HIP_CHECK(fill<std::uint64_t>(marks, markWords, 0, st));
    }
#define CALL(T, N) (grad_launch<T, N>(a, st))
    if (dtype == TCC_F32) TCC_BY_WIDTH(float, 4, w, CALL);
    if (dtype == TCC_BF16) TCC_BY_WIDTH(bf16_t, 8, w, CALL);
    TCC_BY_WIDTH(f16_t, 8, w, CALL);
#undef CALL
}

}  // extern "C"
