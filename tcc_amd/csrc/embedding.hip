// Rows of an embedding table and their gradient (include/tcc_training.h).
//
//   lookup:   out[i]  = scale * table[ids[i]]
//   gradient: grad[v] = scale * sum over {i : ids[i] = v} of dOut[i]
//
// Both move bytes and compute next to nothing.  The gradient sorts the ids
// with their positions (stable, so that a row's terms have one order and the
// sums the same bits every time), then walks the sorted positions in chunks
// of equal length, whatever the ids' frequencies: a hub node with thousands
// of rows is spread over as many chunks as it needs, and its parts are joined
// afterwards in chunk order.
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
        const std::int64_t id = wide ? load_global<std::int64_t>(static_cast<const std::int64_t*>(p) + i)
                                     : load_global<std::int32_t>(static_cast<const std::int32_t*>(p) + i);
        if (static_cast<std::uint64_t>(id) >= V) {
            bad = true;
            return kNoRow;
        }
        return id == padding ? kNoRow : static_cast<std::uint32_t>(id);
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
template <typename T, int N>
__global__ void __launch_bounds__(kThreads) lookup_kernel(const T* __restrict__ table, std::uint64_t ldt, Ids ids,
                                                         std::uint64_t n, std::uint32_t colsV, float scale,
                                                         T* __restrict__ out, std::uint64_t ldo, bool once, std::uint32_t* err) {
    const std::uint64_t first = static_cast<std::uint64_t>(blockIdx.x) * (kThreads * kLookupUnroll);
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
        if (i[u] < n) write_out<T, N>(once, out + i[u] * ldo + c[u], x[u]);
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
        const std::uint64_t last = n - 1;
#pragma unroll
        for (int r = 0; r < kPrimRounds; ++r) {
            const std::uint64_t i = min(first + static_cast<std::uint64_t>(r) * kWave, last);
            const std::uint32_t v = ids.row(i, bad);
            k[r] = (v == kNoRow ? ids.V : static_cast<std::uint64_t>(v)) << 32 | i;
        }
    }
    __device__ __forceinline__ void report(bool bad) const { tcc::report(err, bad); }
};

// Marks the rows that occur, from the sorted keys: neighbours in memory (from
// the ids as they come, 2.45M of them took 16 us instead of TODO).
__global__ void __launch_bounds__(kThreads) mark_kernel(const std::uint64_t* __restrict__ keys, std::uint64_t n,
                                                       std::uint64_t V, std::uint8_t* __restrict__ mark) {
    const std::uint64_t i = static_cast<std::uint64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= n) return;
    const std::uint32_t v = static_cast<std::uint32_t>(keys[i] >> 32);
    if (v < V && (i == 0 || static_cast<std::uint32_t>(keys[i - 1] >> 32) != v)) mark[v] = 1;
}

struct GradArgs {
    const std::uint64_t* keys;  // sorted
    const void* dOut;
    void* grad;
    float* parts;  // [2 * chunks][D]: sums of a chunk's first row (begun before it) and last row (going on after it)
    const std::uint8_t* mark;
    std::uint64_t n, V, ldd, ldg;
    std::uint32_t D, chunk, chunks, laneBits, sumBlocks;
    float scale;
    int accumulate;
    bool once;  // the gradient is too large for the caches
};

__device__ __forceinline__ std::uint32_t key_row(std::uint64_t k) { return static_cast<std::uint32_t>(k >> 32); }

template <typename T, int N>
__device__ __forceinline__ void write_sum(const GradArgs& a, std::uint32_t v, std::uint32_t c, vec_t<float, N> s) {
    T* p = static_cast<T*>(a.grad) + v * a.ldg + c;
    s *= a.scale;
    if (a.accumulate) s += load_row<T, N>(p);
    write_out<T, N>(a.once, p, s);
}

constexpr int kGradUnroll = 4;  // rows a lane has in flight: with 8, half the waves fit and 2.45M x 100 take 585 us, not TODO

// Blocks below sumBlocks: a team of 2^laneBits lanes sums one chunk of the
// sorted rows, the block's keys in LDS.  The others write zeros to the rows
// that do not occur.
template <typename T, int N>
__global__ void __launch_bounds__(kThreads) grad_kernel(GradArgs a) {
    extern __shared__ std::uint64_t ldsKeys[];
    if (blockIdx.x >= a.sumBlocks) {
        const std::uint64_t w = static_cast<std::uint64_t>(blockIdx.x - a.sumBlocks) * (kThreads / kWave) +
                                threadIdx.x / kWave;
        const std::uint32_t lane = __lane_id();
        const std::uint64_t v0 = w * kWave;
        if (v0 >= a.V) return;
        std::uint64_t absent = __ballot(v0 + lane < a.V && a.mark[min(v0 + lane, a.V - 1)] == 0);
        while (absent != 0) {
            const std::uint32_t r = static_cast<std::uint32_t>(__builtin_ctzll(absent));
            absent &= absent - 1;
            T* p = static_cast<T*>(a.grad) + (v0 + r) * a.ldg;
            for (std::uint32_t c = lane * N; c < a.D; c += kWave * N) write_out<T, N>(a.once, p + c, vec_t<float, N>(0.0f));
        }
        return;
    }
    const std::uint32_t teams = kThreads >> a.laneBits;
    const std::uint64_t base = static_cast<std::uint64_t>(blockIdx.x) * teams * a.chunk;
    const std::uint32_t here = static_cast<std::uint32_t>(min(a.n - base, static_cast<std::uint64_t>(teams * a.chunk)));
    for (std::uint32_t i = threadIdx.x; i < here; i += kThreads) ldsKeys[i] = a.keys[base + i];
    const std::uint32_t none = static_cast<std::uint32_t>(a.V);
    const std::uint32_t blockBefore = base > 0 ? key_row(a.keys[base - 1]) : none;
    const std::uint32_t blockAfter = base + here < a.n ? key_row(a.keys[base + here]) : none;
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
        std::uint32_t cur = none;
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
                if (cur != none) {
                    if (head) *reinterpret_cast<vec_t<float, N>*>(headPart + c) = s;
                    else write_sum<T, N>(a, cur, c, s);
                }
                head = i + u == lo && v[u] == before;
                cur = v[u];
                s = f;
            }
        }
        if (cur == none) continue;
        if (head) *reinterpret_cast<vec_t<float, N>*>(headPart + c) = s;
        else if (cur == after) *reinterpret_cast<vec_t<float, N>*>(headPart + a.D + c) = s;
        else write_sum<T, N>(a, cur, c, s);
    }
}

// Adds the parts of the rows that go on after the chunk they begin in, a team
// for each such chunk; a row of many parts (a hub's) is added by the whole
// workgroup, each of its teams taking every so many-th part.
constexpr std::uint32_t kLongRow = 16;
template <typename T, int N>
__global__ void __launch_bounds__(kThreads) join_kernel(GradArgs a) {
    __shared__ std::uint32_t rowOf[kThreads], partsOf[kThreads];
    __shared__ float sums[kThreads * N];
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
            std::uint64_t l = hi, h = a.n;  // the first key past the row
            while (l < h) {
                const std::uint64_t m = (l + h) / 2;
                if (key_row(a.keys[m]) <= v) l = m + 1;
                else h = m;
            }
            count = static_cast<std::uint32_t>((l - 1) / a.chunk) - team;
        }
    }
    if (lane == 0) {
        rowOf[mine] = v;
        partsOf[mine] = count;
    }
    const auto part = [&](std::uint64_t k, std::uint32_t c) {
        return load_global<vec_t<float, N>>(a.parts + k * a.D + c);
    };
    if (v != none && count <= kLongRow) {
        for (std::uint32_t c = lane * N; c < a.D; c += N << a.laneBits) {
            vec_t<float, N> s = part(2ull * team + 1, c);
            for (std::uint32_t k = 1; k <= count; ++k) s += part(2ull * (team + k), c);
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
#pragma unroll 4
                for (std::uint32_t k = 1 + mine; k <= many; k += teams) s += part(2ull * (first + t + k), c);
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

// The lanes of a team, as a power of two, for lanes of `width` elements.
unsigned team_bits(std::uint32_t D, std::uint32_t width) {
    unsigned bits = 0;
    while (bits < 6 && (width << bits) < D) ++bits;
    return bits;
}

// Rows a chunk: short ones give few rows enough teams, long ones keep the
// parts few.
std::uint32_t grad_chunk(std::uint64_t n) { return n < (1u << 16) ? 16u : n < (1u << 19) ? 32u : 64u; }

unsigned id_bits(std::uint64_t V) {  // of the values 0 .. V
    unsigned b = 1;
    while (b < 64 && (V >> b) != 0) ++b;
    return b;
}

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
        mark = take(V);
        bytes = at;
    }
};

template <typename T, int N>
int lookup_launch(const void* table, std::uint64_t ldt, const Ids& ids, std::uint64_t n, std::uint32_t D, float scale,
                  void* out, std::uint64_t ldo, std::uint32_t* err, hipStream_t st) {
    const std::uint32_t colsV = D / N;
    const std::uint64_t vecs = n * colsV;
    const std::uint64_t blocks = (vecs + kThreads * kLookupUnroll - 1) / (kThreads * kLookupUnroll);
    TCC_REQUIRE(blocks < (1ull << 31), TCC_ERR_UNSUPPORTED, "embedding lookup output too large for one call");
    hipLaunchKernelGGL((lookup_kernel<T, N>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, st,
                       static_cast<const T*>(table), ldt, ids, n, colsV, scale, static_cast<T*>(out), ldo,
                       n * D * sizeof(T) > kCacheBytes, err);
    TCC_LAUNCH_CHECK();
    return TCC_OK;
}

template <typename T, int N>
int grad_launch(GradArgs a, hipStream_t st) {
    a.laneBits = team_bits(a.D, N);
    a.once = a.V * a.D * sizeof(T) > kCacheBytes;
    a.sumBlocks = grid_for(static_cast<std::uint64_t>(a.chunks) << a.laneBits, kThreads);
    const std::uint32_t lds = (kThreads >> a.laneBits) * a.chunk * sizeof(std::uint64_t);
    const unsigned fillBlocks = a.accumulate ? 0u : grid_for(a.V, kThreads);
    if (a.sumBlocks + fillBlocks > 0)
        hipLaunchKernelGGL((grad_kernel<T, N>), dim3(a.sumBlocks + fillBlocks), dim3(kThreads), lds, st, a);
    TCC_LAUNCH_CHECK();
    if (a.chunks > 1) {
        hipLaunchKernelGGL((join_kernel<T, N>), dim3(a.sumBlocks), dim3(kThreads), 0, st, a);
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
    if (n > 0) {
        std::uint64_t* sorted = nullptr;
        TCC_HIP_CHECK(partition_by(IdKeys{rows, n, deviceError}, reinterpret_cast<std::uint64_t*>(ws + lay.keysA),
                                   reinterpret_cast<std::uint64_t*>(ws + lay.keysB), n, 32, id_bits(V),
                                   reinterpret_cast<std::uint32_t*>(ws + lay.hist),
                                   reinterpret_cast<std::uint32_t*>(ws + lay.total), &sorted, st));
        a.keys = sorted;
    }
    std::uint8_t* mark = reinterpret_cast<std::uint8_t*>(ws + lay.mark);
    if (!accumulate) {
        TCC_HIP_CHECK(fill<std::uint8_t>(mark, V, 0, st));
        if (n > 0)
            hipLaunchKernelGGL(mark_kernel, dim3(grid_for(n, kThreads)), dim3(kThreads), 0, st, a.keys, n, V, mark);
        TCC_LAUNCH_CHECK();
    }
    a.dOut = dOut;
    a.grad = grad;
    a.parts = reinterpret_cast<float*>(ws + lay.parts);
    a.mark = mark;
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
#define CALL(T, N) (grad_launch<T, N>(a, st))
    if (dtype == TCC_F32) TCC_BY_WIDTH(float, 4, w, CALL);
    if (dtype == TCC_BF16) TCC_BY_WIDTH(bf16_t, 8, w, CALL);
    TCC_BY_WIDTH(f16_t, 8, w, CALL);
#undef CALL
}

}  // extern "C"
