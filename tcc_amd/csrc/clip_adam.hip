// The global gradient norm over a list of tensors, clipping, and the Adam
// update that takes the clipped gradient (include/tcc_training.h).
//
// All of it is bound by memory: the norm reads every gradient once, and
// clipping (one factor for all of them) can begin only when it is known, so
// the gradients are read twice.  The Adam kernel applies the factor as it
// reads the gradient, so the clipped gradient is never written.  A list of
// tensors is one launch: its elements are cut into units that a fixed grid
// walks, and a workgroup finds a unit's tensor in the kernel's arguments.
// 245M fp32 values in one aligned run are clipped in 535 us (the norm 160); a run
// at an odd address goes element by element (726, the norm 291), and so do rows
// of a wider buffer, with a division for each (919 and 358 for 2.45M rows of 99 in
// 100).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../../include/tcc_swtcf.h"
#include "../../include/tcc_training.h"
#include "primitives.hpp"
#include "row_types.hpp"

namespace tcc {
namespace {

constexpr int kThreads = 256;
constexpr int kLaneElems = 8;                        // elements a lane takes at once
// Times that a lane does so in a unit of work: four where the units fill the GPU
// many times over, one where they would leave most of it idle.
constexpr int kManyRounds = 4, kFewRounds = 1;
template <int R>
constexpr int kUnit = kThreads * kLaneElems * R;  // elements of a unit
constexpr std::uint32_t kMaxParts = 2048;            // workgroups of the norm: 8 a CU

// An operand of a list's tensor.
struct Operand {
    void* data;
    std::uint64_t ld;
};

template <int OPS>
struct Item {
    Operand op[OPS];
    std::uint64_t cols, count, unit0;  // rows * cols elements, units from unit0
    std::uint8_t dtype[OPS];
    std::uint8_t flat;  // one run of memory in every operand, aligned to a lane's elements
};

// As many as 4 KB of kernel arguments hold, with room for the other arguments;
// a few where those do, as every launch copies them all.
template <int OPS>
constexpr int kItems = 3800 / sizeof(Item<OPS>);
constexpr int kFewItems = 8;

template <int OPS, int CAP, int R>
struct List {
    std::uint32_t count;
    std::uint64_t units;
    Item<OPS> item[CAP];
};

template <int OPS, int CAP, int R>
__device__ __forceinline__ const Item<OPS>& find_item(const List<OPS, CAP, R>& list, std::uint64_t unit) {
    std::uint32_t lo = 0, hi = list.count;
    while (hi - lo > 1) {
        const std::uint32_t m = (lo + hi) / 2;
        if (list.item[m].unit0 <= unit) lo = m;
        else hi = m;
    }
    return list.item[lo];
}

// A unit's elements as kThreads threads take them: vec(e, rounds) for 8
// elements from each of e, e + 8 * kThreads, ..., one(at) for a single element
// by its places in the operands.
template <int N>
using Rounds = std::integral_constant<int, N>;
template <int R, int OPS, typename Vec, typename One>
__device__ __forceinline__ void each_element(const Item<OPS>& it, std::uint64_t unit, std::uint32_t thread, Vec vec, One one) {
    const std::uint64_t first = (unit - it.unit0) * kUnit<R>, end = min(first + kUnit<R>, it.count);
    std::uint64_t at[OPS];
    if (it.flat) {
        const std::uint64_t e0 = first + thread * kLaneElems;
        if (end - first == kUnit<R>) {
            vec(e0, Rounds<R>{});
            return;
        }
        for (std::uint64_t e = e0; e + kLaneElems <= end; e += kThreads * kLaneElems) vec(e, Rounds<1>{});
        const std::uint64_t rest = first + (end - first) / kLaneElems * kLaneElems + thread;
        if (rest < end) {
#pragma unroll
            for (int o = 0; o < OPS; ++o) at[o] = rest;
            one(at);
        }
        return;
    }
    for (std::uint64_t e = first + thread; e < end; e += kThreads) {
#pragma unroll
        for (int o = 0; o < OPS; ++o) {
            const std::uint64_t ld = it.op[o].ld;
            at[o] = ld == it.cols ? e : e / it.cols * ld + e % it.cols;
        }
        one(at);
    }
}

using vf8 = vec_t<float, kLaneElems>;

template <typename T>
__device__ __forceinline__ float load_at(const Operand& o, std::uint64_t at) {
    return static_cast<float>(load_global<T>(static_cast<const T*>(o.data) + at));
}

__device__ __forceinline__ float load_any(const Operand& o, std::uint32_t dtype, std::uint64_t at) {
    return dtype == TCC_F32 ? load_at<float>(o, at) : dtype == TCC_BF16 ? load_at<bf16_t>(o, at) : load_at<f16_t>(o, at);
}

__device__ __forceinline__ void store_any(const Operand& o, std::uint32_t dtype, std::uint64_t at, float v) {
    if (dtype == TCC_F32) static_cast<float*>(o.data)[at] = v;
    else if (dtype == TCC_BF16) static_cast<bf16_t*>(o.data)[at] = static_cast<bf16_t>(v);
    else static_cast<f16_t*>(o.data)[at] = static_cast<f16_t>(v);
}

// ONCE: past the caches' order.
template <bool ONCE, typename V>
__device__ __forceinline__ V load_as(const void* p) {
    const auto* g = (const __attribute__((address_space(1))) V*)(reinterpret_cast<std::uintptr_t>(p));
    if constexpr (ONCE) return __builtin_nontemporal_load(g);
    else return *g;
}

template <bool ONCE = false>
__device__ __forceinline__ vf8 load8(const Operand& o, std::uint32_t dtype, std::uint64_t at) {
    if (dtype == TCC_F32) {
        const vf4 a = load_as<ONCE, vf4>(static_cast<const float*>(o.data) + at);
        const vf4 b = load_as<ONCE, vf4>(static_cast<const float*>(o.data) + at + 4);
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    if (dtype == TCC_BF16)
        return __builtin_convertvector(load_as<ONCE, vec_t<bf16_t, 8>>(static_cast<const bf16_t*>(o.data) + at), vf8);
    return __builtin_convertvector(load_as<ONCE, vec_t<f16_t, 8>>(static_cast<const f16_t*>(o.data) + at), vf8);
}

__device__ __forceinline__ void store8(const Operand& o, std::uint32_t dtype, std::uint64_t at, vf8 v) {
    if (dtype == TCC_F32) {
        vf4* p = reinterpret_cast<vf4*>(static_cast<float*>(o.data) + at);
        p[0] = __builtin_shufflevector(v, v, 0, 1, 2, 3);
        p[1] = __builtin_shufflevector(v, v, 4, 5, 6, 7);
    } else if (dtype == TCC_BF16) {
        store_row<bf16_t, 8>(static_cast<bf16_t*>(o.data) + at, v);
    } else {
        store_row<f16_t, 8>(static_cast<f16_t*>(o.data) + at, v);
    }
}

// The sum of a workgroup's values, in the same order every time.
__device__ __forceinline__ double block_sum(double v, double* shared) {
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, kWave);
    if (__lane_id() == 0) shared[threadIdx.x / kWave] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) s += shared[w];
    __syncthreads();
    return s;
}

// What the norm's kernel leaves to the next one.
struct Shared {
    double corr1, corr2;  // Adam's 1 - beta^t
    double part[kMaxParts];
};

struct StepArgs {
    std::int64_t* step;  // NULL: no step to take
    double beta1, beta2;
};

// A thread's part of the sum of squares over a list's units.
template <bool ONCE, int OPS, int CAP, int R>
__device__ __forceinline__ double squares(const List<OPS, CAP, R>& list, int op, std::uint32_t block, std::uint32_t blocks,
                                          std::uint32_t thread) {
    double s = 0.0;
    for (std::uint64_t u = block; u < list.units; u += blocks) {
        const Item<OPS>& it = find_item(list, u);
        const Operand& o = it.op[op];
        const std::uint32_t dt = it.dtype[op];
        each_element<R>(
            it, u, thread,
            [&](std::uint64_t e, auto rounds) {
                constexpr int M = decltype(rounds)::value;
                vf8 x[M];
#pragma unroll
                for (int r = 0; r < M; ++r) x[r] = load8<ONCE>(o, dt, e + r * kThreads * kLaneElems);
#pragma unroll
                for (int r = 0; r < M; ++r)
#pragma unroll
                    for (int q = 0; q < kLaneElems; ++q) {
                        const double d = x[r][q];
                        s = fma(d, d, s);
                    }
            },
            [&](const std::uint64_t(&at)[OPS]) {
                const double d = load_any(o, dt, at[op]);
                s = fma(d, d, s);
            });
    }
    return s;
}

// `add`: a list's later items, over the earlier ones' parts.
template <int CAP, int R, bool ONCE>
__global__ void __launch_bounds__(kThreads) norm_kernel(List<1, CAP, R> list, Shared* sh, int add, StepArgs st) {
    __shared__ double red[kThreads / kWave];
    const double s = block_sum(squares<ONCE>(list, 0, blockIdx.x, gridDim.x, threadIdx.x), red);
    if (threadIdx.x == 0) {
        sh->part[blockIdx.x] = add ? sh->part[blockIdx.x] + s : s;
        if (blockIdx.x == 0 && st.step != nullptr) {
            const double t = static_cast<double>(++*st.step);
            sh->corr1 = 1.0 - pow(st.beta1, t);
            sh->corr2 = 1.0 - pow(st.beta2, t);
        }
    }
}

// The norm of `parts` partial sums, the same in every workgroup.
__device__ __forceinline__ float total_norm(const Shared* sh, std::uint32_t parts, double* red) {
    double s = 0.0;
    for (std::uint32_t i = threadIdx.x; i < parts; i += kThreads) s += sh->part[i];
    return static_cast<float>(sqrt(block_sum(s, red)));
}

// NaN stays NaN.
__device__ __forceinline__ float clip_factor(float norm, float maxNorm) {
    const float c = maxNorm / (norm + 1e-6f);
    return c > 1.0f ? 1.0f : c;
}

__global__ void __launch_bounds__(kThreads) total_kernel(const Shared* sh, std::uint32_t parts, float* norm) {
    __shared__ double red[kThreads / kWave];
    const float n = total_norm(sh, parts, red);
    if (threadIdx.x == 0) *norm = n;
}

// Operands: gradient, output.
template <int CAP, int R>
__device__ __forceinline__ void scale_list(const List<2, CAP, R>& list, float c, std::uint32_t block, std::uint32_t blocks,
                                           std::uint32_t thread) {
    for (std::uint64_t u = block; u < list.units; u += blocks) {
        const Item<2>& it = find_item(list, u);
        const std::uint32_t dt = it.dtype[0];
        each_element<R>(
            it, u, thread,
            [&](std::uint64_t e, auto rounds) {
                constexpr int M = decltype(rounds)::value;
                vf8 x[M];
#pragma unroll
                for (int r = 0; r < M; ++r) x[r] = load8(it.op[0], dt, e + r * kThreads * kLaneElems);
#pragma unroll
                for (int r = 0; r < M; ++r) store8(it.op[1], dt, e + r * kThreads * kLaneElems, x[r] * c);
            },
            [&](const std::uint64_t(&at)[2]) { store_any(it.op[1], dt, at[1], load_any(it.op[0], dt, at[0]) * c); });
    }
}

template <int CAP, int R>
__global__ void __launch_bounds__(kThreads) clip_kernel(List<2, CAP, R> list, const Shared* sh, std::uint32_t parts,
                                                       float maxNorm, float* norm) {
    __shared__ double red[kThreads / kWave];
    const float n = total_norm(sh, parts, red);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = n;
    scale_list(list, clip_factor(n, maxNorm), blockIdx.x, gridDim.x, threadIdx.x);
}

struct AdamArgs {
    double lr;
    float beta1, beta2, rest1, rest2, eps, decay, keep, maxNorm;  // keep: 1 - lr * weightDecay, or 1
};

struct AdamFactors {
    float clip, size, root2;  // lr / corr1, sqrt(corr2)
    __device__ __forceinline__ AdamFactors(const AdamArgs& a, float c, double corr1, double corr2)
        : clip(c), size(static_cast<float>(a.lr / corr1)), root2(static_cast<float>(sqrt(corr2))) {}
};

__device__ __forceinline__ void adam_one(float& p, float g, float& m, float& v, const AdamArgs& a,
                                         const AdamFactors& f) {
    g *= f.clip;
    if (a.decay != 0.0f) g += a.decay * p;  // without decay an infinite parameter is none of the moments'
    m = a.beta1 * m + a.rest1 * g;
    v = a.beta2 * v + a.rest2 * g * g;
    p = a.keep * p - f.size * (m / (sqrtf(v) / f.root2 + a.eps));
}

// Operands: parameter, gradient, first and second moment (both fp32).
template <int CAP, int R>
__device__ __forceinline__ void adam_list(const List<4, CAP, R>& list, const AdamArgs& a, const AdamFactors& f,
                                          std::uint32_t block, std::uint32_t blocks, std::uint32_t thread) {
    for (std::uint64_t u = block; u < list.units; u += blocks) {
        const Item<4>& it = find_item(list, u);
        const std::uint32_t dp = it.dtype[0], dg = it.dtype[1];
        each_element<R>(
            it, u, thread,
            [&](std::uint64_t e0, auto rounds) {
#pragma unroll 2
                for (int r = 0; r < decltype(rounds)::value; ++r) {
                    const std::uint64_t e = e0 + r * kThreads * kLaneElems;
                    vf8 p = load8(it.op[0], dp, e), m = load8(it.op[2], TCC_F32, e), v = load8(it.op[3], TCC_F32, e);
                    const vf8 g = load8(it.op[1], dg, e);
#pragma unroll
                    for (int q = 0; q < kLaneElems; ++q) {
                        float pq = p[q], mq = m[q], vq = v[q];
                        adam_one(pq, g[q], mq, vq, a, f);
                        p[q] = pq;
                        m[q] = mq;
                        v[q] = vq;
                    }
                    store8(it.op[0], dp, e, p);
                    store8(it.op[2], TCC_F32, e, m);
                    store8(it.op[3], TCC_F32, e, v);
                }
            },
            [&](const std::uint64_t(&at)[4]) {
                float p = load_any(it.op[0], dp, at[0]), m = load_at<float>(it.op[2], at[2]),
                      v = load_at<float>(it.op[3], at[3]);
                adam_one(p, load_any(it.op[1], dg, at[1]), m, v, a, f);
                store_any(it.op[0], dp, at[0], p);
                store_any(it.op[2], TCC_F32, at[2], m);
                store_any(it.op[3], TCC_F32, at[3], v);
            });
    }
}

template <int CAP, int R>
__global__ void __launch_bounds__(kThreads) adam_kernel(List<4, CAP, R> list, const Shared* sh, std::uint32_t parts, AdamArgs a,
                                                       float* norm) {
    __shared__ double red[kThreads / kWave];
    float clip = 1.0f;
    if (parts > 0) {
        const float n = total_norm(sh, parts, red);
        if (a.maxNorm >= 0.0f) clip = clip_factor(n, a.maxNorm);
        if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = n;
    }
    adam_list(list, a, AdamFactors(a, clip, sh->corr1, sh->corr2), blockIdx.x, gridDim.x, threadIdx.x);
}

// ---------------------------------------------------------------- host side

int check_tensor(const tcc_tensor& t) {
    TCC_REQUIRE(dtype_bytes(t.dtype) != 0, TCC_ERR_INVALID_ARGUMENT, "tensors are fp32, bf16 or fp16");
    TCC_REQUIRE(t.rows == 0 || t.cols == 0 || (t.data != nullptr && t.ld >= t.cols), TCC_ERR_INVALID_ARGUMENT,
                "invalid tensor in a list");
    TCC_REQUIRE(t.cols == 0 || t.rows <= (1ull << 48) / t.cols, TCC_ERR_UNSUPPORTED, "tensor too large");
    return TCC_OK;
}

std::uint64_t units_of(const tcc_tensor& t, int unit) { return (t.rows * t.cols + unit - 1) / unit; }

// What a list holds in all.
struct Sizes {
    std::uint64_t elems = 0, bytes = 0;
    bool many;             // units of kManyRounds
    std::uint32_t parts;   // workgroups of the norm
    Sizes(const tcc_tensor* t, std::uint32_t count) {
        for (std::uint32_t i = 0; i < count; ++i) {
            elems += t[i].rows * t[i].cols;
            bytes += t[i].rows * t[i].cols * dtype_bytes(t[i].dtype);
        }
        many = elems > static_cast<std::uint64_t>(kMaxParts) * kUnit<kFewRounds>;
        std::uint64_t units = 0;
        for (std::uint32_t i = 0; i < count; ++i) units += units_of(t[i], many ? kUnit<kManyRounds> : kUnit<kFewRounds>);
        parts = grid_of(units);
    }
    static std::uint32_t grid_of(std::uint64_t units) {
        return static_cast<std::uint32_t>(std::min<std::uint64_t>(std::max<std::uint64_t>(units, 1), kMaxParts));
    }
};

// The next items from `at` on, of the lists ops[0 .. OPS).
template <int OPS, int CAP, int R>
List<OPS, CAP, R> take_items(const tcc_tensor* const (&ops)[OPS], std::uint32_t count, std::uint32_t& at) {
    List<OPS, CAP, R> list;
    list.count = 0;
    list.units = 0;
    for (; at < count && list.count < static_cast<std::uint32_t>(CAP); ++at) {
        const tcc_tensor& t = ops[0][at];
        const std::uint64_t n = t.rows * t.cols;
        if (n == 0) continue;
        Item<OPS>& it = list.item[list.count++];
        it.cols = t.cols;
        it.count = n;
        it.unit0 = list.units;
        it.flat = 1;
        for (int o = 0; o < OPS; ++o) {
            const tcc_tensor& x = ops[o][at];
            it.op[o] = Operand{x.data, t.rows == 1 ? t.cols : x.ld};
            it.dtype[o] = static_cast<std::uint8_t>(x.dtype);
            const std::uint64_t lane = std::min<std::uint64_t>(16, kLaneElems * dtype_bytes(x.dtype));
            if (it.op[o].ld != t.cols || reinterpret_cast<std::uintptr_t>(x.data) % lane != 0) it.flat = 0;
        }
        list.units += units_of(t, kUnit<R>);
    }
    return list;
}

// Calls f(list, first) for as many lists as hold the tensors, with short
// lists where they are few.
template <int R, int OPS, typename F>
int each_list_of(const tcc_tensor* const (&ops)[OPS], std::uint32_t count, F f) {
    std::uint32_t at = 0;
    if (count <= kFewItems) return f(take_items<OPS, kFewItems, R>(ops, count, at), true);
    bool first = true;
    do {
        if (const int rc = f(take_items<OPS, kItems<OPS>, R>(ops, count, at), first)) return rc;
        first = false;
    } while (at < count);
    return TCC_OK;
}
template <int OPS, typename F>
int each_list(const Sizes& z, const tcc_tensor* const (&ops)[OPS], std::uint32_t count, F f) {
    return z.many ? each_list_of<kManyRounds>(ops, count, f) : each_list_of<kFewRounds>(ops, count, f);
}

template <int CAP, int R>
auto* norm_form(const List<1, CAP, R>&, bool once) {
    return once ? &norm_kernel<CAP, R, true> : &norm_kernel<CAP, R, false>;
}
template <int CAP, int R>
auto* clip_form(const List<2, CAP, R>&) {
    return &clip_kernel<CAP, R>;
}
template <int CAP, int R>
auto* adam_form(const List<4, CAP, R>&) {
    return &adam_kernel<CAP, R>;
}

// Gradients larger than the caches are read past their order: 245M fp32 values
// 160 us instead of 210, while those that fit are there for the next kernel.
int norm_launches(const Sizes& z, const tcc_tensor* grads, std::uint32_t count, Shared* sh, StepArgs step, hipStream_t st) {
    const tcc_tensor* const ops[1] = {grads};
    return each_list(z, ops, count, [&](const auto& list, bool first) {
        hipLaunchKernelGGL(norm_form(list, z.bytes > kCacheBytes), dim3(z.parts), dim3(kThreads), 0, st, list, sh,
                           first ? 0 : 1, first ? step : StepArgs{});
        TCC_LAUNCH_CHECK();
        return TCC_OK;
    });
}

int check_workspace(const void* ws, std::size_t bytes) {
    TCC_REQUIRE(ws != nullptr && bytes >= sizeof(Shared) && reinterpret_cast<std::uintptr_t>(ws) % 16 == 0,
                TCC_ERR_INVALID_ARGUMENT, "gradient norm workspace too small or unaligned (tcc_grad_norm_workspace_bytes)");
    return TCC_OK;
}

int check_list(const tcc_tensor* t, std::uint32_t count) {
    TCC_REQUIRE(count == 0 || t != nullptr, TCC_ERR_INVALID_ARGUMENT, "a tensor list is missing");
    for (std::uint32_t i = 0; i < count; ++i)
        if (const int rc = check_tensor(t[i])) return rc;
    return TCC_OK;
}

int check_same(const tcc_tensor* a, const tcc_tensor* b, std::uint32_t count) {
    for (std::uint32_t i = 0; i < count; ++i)
        TCC_REQUIRE(a[i].rows == b[i].rows && a[i].cols == b[i].cols, TCC_ERR_INVALID_ARGUMENT,
                    "tensors of two lists differ in shape");
    return TCC_OK;
}

}  // namespace
}  // namespace tcc

using namespace tcc;

extern "C" {

size_t tcc_grad_norm_workspace_bytes(void) { return sizeof(Shared); }

int tcc_grad_norm(const tcc_tensor* grads, uint32_t count, float* norm, void* workspace, size_t workspaceBytes,
                  void* stream) {
    if (const int rc = check_list(grads, count)) return rc;
    if (const int rc = check_workspace(workspace, workspaceBytes)) return rc;
    TCC_REQUIRE(norm, TCC_ERR_INVALID_ARGUMENT, "gradient norm: no place for the norm");
    Shared* sh = static_cast<Shared*>(workspace);
    const Sizes z(grads, count);
    const hipStream_t st = as_stream(stream);
    if (const int rc = norm_launches(z, grads, count, sh, StepArgs{}, st)) return rc;
    hipLaunchKernelGGL(total_kernel, dim3(1), dim3(kThreads), 0, st, sh, z.parts, norm);
    TCC_LAUNCH_CHECK();
    return TCC_OK;
}

int tcc_clip_grad_norm(const tcc_tensor* grads, const tcc_tensor* out, uint32_t count, float maxNorm, float* norm,
                       void* workspace, size_t workspaceBytes, void* stream) {
    for (const tcc_tensor* t : {grads, out})
        if (const int rc = check_list(t, count)) return rc;
    if (const int rc = check_same(grads, out, count)) return rc;
    for (std::uint32_t i = 0; i < count; ++i)
        TCC_REQUIRE(grads[i].dtype == out[i].dtype, TCC_ERR_INVALID_ARGUMENT, "clipped gradients keep their type");
    if (const int rc = check_workspace(workspace, workspaceBytes)) return rc;
    TCC_REQUIRE(maxNorm >= 0.0f, TCC_ERR_INVALID_ARGUMENT, "the largest norm is not negative");
    TCC_REQUIRE(norm, TCC_ERR_INVALID_ARGUMENT, "gradient norm: no place for the norm");
    Shared* sh = static_cast<Shared*>(workspace);
    const hipStream_t st = as_stream(stream);
    const tcc_tensor* const ops[2] = {grads, out};
    const Sizes z(grads, count);
    if (const int rc = norm_launches(z, grads, count, sh, StepArgs{}, st)) return rc;
    return each_list(z, ops, count, [&](const auto& list, bool) {
        hipLaunchKernelGGL(clip_form(list), dim3(Sizes::grid_of(list.units)), dim3(kThreads), 0, st, list, sh, z.parts,
                           maxNorm, norm);
        TCC_LAUNCH_CHECK();
        return TCC_OK;
    });
}

int tcc_adam_step(const tcc_tensor* params, const tcc_tensor* grads, const tcc_tensor* expAvg,
                  const tcc_tensor* expAvgSq, uint32_t count, const tcc_adam* a, int64_t* step, float* norm,
                  void* workspace, size_t workspaceBytes, void* stream) {
    TCC_REQUIRE(a && step, TCC_ERR_INVALID_ARGUMENT, "invalid Adam arguments");
    TCC_REQUIRE(a->beta1 >= 0 && a->beta1 < 1 && a->beta2 >= 0 && a->beta2 < 1 && a->eps >= 0, TCC_ERR_INVALID_ARGUMENT,
                "Adam's betas are in [0, 1) and eps is not negative");
    for (const tcc_tensor* t : {params, grads, expAvg, expAvgSq})
        if (const int rc = check_list(t, count)) return rc;
    for (const tcc_tensor* t : {grads, expAvg, expAvgSq})
        if (const int rc = check_same(params, t, count)) return rc;
    for (const tcc_tensor* t : {expAvg, expAvgSq})
        for (std::uint32_t i = 0; i < count; ++i)
            TCC_REQUIRE(t[i].dtype == TCC_F32, TCC_ERR_INVALID_ARGUMENT, "Adam's moments are fp32");
    if (const int rc = check_workspace(workspace, workspaceBytes)) return rc;
    Shared* sh = static_cast<Shared*>(workspace);
    const hipStream_t st = as_stream(stream);
    AdamArgs k{};
    k.lr = a->lr;
    k.beta1 = static_cast<float>(a->beta1);
    k.beta2 = static_cast<float>(a->beta2);
    k.rest1 = static_cast<float>(1.0 - a->beta1);
    k.rest2 = static_cast<float>(1.0 - a->beta2);
    k.eps = static_cast<float>(a->eps);
    k.decay = a->decoupled ? 0.0f : static_cast<float>(a->weightDecay);
    k.keep = a->decoupled ? static_cast<float>(1.0 - a->lr * a->weightDecay) : 1.0f;
    k.maxNorm = static_cast<float>(a->maxNorm);
    const tcc_tensor* const ops[4] = {params, grads, expAvg, expAvgSq};
    const StepArgs next{step, a->beta1, a->beta2};
    const bool wantNorm = norm != nullptr || a->maxNorm >= 0;
    const Sizes z(grads, count);
    if (const int rc = norm_launches(z, grads, wantNorm ? count : 0, sh, next, st)) return rc;
    return each_list(z, ops, count, [&](const auto& list, bool) {
        hipLaunchKernelGGL(adam_form(list), dim3(Sizes::grid_of(list.units)), dim3(kThreads), 0, st, list, sh,
                           wantNorm ? z.parts : 0u, k, norm);
        TCC_LAUNCH_CHECK();
        return TCC_OK;
    });
}

}  // extern "C"
