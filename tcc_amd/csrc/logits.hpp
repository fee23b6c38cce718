// Softmax sums over rows of logits (distill.hip, top_logits.hip).
#pragma once

#include "row_types.hpp"

namespace tcc {

constexpr float kLn2 = 0.693147181f;
constexpr float kNone = -__builtin_huge_valf();  // the logit of nothing

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_of(float x) { return __builtin_amdgcn_logf(x); }
__device__ __forceinline__ float inverse_of(float x) { return __builtin_amdgcn_rcpf(x); }
// log2(x) as a whole number and a fraction of [-1, 0): differences of two keep the
// digits that the logarithm of a large sum rounds away (v_log_f32 does so to one
// side, which the mean of many rows does not even out).
struct Log2 {
    float whole, part;
    __device__ __forceinline__ explicit Log2(float x)
        : whole(static_cast<float>(__builtin_amdgcn_frexp_expf(x))), part(log2_of(__builtin_amdgcn_frexp_mantf(x))) {}
    __device__ __forceinline__ float over(const Log2& o) const { return (whole - o.whole) + (part - o.part); }
};
// A maximum as it is subtracted: 0 for that of nothing.  OPEN: and for +inf, so that
// a sum with an infinity is infinite, and NaN only with a NaN.
template <bool OPEN = false>
__device__ __forceinline__ float base_of(float m) {
    return (OPEN ? fabsf(m) == -kNone : m == kNone) ? 0.0f : m;
}

// The maximum m of some logits and s = sum of 2^((z - m) c).
template <bool OPEN>
struct ShareOf {
    float m = kNone, s = 0.0f;
    __device__ __forceinline__ void scale_to(float top, float c) {
        s *= exp2_of((m - base_of<OPEN>(top)) * c);
        m = top;
    }
    __device__ __forceinline__ ShareOf with(ShareOf o, float c) const {
        const float top = fmaxf(m, o.m);
        const float b = base_of<OPEN>(top);
        return {top, s * exp2_of((m - b) * c) + o.s * exp2_of((o.m - b) * c)};
    }
};

// The same of a row of any length, held in 64 bits under a reference that the
// maximum passes by a factor of 2 at most: batches that are summed in 32 bits are
// added without a rounding of that size each, and a maximum that rises with every
// one does not scale (and round) the sum every time.
template <bool OPEN>
struct LongShareOf {
    float m = kNone, ref = kNone;
    double s = 0.0;
    // Takes in logits up to `top`; what is subtracted from them.
    __device__ __forceinline__ float raise(float top, float c) {
        m = fmaxf(m, top);
        if ((m - ref) * c > 1.0f) {
            s *= exp2_of((ref - base_of<OPEN>(m)) * c);
            ref = m;
        }
        return base_of<OPEN>(ref);
    }
    __device__ __forceinline__ void add(float z, float c) {
        const float b = raise(z, c);
        s += exp2_of((z - b) * c);
    }
    __device__ __forceinline__ ShareOf<OPEN> share(float c) const {
        return {m, static_cast<float>(s * exp2_of((ref - base_of<OPEN>(m)) * c))};
    }
};

// A vector of V of a row's elements; the last one is moved back to end with the
// row.
template <int V>
struct Place {
    std::uint32_t at, skip;  // first element, and how many of them are another vector's (V: all)
    // (a row has fewer than 2^31 elements, and vectors a batch past its end)
    __device__ __forceinline__ Place(std::uint32_t vector, std::uint32_t C) {
        const std::uint32_t c = vector * V, last = C - V;
        at = c < last ? c : last;
        skip = c - at < V ? c - at : V;
    }
    __device__ __forceinline__ bool any() const { return skip < V; }
};

}  // namespace tcc
