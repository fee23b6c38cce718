// The weights, biases and activations of the norms (group_norm.hip,
// layer_norm.hip) and their derivatives, in fp32.
#pragma once

#include "../../include/tcc_training.h"
#include "row_types.hpp"

namespace tcc {

// Channels c .. c + N of a weight or bias: one branch and one load for all of
// them (a branch for each put every load behind the one before).  The caller's
// array need only be aligned to its elements, and c is any channel.
template <int N>
__device__ __forceinline__ vec_t<float, N> load_params(const void* p, std::uint32_t type, std::uint32_t c, float none) {
    vec_t<float, N> v(none);
    if (p == nullptr) return v;
    if (type == TCC_F32) {
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] = load_global<float>(static_cast<const float*>(p) + c + q);
    } else if (type == TCC_BF16) {
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] = static_cast<float>(load_global<bf16_t>(static_cast<const bf16_t*>(p) + c + q));
    } else {
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] = static_cast<float>(load_global<f16_t>(static_cast<const f16_t*>(p) + c + q));
    }
    return v;
}

// z with a rounding after each operation, in the forward as in the gradient.
__device__ __forceinline__ float normalise(float x, float mean, float rstd) {
#pragma clang fp contract(off)
    return (x - mean) * rstd;
}
__device__ __forceinline__ float affine(float xh, float w, float b) {
#pragma clang fp contract(off)
    const float m = xh * w;
    return m + b;
}

// exp, and 1 / x, by the hardware's instructions.
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }
__device__ __forceinline__ float fast_rcp(float x) { return __builtin_amdgcn_rcpf(x); }

// FINE, below: for rows of fp32, whose results are as close to the exact ones as
// a plain evaluation in 32 bits comes.  For 16-bit rows a few 2^-24 are lost in
// the rounding of the output, and the instructions are saved.

// Phi(z) of the normal distribution, and e = exp(-z^2 / 2), from which its tail
// comes.
//  16 bits: erf by Abramowitz and Stegun's 7.1.26, off by 1.5e-7 at most, with
//    z scaled once for both (v^2 log 2 = z^2 / 2) and the halves in the
//    coefficients.
//  FINE: the tail as e t q(t), t = 1 / (1 + 0.375 |z|), and 1/2 + z r(z^2) where
//    the roundings of e, t and q would be those of values near 1/2; q and r are
//    minimax fits of Phi(-|z|) / (e t) and (Phi(z) - 1/2) / z, off by 1.6e-8 and
//    1.4e-8 in Phi.  600,000 x 256 fp32 rows, gradient: 583 us instead of 532.
// The library's erff and expf cost the gradient twice the instructions.
template <bool FINE>
__device__ __forceinline__ float normal_cdf(float z, float& e) {
    if (FINE) {
        const float u = z * z;
        e = __builtin_amdgcn_exp2f(u * -0.721347520f);  // log2(e) / 2
        const float t = fast_rcp(fmaf(0.375f, fabsf(z), 1.0f));
        float q = fmaf(t, -0.0984848365f, 0.217022926f);
        q = fmaf(t, q, 0.0710222051f);
        q = fmaf(t, q, 0.161572173f);
        q = fmaf(t, q, 0.148667201f);
        q = q * (t * e);
        float r = fmaf(u, 8.99027509e-05f, -0.00115990336f);
        r = fmaf(u, r, 0.00996036921f);
        r = fmaf(u, r, -0.0664877668f);
        r = fmaf(u, r, 0.398942143f);
        return fabsf(z) < 1.0625f ? fmaf(z, r, 0.5f) : z > 0.0f ? 1.0f - q : q;
    }
    const float v = z * 0.849321800f;                              // sqrt(log2(e) / 2)
    const float t = fast_rcp(fmaf(0.272737481f, fabsf(v), 1.0f));  // 0.3275911 sqrt(log 2)
    e = __builtin_amdgcn_exp2f(-v * v);
    float q = fmaf(t, 0.5307027145f, -0.7265760135f);
    q = fmaf(t, q, 0.7107068705f);
    q = fmaf(t, q, -0.142248368f);
    q = fmaf(t, q, 0.127414796f);
    q = q * (t * e);
    return z > 0.0f ? 1.0f - q : q;
}

// p = 1 / (1 + exp(-z)) and 1 - p of rows of fp32, each to its own last digits.
__device__ __forceinline__ float fine_sigmoid(float z, float& rest) {
    const float e = fast_exp(-fabsf(z)), d = 1.0f + e, r0 = fast_rcp(d);
    const float r = fmaf(r0, fmaf(-d, r0, 1.0f), r0);  // a Newton step
    const float s = e * r;
    rest = z > 0.0f ? s : r;
    return z > 0.0f ? r : s;
}

template <std::uint32_t ACT, bool FINE>
__device__ __forceinline__ float activate(float z) {
    if (ACT == TCC_ACT_NONE) return z;
    if (ACT == TCC_ACT_RELU) return z <= 0.0f ? 0.0f : z;  // keeps NaN
    float e;
    if (ACT == TCC_ACT_SILU) return z * (FINE ? fine_sigmoid(z, e) : fast_rcp(1.0f + fast_exp(-z)));
    return z * normal_cdf<FINE>(z, e);
}

// d act'(z).  What relu masks is 0 whatever it is, an infinity too.
template <std::uint32_t ACT, bool FINE>
__device__ __forceinline__ float through(float d, float z) {
    if (ACT == TCC_ACT_NONE) return d;
    if (ACT == TCC_ACT_RELU) return z <= 0.0f ? 0.0f : d;
    float e;
    if (ACT == TCC_ACT_SILU) {
        if (FINE) {
            const float p = fine_sigmoid(z, e);
            return d * fmaf(z * p, e, p);
        }
        const float p = fast_rcp(1.0f + fast_exp(-z));
        return d * (p * fmaf(z, 1.0f - p, 1.0f));
    }
    const float p = normal_cdf<FINE>(z, e);
    return d * fmaf(z * 0.39894228f, e, p);
}
template <typename T>
constexpr bool kFine = sizeof(T) == 4;

}  // namespace tcc
