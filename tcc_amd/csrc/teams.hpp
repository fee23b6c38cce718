// Sums, maxima and the like over a team of lanes: a power of two of them in a
// wave, or several waves that are a whole workgroup.
#pragma once

#include "common.hpp"

namespace tcc {

// v of the lane at distance D (1 to 32, a power of two) by exclusive or,
// provided that v is already the same within aligned groups of D lanes: lanes
// are mirrored then instead of exchanged, which costs one instruction without
// a trip through LDS.
template <int D>
__device__ __forceinline__ std::uint32_t across(std::uint32_t v) {
    static_assert(D == 1 || D == 2 || D == 4 || D == 8 || D == 16 || D == 32);
    const int i = static_cast<int>(v);
    if constexpr (D == 1) return __builtin_amdgcn_update_dpp(i, i, 0xB1, 0xF, 0xF, false);   // quad_perm [1,0,3,2]
    if constexpr (D == 2) return __builtin_amdgcn_update_dpp(i, i, 0x4E, 0xF, 0xF, false);   // quad_perm [2,3,0,1]
    if constexpr (D == 4) return __builtin_amdgcn_update_dpp(i, i, 0x141, 0xF, 0xF, false);  // row_half_mirror
    if constexpr (D == 8) return __builtin_amdgcn_update_dpp(i, i, 0x140, 0xF, 0xF, false);  // row_mirror
    if constexpr (D >= 16) return static_cast<std::uint32_t>(__shfl_xor(i, D, kWave));
}
template <int D>
__device__ __forceinline__ float across(float v) { return __uint_as_float(across<D>(__float_as_uint(v))); }

template <int D>
__device__ __forceinline__ double across(double v) {
    const std::uint64_t b = static_cast<std::uint64_t>(__double_as_longlong(v));
    const std::uint64_t lo = across<D>(static_cast<std::uint32_t>(b)), hi = across<D>(static_cast<std::uint32_t>(b >> 32));
    return __longlong_as_double(static_cast<long long>(hi << 32 | lo));
}

// f(v, v of the other half) from groups of 1 lane to TEAM lanes of a wave: the
// same value in all of them.
template <int TEAM, int D = 1, typename V, typename F>
__device__ __forceinline__ V wave_join(V v, F f) {
    if constexpr (D < TEAM) return wave_join<TEAM, 2 * D>(f(v, across<D>(v)), f);
    else return v;
}

struct Add {
    template <typename V>
    __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
};
struct Larger {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};

// Sums over a team of TEAM lanes, in 64 bits or two in 32.  Teams of more than a
// wave are the whole workgroup, and every thread of it calls; the places in LDS
// alternate, so that one barrier a call is enough.
template <int TEAM>
struct TeamSum {
    static constexpr int waves = TEAM > kWave ? TEAM / kWave : 1;
    union Place {
        float2 two;
        double one;
    };
    struct Shared {
        Place part[2][waves];
    };
    Shared& s;
    int turn = 0;
    __device__ __forceinline__ explicit TeamSum(Shared& shared) : s(shared) {}

    __device__ __forceinline__ double operator()(double v) {
        v = wave_join<(TEAM < kWave ? TEAM : kWave)>(v, Add());
        if constexpr (TEAM > kWave) {
            if (__lane_id() == 0) s.part[turn][threadIdx.x / kWave].one = v;
            __syncthreads();
            v = wave_join<waves>(s.part[turn][__lane_id() % waves].one, Add());
            turn ^= 1;
        }
        return v;
    }
    __device__ __forceinline__ float2 operator()(float a, float b) {
        a = wave_join<(TEAM < kWave ? TEAM : kWave)>(a, Add());
        b = wave_join<(TEAM < kWave ? TEAM : kWave)>(b, Add());
        if constexpr (TEAM > kWave) {
            if (__lane_id() == 0) s.part[turn][threadIdx.x / kWave].two = make_float2(a, b);
            __syncthreads();
            const float2 v = s.part[turn][__lane_id() % waves].two;
            a = wave_join<waves>(v.x, Add());
            b = wave_join<waves>(v.y, Add());
            turn ^= 1;
        }
        return make_float2(a, b);
    }
};

}  // namespace tcc
