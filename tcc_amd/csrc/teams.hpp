// Sums, maxima and the like over a team of lanes: a power of two of them in a
// wave, or several waves that are a whole workgroup.
#pragma once

#include "common.hpp"

namespace tcc {

// v of the lane whose number differs in bit D (16 or 32).
template <int D>
__device__ __forceinline__ std::uint32_t swapped(std::uint32_t v) {
    static_assert(D == 16 || D == 32);
    if constexpr (D == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return (__lane_id() & 16) ? r[0] : r[1];
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return (__lane_id() & 32) ? r[0] : r[1];
    }
}

// v of the lane whose number differs in bit D, whatever its neighbours hold.
template <int D>
__device__ __forceinline__ std::uint32_t other(std::uint32_t v) {
    const int i = static_cast<int>(v);
    if constexpr (D == 1) return __builtin_amdgcn_update_dpp(i, i, 0xB1, 0xF, 0xF, false);  // quad_perm [1,0,3,2]
    if constexpr (D == 2) return __builtin_amdgcn_update_dpp(i, i, 0x4E, 0xF, 0xF, false);  // quad_perm [2,3,0,1]
    if constexpr (D == 4) {  // row_half_mirror, then quad_perm [3,2,1,0]: 7 - i, then ^ 3
        const int h = __builtin_amdgcn_update_dpp(i, i, 0x141, 0xF, 0xF, false);
        return __builtin_amdgcn_update_dpp(h, h, 0x1B, 0xF, 0xF, false);
    }
    if constexpr (D == 8) return __builtin_amdgcn_update_dpp(i, i, 0x128, 0xF, 0xF, false);  // row_ror:8
    if constexpr (D >= 16) return swapped<D>(v);
}
template <int D>
__device__ __forceinline__ std::uint64_t other(std::uint64_t v) {
    const std::uint64_t lo = other<D>(static_cast<std::uint32_t>(v)), hi = other<D>(static_cast<std::uint32_t>(v >> 32));
    return hi << 32 | lo;
}

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
    if constexpr (D >= 16) return swapped<D>(v);
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
struct Smaller {
    __device__ __forceinline__ float operator()(float a, float b) const { return fminf(a, b); }
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
