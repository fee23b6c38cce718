// Rows of fp32, bf16 or fp16 elements read and written a few elements a lane,
// computed in fp32 (the kernels of include/tcc_training.h).
#pragma once

#include "common.hpp"

namespace tcc {

using bf16_t = __bf16;
using f16_t = _Float16;

template <typename T, int N>
using vec_t = T __attribute__((ext_vector_type(N)));

// N consecutive elements, aligned to N elements, as fp32.
template <typename T, int N>
__device__ __forceinline__ vec_t<float, N> load_row(const T* p) {
    return __builtin_convertvector(load_global<vec_t<T, N>>(p), vec_t<float, N>);
}

// fp32 values rounded once to T (nearest even).
template <typename T, int N>
__device__ __forceinline__ void store_row(T* p, vec_t<float, N> v) {
    *reinterpret_cast<vec_t<T, N>*>(p) = __builtin_convertvector(v, vec_t<T, N>);
}

// Bytes that the last level of cache holds: larger outputs are written past
// its order (ONCE).  A constant, as the compiler makes one plain store of two
// that a value at run time chooses between.
constexpr std::uint64_t kCacheBytes = 256 << 20;

template <bool ONCE, typename T, int N>
__device__ __forceinline__ void write_out(T* p, vec_t<float, N> v) {
    if constexpr (ONCE) __builtin_nontemporal_store(__builtin_convertvector(v, vec_t<T, N>), reinterpret_cast<vec_t<T, N>*>(p));
    else store_row<T, N>(p, v);
}

// N elements at any address of an element: CDNA4 reads and writes 16 bytes a lane
// at any of them, and a copy of 2 GiB runs as fast (4.6 TB/s at odd 16-bit
// elements as at aligned ones; with 2 bytes a lane 2.7).
template <typename T, int N>
using any_vec_t = T __attribute__((ext_vector_type(N), aligned(sizeof(T))));

template <typename T, int N, bool ONCE = false>
__device__ __forceinline__ vec_t<T, N> load_as(const T* p) {
    const auto* g = (const __attribute__((address_space(1))) any_vec_t<T, N>*)(reinterpret_cast<std::uintptr_t>(p));
    if constexpr (ONCE) return __builtin_nontemporal_load(g);
    else return *g;
}
template <typename T, int N, bool ONCE = false>
__device__ __forceinline__ vec_t<float, N> load_any(const T* p) {
    return __builtin_convertvector(load_as<T, N, ONCE>(p), vec_t<float, N>);
}
template <typename T, int N, bool ONCE = false>
__device__ __forceinline__ void store_any(T* p, vec_t<float, N> v) {
    auto* to = reinterpret_cast<any_vec_t<T, N>*>(p);
    if constexpr (ONCE) __builtin_nontemporal_store(static_cast<any_vec_t<T, N>>(__builtin_convertvector(v, vec_t<T, N>)), to);
    else *to = __builtin_convertvector(v, vec_t<T, N>);
}

// Elements of a 16-byte vector.
template <typename T>
constexpr int kVec = 16 / sizeof(T);

// Element bytes of a TCC_F32 / TCC_BF16 / TCC_F16 code, 0 for any other.
inline std::uint32_t dtype_bytes(std::uint64_t dtype) { return dtype == 0 ? 4u : (dtype == 1 || dtype == 2) ? 2u : 0u; }

// The most elements (a power of two, at most 16 bytes) that a lane can take
// at once of rows of `cols` elements, given the addresses and byte strides
// that have to keep the alignment.
struct RowWidth {
    std::uint64_t bits;
    explicit RowWidth(std::uint64_t cols, std::uint32_t elem) : elem_(elem) { bits = (16 | cols * elem); }
    RowWidth& with(const void* p) {
        bits |= reinterpret_cast<std::uintptr_t>(p);
        return *this;
    }
    RowWidth& stride(std::uint64_t elems) {
        bits |= elems * elem_;
        return *this;
    }
    std::uint32_t elems() const { return static_cast<std::uint32_t>(bits & (~bits + 1)) / elem_; }

private:
    std::uint32_t elem_;
};

}  // namespace tcc
