// Shared by the head operators (scores.hip, linear.hip): element types, argument checks.
#pragma once

#include "ssmap_internal.h"

namespace ssmap {

// Defined in engine.cpp: keeps the text for ssmap_last_error() and returns `code`.  Never throws.
int head_error(int code, const char *text) noexcept;

// Element types as the kernels hold them in memory.  Arithmetic is in float; storing rounds once, to
// nearest even.
template <int DT>
struct Elem;
template <>
struct Elem<SSMAP_F32> {
    using type = float;
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Elem<SSMAP_BF16> {
    using type = __bf16;
    static __device__ __forceinline__ float get(__bf16 v) {
        return __builtin_bit_cast(float, (uint32_t)__builtin_bit_cast(uint16_t, v) << 16);
    }
    static __device__ __forceinline__ __bf16 put(float v) { return (__bf16)v; }
};
template <>
struct Elem<SSMAP_F16> {
    using type = _Float16;
    static __device__ __forceinline__ float get(_Float16 v) { return (float)v; }
    static __device__ __forceinline__ _Float16 put(float v) { return (_Float16)v; }
};
template <int DT>
using elem_t = typename Elem<DT>::type;

constexpr bool head_dtype_ok(int dt) { return dt == SSMAP_F32 || dt == SSMAP_BF16 || dt == SSMAP_F16; }
constexpr int head_dtype_size(int dt) { return dt == SSMAP_F32 ? 4 : 2; }

// a * b * c of non-negative sizes stays below 2^40 (addresses and grids are computed in 64 bits; a tensor
// of 2^40 elements is larger than the card's memory)
inline bool head_sizes_ok(int64_t a, int64_t b, int64_t c) {
    constexpr int64_t most = (int64_t)1 << 40;
    if (a < 0 || b < 0 || c < 0 || a > most || b > most || c > most) return false;
    if (a == 0 || b == 0 || c == 0) return true;
    return a <= most / b && a * b <= most / c;
}

inline int head_launch_error(hipError_t e) { return e == hipSuccess ? SSMAP_OK : head_error(SSMAP_ERR_HIP, hipGetErrorString(e)); }

}  // namespace ssmap
