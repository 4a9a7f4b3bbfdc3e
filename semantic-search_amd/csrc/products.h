// A product of linear.hip and the launcher of its kernels, which are compiled one operand type a file.
#pragma once

#include <math.h>

#include <type_traits>

#include "heads.h"

namespace ssmap {

struct Product {
    int64_t M, N, K;
    int64_t out_batches;                    // out, a, b and the epilogue advance together
    int64_t sum_batches;                    // the sum runs over this many blocks of K as well (over the envs, over dz's parts)
    int64_t b_again;                        // after this many of them b starts over
    const void *a, *b;
    int64_t a_m, a_k, a_out, a_sum;         // strides in elements; of an out batch; of a sum batch
    int64_t b_n, b_k, b_out, b_sum;
    // Which axis of an operand is dense in memory (its stride is 1): the sum's, or the result's.  The builder says so;
    // strides cannot, as overlapping or single lines may have a stride of 1 along both.  b is dense along the sum only
    // where a is: those three forms have kernels.
    bool a_sums, b_sums;
    void *out;                              // dense [out_batches][M][N]
    void *pre;                              // the same in the operands' type, or NULL
    const float *unscale;                   // fp16: the products' sums are multiplied by this, on the device; or NULL
    const void *bias, *res;
    int32_t bias_f32, bias_along_m, act, pad;
    int64_t res_out, res_m;
    // the sum is split into `splits` parts of `part_steps` stages of 128 bytes a row; more than one: float32 partial results go to
    // parts[split][out_batches][M][N] and are joined afterwards
    int64_t part_steps;
    int32_t splits, shape;                  // shape: see plan_product
    float *parts;
    // operands whose lines do not start at multiples of 16 bytes are copied first, to lines that do: places
    // behind `parts`, or -1
    int64_t pack_a, pack_b;
    bool a_pads;                            // a's lines are filled up with zeros to multiples of 16 bytes
};

// Tile shapes (m x n).
enum Shape { kTileBig = 0, kTileMid = 1, kTileLow = 2, kTileTall = 3, kTileMidAny = 4, kFewRows = 5, kHead = 6, kTileSmallAny = 7, kTileSmall = 8 };
constexpr int kFewMost = 32;                // rows of a that kFewRows takes at most
constexpr int kHeadMost = 64;               // rows of a that kHead takes at most, and their bytes in LDS
constexpr int kHeadBytes = 64 << 10;
// kHead's LDS rows: chunks, rounded up to whole swizzles of eight
inline int64_t head_pitch(const Product &p, int size) { return (p.K * size / 16 + 7) / 8 * 8; }
inline int64_t head_bytes(const Product &p, int size) { return (p.M + 15) / 16 * 16 * head_pitch(p, size) * 16; }

inline unsigned blocks(int64_t n) { return (unsigned)(n < 1 ? 1 : n < (1 << 20) ? n : (1 << 20)); }

// Chooses p.shape, p.splits, p.part_steps and the copies by sizes, strides and alignment; returns the bytes that
// p.parts needs.
int64_t plan_product(Product &p, int dtype);
// FINE: for results in float32.  Results of 16 bits take erfc(x) exp(x^2) / 2 = t P(t) with t = 1 / (1 + 0.5125 x), a
// least-maximum fit relative to the value over 0 <= x <= 10: it is off by at most 7.7e-7 of it, and by 1.7e-5 with the
// rounding of x^2 at z = -13, which is far below the rounding of the results (2^-11, 2^-8) out to the smallest of them.
constexpr float kErfcAt = 0.5125f;
__device__ __forceinline__ float erfc_ratio(float t) {
    return t * (0.14465798f + t * (0.142883733f + t * (0.13929078f + t * (0.029507799f + t * (0.17541796f + t * (-0.179791331f + t * 0.0480334461f))))));
}
template <bool FINE>
__device__ __forceinline__ float half_erfc(float x) {   // erfc(x) / 2
    if constexpr (FINE) return 0.5f * erfcf(x);
    const float a = fabsf(x), t = __builtin_amdgcn_rcpf(1.0f + kErfcAt * a);
    const float v = erfc_ratio(t) * __builtin_amdgcn_exp2f(-1.44269504088896341f * a * a);
    return x < 0.0f ? 1.0f - v : v;
}
template <bool FINE>
__device__ __forceinline__ float logistic(float x) {    // 1 / (1 + exp(-x))
    if constexpr (FINE) return 1.0f / (1.0f + expf(-x));
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896341f * x));
}
template <int ACT, bool FINE>
__device__ __forceinline__ float activate(float z) {
    if constexpr (ACT == SSMAP_ACT_RELU) return z < 0.0f ? 0.0f : z;
    if constexpr (ACT == SSMAP_ACT_GELU) return z * half_erfc<FINE>(-0.70710678118654752f * z);
    // (1 + tanh u) / 2 = 1 / (1 + exp(-2u))
    if constexpr (ACT == SSMAP_ACT_GELU_TANH) return z * logistic<FINE>(1.5957691216057308f * (z + 0.044715f * z * z * z));
    if constexpr (ACT == SSMAP_ACT_SILU) return z * logistic<FINE>(z);
    return z;
}
template <int ACT, bool FINE>
__device__ __forceinline__ float slope(float z) {
    if constexpr (ACT == SSMAP_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
    if constexpr (ACT == SSMAP_ACT_GELU) {
        // the second term's limit is 0 where z may be infinite
        if constexpr (FINE) {
            const float bell = expf(-0.5f * z * z);
            return half_erfc<true>(-0.70710678118654752f * z) + (bell > 0.0f ? z * 0.39894228040143268f * bell : 0.0f);
        }
        // the formula of half_erfc at z / sqrt 2: its exponential is the bell
        const float a = fabsf(z), t = __builtin_amdgcn_rcpf(1.0f + kErfcAt * 0.70710678118654752f * a);
        const float bell = __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z);
        const float tail = bell * erfc_ratio(t);
        return (z < 0.0f ? tail : 1.0f - tail) + (bell > 0.0f ? z * 0.39894228040143268f * bell : 0.0f);
    }
    if constexpr (ACT == SSMAP_ACT_GELU_TANH) {
        // q = (1 + tanh u) / 2; its slope in u is 2 q (1 - q), which is 0 where z may be infinite
        const float q = logistic<FINE>(1.5957691216057308f * (z + 0.044715f * z * z * z));
        const float du = 0.79788456080286536f * (1.0f + 3.0f * 0.044715f * z * z);
        return q + (q > 0.0f && q < 1.0f ? z * 2.0f * q * (1.0f - q) * du : 0.0f);
    }
    if constexpr (ACT == SSMAP_ACT_SILU) {
        const float q = logistic<FINE>(z);
        return q + (q > 0.0f && q < 1.0f ? z * q * (1.0f - q) : 0.0f);
    }
    return 1.0f;
}
// Calls f with the activation as a constant: one branch for a run of values, not one for each.
template <typename F>
__device__ __forceinline__ void with_activation(int act, F f) {
    if (act == SSMAP_ACT_RELU) f(std::integral_constant<int, SSMAP_ACT_RELU>{});
    else if (act == SSMAP_ACT_GELU) f(std::integral_constant<int, SSMAP_ACT_GELU>{});
    else if (act == SSMAP_ACT_GELU_TANH) f(std::integral_constant<int, SSMAP_ACT_GELU_TANH>{});
    else if (act == SSMAP_ACT_SILU) f(std::integral_constant<int, SSMAP_ACT_SILU>{});
}

// Enqueues a planned product of operands of type DT with results of type OT (DT or SSMAP_F32).
template <int DT, int OT>
void launch_product(Product p, hipStream_t st);

}  // namespace ssmap
