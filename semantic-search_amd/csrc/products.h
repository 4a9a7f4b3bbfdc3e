// A product of linear.hip and the launcher of its kernels, which are compiled one operand type a file.
#pragma once

#include "heads.h"

namespace ssmap {

struct Product {
    int64_t M, N, K;
    int64_t out_batches;                    // out, a, b and the epilogue advance together
    int64_t sum_batches;                    // the sum runs over this many blocks of K as well (planes: over the envs)
    const void *a, *b;
    int64_t a_m, a_k, a_out, a_sum;         // strides in elements; of an out batch; of a sum batch
    int64_t b_n, b_k, b_out, b_sum;
    void *out;                              // dense [out_batches][M][N]
    void *pre;                              // the same in the operands' type, or NULL
    const void *bias, *res;
    int32_t bias_f32, bias_along_m, act, pad;
    int64_t res_out, res_m;
    // the sum is split into `splits` parts of `part_steps` stages; more than one: float32 partial results go to
    // parts[split][out_batches][M][N] and are joined afterwards
    int64_t part_steps;
    int32_t splits, pad2;
    float *parts;
};

inline unsigned blocks(int64_t n) { return (unsigned)(n < 1 ? 1 : n < (1 << 20) ? n : (1 << 20)); }

// Enqueues a product of operands of type DT with results of type OT (DT or SSMAP_F32).
template <int DT, int OT>
void launch_product(const Product &p, hipStream_t st);

}  // namespace ssmap
