// y = act(x w^T + bias) + residual and its gradients (the formulas are at ssmap_linear and
// ssmap_linear_grad in ssmap.h).
//
// Every product here is out[m][n] = sum_k a(m, k) b(n, k) over operands given by strides.  rows: m is a
// position, n an output, so bias lies along n.  planes: the operands change places, m is an output and n
// a position, so that the dense axis of the planes is the dense axis of the tiles.
#include <math.h>

#include "heads.h"
#include "products.h"
#include "tiles.h"

using namespace ssmap;

namespace {

__device__ __forceinline__ float slope(float z, int act) {
    if (act == SSMAP_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
    if (act == SSMAP_ACT_GELU)
        return 0.5f * erfcf(-0.70710678118654752f * z) + z * 0.39894228040143268f * expf(-0.5f * z * z);
    if (act == SSMAP_ACT_GELU_TANH) {
        const float u = 0.79788456080286536f * (z + 0.044715f * z * z * z);
        const float q = 1.0f / (1.0f + expf(-2.0f * u));     // (1 + tanh u) / 2; its slope in u is 2 q (1 - q)
        const float du = 0.79788456080286536f * (1.0f + 3.0f * 0.044715f * z * z);
        return q + (1.0f - q > 0.0f && q > 0.0f ? z * 2.0f * q * (1.0f - q) * du : 0.0f);
    }
    if (act == SSMAP_ACT_SILU) {
        const float q = 1.0f / (1.0f + expf(-z));
        return q + (q > 0.0f && q < 1.0f ? z * q * (1.0f - q) : 0.0f);
    }
    return 1.0f;
}

// dz = g act'(pre) in the products' type, dense.  out: [batch][P][Q], g strided by (batch, P).
template <int DT, int OT>
__global__ __launch_bounds__(256) void k_dz(int64_t batch, int64_t P, int64_t Q, const elem_t<OT> *g, int64_t g_batch, int64_t g_p,
                                            const elem_t<DT> *pre, int act, elem_t<DT> *dz) {
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < batch * P * Q; i += gridDim.x * 256ll) {
        const int64_t q = i % Q, pp = i / Q % P, b = i / Q / P;
        float v = Elem<OT>::get(g[b * g_batch + pp * g_p + q]);
        if (pre) v *= slope(Elem<DT>::get(pre[i]), act);
        dz[i] = Elem<DT>::put(v);
    }
}

// g_bias: one block per output sums its dz over the positions, each thread a fixed share, joined in a fixed order.
template <int DT, int OT>
__global__ __launch_bounds__(256) void k_bias_grad(int64_t batch, int64_t rows, int64_t outer, const elem_t<OT> *g, int64_t g_batch,
                                                   int64_t g_row, int64_t g_out, const elem_t<DT> *pre, int64_t pre_row, int64_t pre_out,
                                                   int act, elem_t<DT> *out) {
    __shared__ float part[256];
    for (int64_t n = blockIdx.x; n < outer; n += gridDim.x) {
        float s = 0.0f;
        for (int64_t i = threadIdx.x; i < batch * rows; i += 256) {
            const int64_t b = i / rows, r = i % rows;
            float v = Elem<OT>::get(g[b * g_batch + r * g_row + n * g_out]);
            if (pre) v *= slope(Elem<DT>::get(pre[b * rows * outer + r * pre_row + n * pre_out]), act);
            s += v;
        }
        part[threadIdx.x] = s;
        __syncthreads();
        for (int d = 128; d; d >>= 1) {
            if (threadIdx.x < d) part[threadIdx.x] += part[threadIdx.x + d];
            __syncthreads();
        }
        if (!threadIdx.x) out[n] = Elem<DT>::put(part[0]);
        __syncthreads();
    }
}

// Calls f with the operand type and the output's type (the same or float) as constants.
template <typename F>
void with_types(int dtype, int other, F f) {
    if (dtype == SSMAP_F32) f(std::integral_constant<int, SSMAP_F32>{}, std::integral_constant<int, SSMAP_F32>{});
    else if (dtype == SSMAP_BF16 && other == SSMAP_BF16) f(std::integral_constant<int, SSMAP_BF16>{}, std::integral_constant<int, SSMAP_BF16>{});
    else if (dtype == SSMAP_BF16) f(std::integral_constant<int, SSMAP_BF16>{}, std::integral_constant<int, SSMAP_F32>{});
    else if (other == SSMAP_F16) f(std::integral_constant<int, SSMAP_F16>{}, std::integral_constant<int, SSMAP_F16>{});
    else f(std::integral_constant<int, SSMAP_F16>{}, std::integral_constant<int, SSMAP_F32>{});
}

template <typename Args>
int check(const Args *a, int other) {
    if (!head_dtype_ok(a->dtype)) return head_error(SSMAP_ERR_INVALID_ARG, "dtype is none of SSMAP_F32, SSMAP_BF16, SSMAP_F16");
    if (other != a->dtype && other != SSMAP_F32) return head_error(SSMAP_ERR_INVALID_ARG, "the results' type must be dtype or SSMAP_F32");
    if (a->layout != SSMAP_ROWS && a->layout != SSMAP_PLANES)
        return head_error(SSMAP_ERR_INVALID_ARG, "layout is neither SSMAP_ROWS nor SSMAP_PLANES");
    if (a->activation < SSMAP_ACT_NONE || a->activation > SSMAP_ACT_SILU) return head_error(SSMAP_ERR_INVALID_ARG, "unknown activation");
    if (!head_sizes_ok(a->batch, a->rows, a->inner) || !head_sizes_ok(a->batch, a->rows, a->outer) || !head_sizes_ok(1, a->outer, a->inner))
        return head_error(SSMAP_ERR_INVALID_ARG, "sizes must not be negative, and no tensor may have 2^40 elements");
    return SSMAP_OK;
}

int check_linear(const ssmap_linear_args *a) {
    if (!a) return head_error(SSMAP_ERR_INVALID_ARG, "null argument");
    if (int rc = check(a, a->out_dtype)) return rc;
    if (a->bias && a->bias_dtype != a->dtype && a->bias_dtype != SSMAP_F32)
        return head_error(SSMAP_ERR_INVALID_ARG, "the bias's type must be dtype or SSMAP_F32");
    return SSMAP_OK;
}

int check_grad(const ssmap_linear_grad_args *a) {
    if (!a) return head_error(SSMAP_ERR_INVALID_ARG, "null argument");
    return check(a, a->grad_dtype);
}

inline int64_t aligned(int64_t bytes) { return (bytes + 255) & ~(int64_t)255; }

}  // namespace

extern "C" {

int64_t ssmap_linear_workspace(const ssmap_linear_args *a) { return check_linear(a) == SSMAP_OK ? 0 : -1; }

int ssmap_linear(const ssmap_linear_args *a, void *stream) {
    if (int rc = check_linear(a)) return rc;
    const int64_t positions = a->batch * a->rows;
    if (positions == 0 || a->outer == 0) return SSMAP_OK;
    if (!a->y || (a->inner && (!a->x || !a->w))) return head_error(SSMAP_ERR_INVALID_ARG, "null argument");
    if (a->workspace_bytes < ssmap_linear_workspace(a)) return head_error(SSMAP_ERR_INVALID_ARG, "the workspace is smaller than ssmap_linear_workspace says");
    const bool planes = a->layout == SSMAP_PLANES;
    Product p{};
    p.K = a->inner; p.out_batches = a->batch; p.sum_batches = 1;
    p.out = a->y; p.pre = a->pre; p.bias = a->bias; p.res = a->residual;
    p.bias_f32 = a->bias_dtype == SSMAP_F32; p.bias_along_m = planes; p.act = a->activation;
    p.res_out = a->res_batch_stride; p.res_m = a->res_inner_stride;
    if (planes) {
        p.M = a->outer; p.N = a->rows;
        p.a = a->w; p.a_m = a->w_row_stride; p.a_k = 1;
        p.b = a->x; p.b_n = a->x_row_stride; p.b_k = 1; p.b_out = a->x_batch_stride;
    } else {
        p.M = a->rows; p.N = a->outer;
        p.a = a->x; p.a_m = a->x_row_stride; p.a_k = 1; p.a_out = a->x_batch_stride;
        p.b = a->w; p.b_n = a->w_row_stride; p.b_k = 1;
    }
    with_types(a->dtype, a->out_dtype, [&](auto dt, auto ot) { launch_product<dt.value, ot.value>(p, static_cast<hipStream_t>(stream)); });
    return head_launch_error(hipGetLastError());
}

int64_t ssmap_linear_grad_workspace(const ssmap_linear_grad_args *a) {
    if (check_grad(a) != SSMAP_OK) return -1;
    return aligned(a->batch * a->rows * a->outer * head_dtype_size(a->dtype));
}

int ssmap_linear_grad(const ssmap_linear_grad_args *a, void *stream) {
    if (int rc = check_grad(a)) return rc;
    const int64_t positions = a->batch * a->rows;
    if (positions && a->outer && !a->g) return head_error(SSMAP_ERR_INVALID_ARG, "null argument");
    if (a->activation != SSMAP_ACT_NONE && positions && a->outer && !a->pre) return head_error(SSMAP_ERR_INVALID_ARG, "an activation's gradient needs pre");
    if ((a->g_x && positions && a->inner && a->outer && !a->w) || (a->g_w && a->outer && a->inner && positions && !a->x))
        return head_error(SSMAP_ERR_INVALID_ARG, "null argument");
    const int64_t need = ssmap_linear_grad_workspace(a);
    if (a->workspace_bytes < need || (need && !a->workspace))
        return head_error(SSMAP_ERR_INVALID_ARG, "the workspace is smaller than ssmap_linear_grad_workspace says");
    const bool planes = a->layout == SSMAP_PLANES;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const void *pre = a->activation == SSMAP_ACT_NONE ? nullptr : a->pre;
    with_types(a->dtype, a->grad_dtype, [&](auto dt, auto ot) {
        constexpr int DT = dt.value, OT = ot.value;
        const int64_t P = planes ? a->outer : a->rows, Q = planes ? a->rows : a->outer;
        const auto *g = static_cast<const elem_t<OT> *>(a->g);
        auto *dz = static_cast<elem_t<DT> *>(a->workspace);
        const auto *z = static_cast<const elem_t<DT> *>(pre);
        if (positions * a->outer)
            k_dz<DT, OT><<<blocks((positions * a->outer + 255) / 256), 256, 0, st>>>(a->batch, P, Q, g, a->g_batch_stride, a->g_inner_stride, z, a->activation, dz);
        if (a->g_bias && a->outer)
            k_bias_grad<DT, OT><<<blocks(a->outer), 256, 0, st>>>(a->batch, a->rows, a->outer, g, a->g_batch_stride, planes ? 1 : a->g_inner_stride,
                                                                  planes ? a->g_inner_stride : 1, z, planes ? 1 : a->outer, planes ? a->rows : 1,
                                                                  a->activation, static_cast<elem_t<DT> *>(a->g_bias));
        if (a->g_x) {
            Product p{};
            p.M = a->rows; p.N = a->inner; p.K = a->outer; p.out_batches = a->batch; p.sum_batches = 1;
            p.a = dz; p.a_out = a->rows * a->outer; p.a_m = planes ? 1 : a->outer; p.a_k = planes ? a->rows : 1;
            p.b = a->w; p.b_n = 1; p.b_k = a->w_row_stride;
            p.out = a->g_x;
            launch_product<DT, DT>(p, st);
        }
        if (a->g_w) {
            Product p{};
            p.M = a->outer; p.N = a->inner; p.K = a->rows; p.out_batches = 1; p.sum_batches = a->batch;
            p.a = dz; p.a_sum = a->rows * a->outer; p.a_m = planes ? a->rows : 1; p.a_k = planes ? 1 : a->outer;
            p.b = a->x; p.b_sum = a->x_batch_stride; p.b_n = 1; p.b_k = a->x_row_stride;
            p.out = a->g_w;
            launch_product<DT, DT>(p, st);
        }
    });
    return head_launch_error(hipGetLastError());
}

}  // extern "C"
