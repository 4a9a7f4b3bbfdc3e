// y = act(x w^T + bias) + residual and its gradients (the formulas are at ssmap_linear and
// ssmap_linear_grad in ssmap.h).
//
// Every product here is out[m][n] = sum_k a(m, k) b(n, k) over operands given by strides.  rows: m is a
// position, n an output, so bias lies along n.  planes: the operands change places, m is an output and n
// a position, so that the dense axis of the planes is the dense axis of the tiles.
#include <math.h>

#include "products.h"

using namespace ssmap;

namespace {

// Whether a side can go straight to LDS: lines at multiples of 16 bytes, no partial chunk, 32-bit offsets
// within a tile.
inline bool direct_side(const void *p, int64_t line, int64_t out, int64_t sum, int64_t dense, int size) {
    const int64_t e = 16 / size;
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && line % e == 0 && out % e == 0 && sum % e == 0 && dense % e == 0 &&
           line >= 0 && line < (int64_t)1 << 21;
}

// dz = g act'(pre) in the products' type, dense, and the sums of its positions for the bias's gradient, in one
// pass over g.  [batch][P][Q], Q dense: rows have the outputs in Q, planes in P.  8192 x 4096 bf16 with gelu takes
// 85 us (the bytes 52): the slope's two transcendentals a value and both parts' roundings fill the rest.
//
// Where 16 bits do not hold dz it is kept as two values, the rounded one and what the rounding left, and the products
// sum over both: dz then counts with 2^-16 (bf16) or 2^-22 (fp16) of its size, and a result is rounded once, as the
// forward product's is.  With the rounded value alone the gradients' distance to the definition grows by 1.4 (8192 x
// 4096 x 4096 bf16 with gelu: 2.35e-3 against 1.66e-3 of the results' size) and the products take half the time (the
// whole call 494 against 930 us).
//
// fp16 holds nothing above 65504 and little below 2^-14, where a float32 gradient averaged over a frame's positions
// lies.  There dz is multiplied by the power of two that brings the largest finite |g| to 2^13 ... 2^14 (no slope exceeds
// 1.13), and the products' sums by its inverse: what is lost of a value is at most 2^-38 of that largest one.
// The look at g takes 11 us for 40 planes of 307200 positions (4.6 TB/s), the scale 4.
constexpr int kDzRows = 128;       // rows: positions a block sums; 8 threads down, 32 packs of 8 outputs across
constexpr int kDzPlane = 16384;    // planes: positions a block sums

struct Dz {
    int64_t batch, rows, outer;
    int64_t g_batch, g_line;           // strides of g
    int64_t line;                      // values a line of dz takes, zeros behind the dense ones
    int64_t rest;                      // what dz's roundings left lies that many values behind it; 0: not kept
    int32_t act;
    const float *scale;                // what dz is multiplied by, or NULL
    float *sums;                       // for the bias's gradient, or NULL
};

// Eight neighbours, of which `left` exist; WHOLE: all, which the caller knows for its whole wave.
template <bool WHOLE, int T>
__device__ __forceinline__ void load8(const elem_t<T> *p, int left, float (&v)[8]) {
    if constexpr (WHOLE) {
        elem_t<T> w[8];
        __builtin_memcpy(w, p, sizeof w);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = Elem<T>::get(w[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < left ? Elem<T>::get(p[e]) : 0.0f;
    }
}
template <bool WHOLE, int DT, int OT>
__device__ __forceinline__ void dz_pack(const Dz &a, float by, const elem_t<OT> *g, const elem_t<DT> *pre, elem_t<DT> *dz, int left, int room,
                                        float (&sum)[8]) {   // room: of dz's line, zeros included
    float v[8];
    load8<WHOLE, OT>(g, left, v);
    if (pre) {
        float z[8];
        load8<WHOLE, DT>(pre, left, z);
        with_activation(a.act, [&](auto act) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= slope<act.value, DT == SSMAP_F32>(z[e]);
        });
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] += WHOLE || e < left ? v[e] : 0.0f;
    if (!dz) return;
    elem_t<DT> w[8];
    const auto keep = [&](elem_t<DT> *to) {
        if constexpr (WHOLE) {
            __builtin_memcpy(to, w, sizeof w);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < room) to[e] = e < left ? w[e] : Elem<DT>::put(0.0f);
        }
    };
    if (DT == SSMAP_F32 || !a.rest) {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = Elem<DT>::put(v[e]);
        return keep(dz);
    }
    // clamped to the type's range, so that what an infinity or NaN leaves is itself
    constexpr float most = DT == SSMAP_BF16 ? 0x1.fep127f : 65504.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (DT == SSMAP_F16) v[e] *= by;
        w[e] = Elem<DT>::put(fminf(fmaxf(v[e], -most), most));
        v[e] -= Elem<DT>::get(w[e]);
    }
    keep(dz);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = Elem<DT>::put(v[e]);
    keep(dz + a.rest);
}

// The largest finite |g| of each block's share: lines of `dense` values, `lines` a batch.
constexpr int kPeaks = 1024;   // blocks at most
template <int OT>
__global__ __launch_bounds__(256) void k_peak(int64_t batch, int64_t lines, int64_t dense, const elem_t<OT> *g, int64_t g_batch, int64_t g_line,
                                              float *peaks) {
    __shared__ float part[4];
    const int64_t per = (dense + 7) / 8, units = batch * lines * per;
    float peak = 0.0f;
    for (int64_t u = blockIdx.x * 256ll + threadIdx.x; u < units; u += gridDim.x * 256ll) {
        const int64_t l = u / per, c = u % per * 8;
        const elem_t<OT> *p = g + l / lines * g_batch + l % lines * g_line + c;
        float v[8];
        if (c + 8 <= dense) load8<true, OT>(p, 8, v);
        else load8<false, OT>(p, (int)(dense - c), v);
#pragma unroll
        for (int e = 0; e < 8; ++e) peak = fabsf(v[e]) < INFINITY ? fmaxf(peak, fabsf(v[e])) : peak;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) peak = fmaxf(peak, __shfl_xor(peak, d));
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = peak;
    __syncthreads();
    if (!threadIdx.x) peaks[blockIdx.x] = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
}
// scale[0]: what dz is multiplied by, scale[1]: its inverse.  One block.
__global__ __launch_bounds__(kPeaks) void k_scale(const float *peaks, int n, float *scale) {
    __shared__ float part[kPeaks / 64];
    float peak = threadIdx.x < n ? peaks[threadIdx.x] : 0.0f;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) peak = fmaxf(peak, __shfl_xor(peak, d));
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = peak;
    __syncthreads();
    if (threadIdx.x) return;
    for (int k = 1; k < kPeaks / 64; ++k) peak = fmaxf(peak, part[k]);
    const int e = (int)(__builtin_bit_cast(uint32_t, peak) >> 23) - 127;   // floor(log2 peak), -127 below the normal ones
    const int by = 13 - e < 126 ? 13 - e : 126;                            // -114 ... 126: both powers are normal
    scale[0] = __builtin_bit_cast(float, (uint32_t)(127 + by) << 23);
    scale[1] = __builtin_bit_cast(float, (uint32_t)(127 - by) << 23);
}

// sums[batch * row chunks][outer]
template <int DT, int OT>
__global__ __launch_bounds__(256) void k_dz_rows(Dz a, const elem_t<OT> *g, const elem_t<DT> *pre, elem_t<DT> *dz) {
    __shared__ float part[8][256];
    const float by = a.scale ? *a.scale : 1.0f;
    const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;
    const int64_t rows = a.rows, outer = a.outer, strips = (outer + 255) / 256, chunks = (rows + kDzRows - 1) / kDzRows;
    for (int64_t unit = blockIdx.x; unit < strips * chunks * a.batch; unit += gridDim.x) {
        const int64_t n = unit % strips * 256 + tx * 8, bc = unit / strips, b = bc / chunks, r0 = bc % chunks * kDzRows;
        const int left = (int)(outer - n < 8 ? outer - n : 8), room = (int)(a.line - n < 8 ? a.line - n : 8);
        float sum[8] = {};
        const int64_t end = r0 + kDzRows < rows ? r0 + kDzRows : rows;
        const auto walk = [&](auto whole) {
#pragma unroll 2
            for (int64_t r = r0 + ty; r < end; r += 8) {
                const int64_t o = (b * rows + r) * outer + n;
                dz_pack<whole.value, DT, OT>(a, by, g + b * a.g_batch + r * a.g_line + n, pre ? pre + o : nullptr,
                                             dz ? dz + (b * rows + r) * a.line + n : nullptr, left, room, sum);
            }
        };
        if (unit % strips * 256 + 256 <= outer) walk(std::true_type{});
        else if (left > 0) walk(std::false_type{});
        if (!a.sums) continue;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) part[ty][tx * 8 + e] = sum[e];
        __syncthreads();
        const int64_t out = unit % strips * 256 + threadIdx.x;
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) s += part[k][threadIdx.x];
        if (out < outer) a.sums[bc * outer + out] = s;
    }
}

// sums[batch * chunks][outer]
template <int DT, int OT>
__global__ __launch_bounds__(256) void k_dz_planes(Dz a, const elem_t<OT> *g, const elem_t<DT> *pre, elem_t<DT> *dz) {
    __shared__ float part[256];
    const float by = a.scale ? *a.scale : 1.0f;
    const int64_t rows = a.rows, outer = a.outer, chunks = (rows + kDzPlane - 1) / kDzPlane;
    for (int64_t unit = blockIdx.x; unit < chunks * outer * a.batch; unit += gridDim.x) {
        const int64_t c = unit % chunks, bn = unit / chunks, b = bn / outer, n = bn % outer;
        float sum[8] = {};
        const int64_t end = (c + 1) * kDzPlane < rows ? (c + 1) * kDzPlane : rows;
        const elem_t<OT> *gp = g + b * a.g_batch + n * a.g_line;
        const elem_t<DT> *zp = pre ? pre + bn * rows : nullptr;
        elem_t<DT> *dp = dz ? dz + bn * a.line : nullptr;
        int64_t r = c * kDzPlane;
#pragma unroll 2
        for (; r + 2048 <= end; r += 2048) {
            const int64_t at = r + threadIdx.x * 8;
            dz_pack<true, DT, OT>(a, by, gp + at, zp ? zp + at : nullptr, dp ? dp + at : nullptr, 8, 8, sum);
        }
        const int64_t at = r + threadIdx.x * 8;
        const int left = (int)(end - at < 8 ? end - at : 8), room = (int)(end < rows ? 8 : a.line - at < 8 ? a.line - at : 8);
        if (at < end) dz_pack<false, DT, OT>(a, by, gp + at, zp ? zp + at : nullptr, dp ? dp + at : nullptr, left, room, sum);
        if (!a.sums) continue;
        part[threadIdx.x] = ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]));
        __syncthreads();
        for (int d = 128; d; d >>= 1) {
            if (threadIdx.x < d) part[threadIdx.x] += part[threadIdx.x + d];
            __syncthreads();
        }
        if (!threadIdx.x) a.sums[(b * chunks + c) * outer + n] = part[0];
        __syncthreads();
    }
}

// g_bias from the chunks' sums: a wave takes 64 chunks of one output at a time.
template <int DT>
__global__ __launch_bounds__(256) void k_bias_grad(int64_t chunks, int64_t outer, const float *sums, elem_t<DT> *out) {
    for (int64_t n = blockIdx.x * 4ll + threadIdx.x / 64; n < outer; n += gridDim.x * 4ll) {
        float s = 0.0f;
        for (int64_t c = threadIdx.x % 64; c < chunks; c += 64) s += sums[c * outer + n];
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
        if (threadIdx.x % 64 == 0) out[n] = Elem<DT>::put(s);
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
    if (a->x_batch_stride < 0 || a->x_row_stride < 0 || a->w_row_stride < 0) return head_error(SSMAP_ERR_INVALID_ARG, "strides must not be negative");
    if (!head_sizes_ok(a->batch, a->rows, a->inner) || !head_sizes_ok(a->batch, a->rows, a->outer) || !head_sizes_ok(1, a->outer, a->inner))
        return head_error(SSMAP_ERR_INVALID_ARG, "sizes must not be negative, and no tensor may have 2^40 elements");
    return SSMAP_OK;
}

int check_linear(const ssmap_linear_args *a) {
    if (!a) return head_error(SSMAP_ERR_INVALID_ARG, "null argument");
    if (int rc = check(a, a->out_dtype)) return rc;
    if (a->bias && a->bias_dtype != a->dtype && a->bias_dtype != SSMAP_F32)
        return head_error(SSMAP_ERR_INVALID_ARG, "the bias's type must be dtype or SSMAP_F32");
    if (a->res_batch_stride < 0 || a->res_inner_stride < 0) return head_error(SSMAP_ERR_INVALID_ARG, "strides must not be negative");
    return SSMAP_OK;
}

int check_grad(const ssmap_linear_grad_args *a) {
    if (!a) return head_error(SSMAP_ERR_INVALID_ARG, "null argument");
    if (a->g_batch_stride < 0 || a->g_inner_stride < 0) return head_error(SSMAP_ERR_INVALID_ARG, "strides must not be negative");
    return check(a, a->grad_dtype);
}

// The workspace of ssmap_linear_grad: dz, its scale and the blocks' peaks, the bias's sums, the partial results of the
// products (one after the other, so they share a place).
struct GradPlan {
    bool planes, copies;               // copies: dz is not g itself
    int64_t dz_line;                   // values a line of dz takes: a multiple of 16 bytes, zeros behind the dense ones
    int64_t dz_rest;                   // values from dz to what its roundings left; 0: dz is exact
    int64_t chunks;                    // sums a block leaves for each output
    Product x, w;
    int64_t dz_bytes, scale_bytes, sum_bytes, part_bytes;
    int64_t bytes() const { return dz_bytes + scale_bytes + sum_bytes + part_bytes; }
};

inline int64_t aligned(int64_t bytes) { return (bytes + 255) & ~(int64_t)255; }

Product forward_product(const ssmap_linear_args *a) {
    const bool planes = a->layout == SSMAP_PLANES;
    Product p{};
    p.K = a->inner; p.out_batches = a->batch; p.sum_batches = p.b_again = 1;
    p.a_sums = p.b_sums = true;
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
    return p;
}

GradPlan plan_grad(const ssmap_linear_grad_args *a) {
    GradPlan q{};
    q.planes = a->layout == SSMAP_PLANES;
    const int size = head_dtype_size(a->dtype);
    const int64_t e = 16 / size, dense = q.planes ? a->rows : a->outer;
    // a dz of one's own also where g's lines are not at multiples of 16 bytes: both products read it
    q.copies = a->activation != SSMAP_ACT_NONE || a->grad_dtype != a->dtype || reinterpret_cast<uintptr_t>(a->g) % 16 || a->g_inner_stride % e ||
               a->g_batch_stride % e || dense % e;
    q.dz_line = (dense + e - 1) / e * e;
    const int64_t chunk = q.planes ? kDzPlane : kDzRows;
    q.chunks = a->batch * ((a->rows + chunk - 1) / chunk);
    const int64_t values = a->batch * (q.planes ? a->outer : a->rows) * q.dz_line;
    const bool slopes = a->activation != SSMAP_ACT_NONE && a->activation != SSMAP_ACT_RELU;   // relu's are 0 and 1: exact
    q.dz_rest = a->dtype != SSMAP_F32 && (slopes || a->grad_dtype != a->dtype) ? values : 0;
    const int64_t parts = q.dz_rest ? 2 : 1;
    q.dz_bytes = q.copies && (a->g_x || a->g_w) ? aligned(parts * values * size) : 0;
    q.scale_bytes = q.dz_bytes && q.dz_rest && a->dtype == SSMAP_F16 ? aligned((2 + kPeaks) * 4) : 0;
    q.sum_bytes = a->g_bias ? aligned(q.chunks * a->outer * 4) : 0;
    // dz: [part][batch][position][output] or [part][batch][output][position]
    const void *dz = q.copies ? a->workspace : a->g;
    const int64_t line = q.copies ? q.dz_line : a->g_inner_stride, batch = q.copies ? (q.planes ? a->outer : a->rows) * q.dz_line : a->g_batch_stride;
    const int64_t to_row = q.planes ? 1 : line, to_out = q.planes ? line : 1;
    Product &x = q.x, &w = q.w;
    x.M = a->rows; x.N = a->inner; x.K = a->outer; x.out_batches = a->batch; x.sum_batches = parts; x.b_again = 1;
    x.a_pads = w.a_pads = q.copies;
    x.a_sums = !q.planes; w.a_sums = q.planes;   // b's dense axis is x's features: the result's
    x.a = dz; x.a_out = batch; x.a_sum = q.dz_rest; x.a_m = to_row; x.a_k = to_out;
    x.b = a->w; x.b_n = 1; x.b_k = a->w_row_stride;
    x.out = a->g_x;
    w.M = a->outer; w.N = a->inner; w.K = a->rows; w.out_batches = 1; w.sum_batches = parts * a->batch; w.b_again = a->batch ? a->batch : 1;
    w.a = dz; w.a_sum = batch; w.a_m = to_out; w.a_k = to_row;
    w.b = a->x; w.b_sum = a->x_batch_stride; w.b_n = 1; w.b_k = a->x_row_stride;
    w.out = a->g_w;
    const int64_t need_x = a->g_x ? plan_product(x, a->dtype) : 0, need_w = a->g_w ? plan_product(w, a->dtype) : 0;
    q.part_bytes = aligned(need_x > need_w ? need_x : need_w);
    return q;
}

}  // namespace

extern "C" {

int64_t ssmap_linear_workspace(const ssmap_linear_args *a) {
    if (check_linear(a) != SSMAP_OK) return -1;
    Product p = forward_product(a);
    return plan_product(p, a->dtype);
}

int ssmap_linear(const ssmap_linear_args *a, void *stream) {
    if (int rc = check_linear(a)) return rc;
    const int64_t positions = a->batch * a->rows;
    if (positions == 0 || a->outer == 0) return SSMAP_OK;
    if (!a->y || (a->inner && (!a->x || !a->w))) return head_error(SSMAP_ERR_INVALID_ARG, "null argument");
    Product p = forward_product(a);
    const int64_t need = plan_product(p, a->dtype);
    if (a->workspace_bytes < need || (need && (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 16)))
        return head_error(SSMAP_ERR_INVALID_ARG, "the workspace is not at a multiple of 16 or smaller than ssmap_linear_workspace says");
    p.parts = static_cast<float *>(a->workspace);
    with_types(a->dtype, a->out_dtype, [&](auto dt, auto ot) { launch_product<dt.value, ot.value>(p, static_cast<hipStream_t>(stream)); });
    return head_launch_error(hipGetLastError());
}

int64_t ssmap_linear_grad_workspace(const ssmap_linear_grad_args *a) {
    if (check_grad(a) != SSMAP_OK) return -1;
    const GradPlan q = plan_grad(a);
    return q.bytes();
}

int ssmap_linear_grad(const ssmap_linear_grad_args *a, void *stream) {
    if (int rc = check_grad(a)) return rc;
    const int64_t positions = a->batch * a->rows;
    if (positions && a->outer && !a->g) return head_error(SSMAP_ERR_INVALID_ARG, "null argument");
    if (a->activation != SSMAP_ACT_NONE && positions && a->outer && !a->pre) return head_error(SSMAP_ERR_INVALID_ARG, "an activation's gradient needs pre");
    if ((a->g_x && positions && a->inner && a->outer && !a->w) || (a->g_w && a->outer && a->inner && positions && !a->x))
        return head_error(SSMAP_ERR_INVALID_ARG, "null argument");
    GradPlan q = plan_grad(a);
    const int64_t need = q.bytes();
    if (a->workspace_bytes < need || (need && (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 16)))
        return head_error(SSMAP_ERR_INVALID_ARG, "the workspace is not at a multiple of 16 or smaller than ssmap_linear_grad_workspace says");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    char *ws = static_cast<char *>(a->workspace);
    float *scale = q.scale_bytes ? reinterpret_cast<float *>(ws + q.dz_bytes) : nullptr;
    float *sums = q.sum_bytes ? reinterpret_cast<float *>(ws + q.dz_bytes + q.scale_bytes) : nullptr;
    q.x.parts = q.w.parts = reinterpret_cast<float *>(ws + q.bytes() - q.part_bytes);
    q.x.unscale = q.w.unscale = scale && positions && a->outer ? scale + 1 : nullptr;   // without a dz nobody writes it
    with_types(a->dtype, a->grad_dtype, [&](auto dt, auto ot) {
        constexpr int DT = dt.value, OT = ot.value;
        const auto *g = static_cast<const elem_t<OT> *>(a->g);
        const auto *pre = a->activation == SSMAP_ACT_NONE ? nullptr : static_cast<const elem_t<DT> *>(a->pre);
        auto *dz = q.dz_bytes ? reinterpret_cast<elem_t<DT> *>(ws) : nullptr;
        if (q.x.unscale) {
            const int64_t lines = q.planes ? a->outer : a->rows, dense = q.planes ? a->rows : a->outer;
            const int64_t want = (a->batch * lines * ((dense + 7) / 8) + 255) / 256;
            const unsigned n = (unsigned)(want < kPeaks ? want : kPeaks);
            k_peak<OT><<<n, 256, 0, st>>>(a->batch, lines, dense, g, a->g_batch_stride, a->g_inner_stride, scale + 2);
            k_scale<<<1, kPeaks, 0, st>>>(scale + 2, (int)n, scale);
        }
        if (positions * a->outer && (dz || sums)) {
            const Dz z{a->batch, a->rows, a->outer, a->g_batch_stride, a->g_inner_stride, q.dz_line, q.dz_rest, a->activation, scale, sums};
            if (q.planes) k_dz_planes<DT, OT><<<blocks(q.chunks * a->outer), 256, 0, st>>>(z, g, pre, dz);
            else k_dz_rows<DT, OT><<<blocks(q.chunks * ((a->outer + 255) / 256)), 256, 0, st>>>(z, g, pre, dz);
        }
        if (a->g_bias && a->outer)
            k_bias_grad<DT><<<blocks((a->outer + 3) / 4), 256, 0, st>>>(q.chunks, a->outer, sums, static_cast<elem_t<DT> *>(a->g_bias));
        if (a->g_x) launch_product<DT, DT>(q.x, st);
        if (a->g_w) launch_product<DT, DT>(q.w, st);
    });
    return head_launch_error(hipGetLastError());
}

}  // extern "C"

int64_t ssmap::plan_product(Product &p, int dtype) {
    const int size = head_dtype_size(dtype);
    const bool ik = p.a_sums, jk = p.b_sums;
    // a line that stands alone has no stride
    if ((ik ? p.M : p.K) == 1) (ik ? p.a_m : p.a_k) = 0;
    if ((jk ? p.N : p.K) == 1) (jk ? p.b_n : p.b_k) = 0;
    if (p.out_batches == 1) p.a_out = p.b_out = 0;
    if (p.sum_batches == 1) p.a_sum = 0;
    if (p.b_again == 1) p.b_sum = 0;
    p.splits = 1;
    p.pack_a = p.pack_b = -1;
    const int64_t steps = (p.K * size + 127) / 128 * p.sum_batches;
    p.part_steps = steps;
    const bool direct_a = direct_side(p.a, ik ? p.a_m : p.a_k, p.a_out, p.a_sum, p.a_pads ? 0 : ik ? p.K : p.M, size);
    const bool direct_b = direct_side(p.b, jk ? p.b_n : p.b_k, p.b_out, p.b_sum, jk ? p.K : p.N, size);
    bool direct = direct_a && direct_b;
    const auto tiles = [&](int bi, int bj) { return (p.M + bi - 1) / bi * ((p.N + bj - 1) / bj) * p.out_batches; };
    const int64_t e = 16 / size;
    if (p.M <= kHeadMost && ik && jk && p.sum_batches == 1 && p.a_out == 0 && p.K >= e && p.K % e == 0 &&
        head_bytes(p, size) <= kHeadBytes && p.N * p.out_batches >= 16384) {
        // 256 bf16 features at 16384 positions: 40 classes 5.6 us and 11.8 in tiles, 16 classes 4.1 and 5.9 as few rows
        // (at 8192 positions 3.9 and 4.0); 64 classes at 65536 positions, all in the caches, 15.9 and 12.4
        p.shape = kHead;
        return 0;
    }
    if (p.M <= kFewMost && ik && jk && p.sum_batches == 1) {
        // 8 x 4096 x 4096 bf16 takes 9.3 us and 15.6 in tiles, 32 rows 14.5 and 19.0 (against 32768 outputs 91 and 58,
        // where a tile reads more of b at once); lines that start anywhere, 255 x 150000: one row 54 and 66, in float32
        // 43 and 133, 32 rows 77 and 74
        p.shape = kFewRows;
        return 0;
    }
    int64_t units = tiles(128, 128), full = 512;   // tiles, and how many are resident at once
    int64_t packed = 0;                            // bytes of the copies
    if (!direct && p.M > 64 && p.N > 64 && (double)p.M * p.N * p.K * p.out_batches * p.sum_batches >= (dtype == SSMAP_F32 ? 1 << 28 : 1 << 30)) {
        // Large enough to copy what is out of line first: 4097 x 4095 x 4099 bf16 takes 247 us with the copies and 361
        // with loads through registers that straddle lines (gradient of x: 260 and 608); for less the launches cost
        // more
        const auto copy = [&](bool kc, int64_t rows, int64_t blocks_in_sum, int64_t out) {
            const int64_t lines = kc ? rows : p.K, dense = kc ? p.K : rows, at = packed;
            packed += aligned((p.sum_batches > 1 ? blocks_in_sum : out ? p.out_batches : 1) * lines * ((dense + e - 1) / e * e) * size);
            return at;
        };
        // every line of a copy lies within 32-bit offsets of its tile
        if (((ik ? p.K : p.M) + e) < (int64_t)1 << 21 && ((jk ? p.K : p.N) + e) < (int64_t)1 << 21) {
            if (!direct_a) p.pack_a = copy(ik, p.M, p.sum_batches, p.a_out);
            if (!direct_b) p.pack_b = copy(jk, p.N, p.b_again, p.b_out);
            direct = true;
        }
    }
    if (dtype == SSMAP_F32 && direct) {
        // float32 matrix instructions take sixteen times as long, so how evenly the tiles fill the CUs decides: the
        // shape and split whose busiest CU is done first, with a stage of a 128 x 128 tile (or its like) at 2.1 us, of a
        // 64 x 64 tile at 0.8 us, and a join at 4 us and its bytes at 4 TB/s (all measured)
        double best = 1e30;
        const auto consider = [&](int shape, int64_t tiles_n, double stage) {
            for (int64_t s = 1; s <= 512 && (s == 1 || steps / s >= 4); s = s < 16 ? s + 1 : s * 2) {
                const int64_t part = (steps + s - 1) / s, n = (steps + part - 1) / part;
                const double us = (double)((tiles_n * n + 255) / 256) * part * stage + (n > 1 ? 4.0 + 8e-6 * n * p.out_batches * p.M * p.N / 4 : 0.0);
                if (us < best) best = us, p.shape = shape, p.part_steps = part, p.splits = (int)n;
            }
        };
        if (steps == 0) p.shape = kTileMid;
        else if (p.M <= 64) consider(kTileLow, tiles(64, 256), 2.1);
        else if (p.N <= 64) consider(kTileTall, tiles(256, 64), 2.1);
        else {
            consider(kTileMid, tiles(128, 128), 2.1);
            consider(kTileSmall, tiles(64, 64), 0.8);
        }
    } else {
        if (units < 128 && p.M > 64 && p.N > 64) {
            p.shape = direct ? kTileSmall : kTileSmallAny;
            units = tiles(64, 64), full = 768;
        } else if (!direct) {
            p.shape = kTileMidAny;
        } else if (p.M <= 64) {
            p.shape = kTileLow;
            units = tiles(64, 256);
        } else if (p.N <= 64) {
            p.shape = kTileTall;
            units = tiles(256, 64);
        } else if (dtype != SSMAP_F32 && tiles(256, 256) >= 192) {
            // Three quarters of a round of the large tile and more.  Sums of 4096, bf16, against middle tiles: 256 tiles
            // 115 and 136 us, 196 tiles 106 and 118, 160 tiles 103 and 111, 128 tiles 93 and 79; behind a whole round
            // 320 tiles 204 and 176.
            p.shape = kTileBig;
            units = tiles(256, 256), full = 256;
        } else {
            p.shape = kTileMid;
        }
        // Few tiles: the sum is split, in parts of eight stages at least; with half of the tiles that fit at once only
        // a long sum.  2048 x 2048 results, bf16: from 8192 products 112 -> 95 us, from 2048 33 -> 42.  In small tiles
        // 256 x 4096 from 4096 products 62 -> 37 us, 1024 x 1024 from 1024 16 -> 20.
        if (units && (units <= 128 ? steps >= 16 : units * 2 <= full && steps >= (full > 512 ? 32 : 96))) {
            const int64_t most = steps / 8, want = full / units < most ? full / units : most;
            p.part_steps = (steps + want - 1) / want;
            p.splits = (int)((steps + p.part_steps - 1) / p.part_steps);
        }
    }
    const int64_t parts = p.splits > 1 ? aligned(p.splits * p.out_batches * p.M * p.N * 4) : 0;
    if (p.pack_a >= 0) p.pack_a += parts;
    if (p.pack_b >= 0) p.pack_b += parts;
    return parts + packed;
}
