// Log probabilities of given ids with entropy and alternatives, and their gradient (the formulas are at
// ssmap_log_probs and ssmap_log_probs_grad in ssmap.h).
//
// With c = log2(e) / T and m the largest logit of a position, t_j = (x_j - m) c and e_j = 2^t_j:
//   S = sum e_j, W = sum e_j t_j,   log p_j = ln2 (t_j - log2 S),   entropy = ln2 (log2 S - W / S).
// Both terms of the entropy are sums of one sign: nothing cancels.  Differences to the maximum are taken
// before scaling, so logits at the type's lowest value or near overflow need no special case; only a
// position of nothing but -inf has no maximum, and takes 0 for it (every e_j is then 2^-inf = 0).
// A NaN or +inf makes S NaN: +inf - +inf is NaN.
#include <math.h>

#include "heads.h"

using namespace ssmap;

namespace {

constexpr int kThreads = 256;
constexpr float kLn2 = 0.693147180559945309f, kLog2e = 1.44269504088896341f;
constexpr float kTiny = -200.0f;   // 2^-200 is 0 in float: exponents are clamped to it where 0 * -inf would be NaN

struct Shape {
    int64_t batch, rows, classes;
    int64_t batch_stride, class_stride, row_stride;
    int64_t ids_batch_stride, ids_row_stride, ignore_id;
    int32_t ids_64, top, layout;
    float inv_t;       // 1 / T
    float scale;       // log2(e) / T
};

// One class as an alternative: larger logits first, the lower class first among equals.
struct Best {
    float v;
    int32_t i;
};
constexpr int32_t kNoId = 0x7FFFFFFF;
__device__ __forceinline__ bool better(const Best &a, const Best &b) { return a.v > b.v || (a.v == b.v && a.i < b.i); }

__device__ __forceinline__ int64_t load_id(const Shape &s, const void *ids, int64_t b, int64_t r) {
    const int64_t at = b * s.ids_batch_stride + r * s.ids_row_stride;
    return s.ids_64 ? static_cast<const int64_t *>(ids)[at] : (int64_t) static_cast<const int32_t *>(ids)[at];
}

struct Out {
    float *log_prob, *entropy, *row_max, *log_sum, *top_log_prob;
    int32_t *top_ids;
};

// Where alternative k of position (b, r) goes.
__device__ __forceinline__ int64_t top_at(const Shape &s, int64_t b, int64_t r, int k) {
    return s.layout == SSMAP_ROWS ? (b * s.rows + r) * s.top + k : (b * s.top + k) * s.rows + r;
}

// What a position's sums say.
struct Said {
    float log_prob, entropy, row_max, log_sum, log2_s;
    bool bad;
};
__device__ __forceinline__ Said say(const Shape &s, float m, float sum, float wsum, int64_t id, float xid) {
    const float nan = __builtin_nanf("");
    const bool bad = !(sum == sum), none = m == -INFINITY && !bad;
    const float log2_s = __log2f(sum);
    float given = (xid - m) * s.inv_t - kLn2 * log2_s;
    if (none) given = -INFINITY;
    if (bad || id < 0 || id >= s.classes) given = nan;
    if (id == s.ignore_id) given = 0.0f;
    return {given, bad ? nan : none ? 0.0f : kLn2 * (log2_s - wsum / sum), m, bad ? nan : none ? -INFINITY : kLn2 * log2_s, log2_s, bad};
}
__device__ __forceinline__ void put(const Out &o, int64_t pos, const Said &w) {
    o.log_prob[pos] = w.log_prob;
    o.entropy[pos] = w.entropy;
    o.row_max[pos] = w.row_max;
    o.log_sum[pos] = w.log_sum;
}

// An alternative's id and log probability.
__device__ __forceinline__ int32_t top_id(Best v, const Said &w) { return w.bad || !(v.v > -INFINITY) ? -1 : v.i; }
__device__ __forceinline__ float top_value(const Shape &s, Best v, const Said &w) {
    return w.bad ? __builtin_nanf("") : !(v.v > -INFINITY) ? -INFINITY : (v.v - w.row_max) * s.inv_t - kLn2 * w.log2_s;
}

__device__ __forceinline__ float wave_max(float v) {
    for (int d = 1; d < 64; d <<= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ Best wave_best(Best v) {
    for (int d = 1; d < 64; d <<= 1) {
        const Best w{__shfl_xor(v.v, d), __shfl_xor(v.i, d)};
        if (better(w, v)) v = w;
    }
    return v;
}

// One block per position, the classes read three times and once more for each alternative.
template <int DT>
__global__ __launch_bounds__(kThreads) void k_scores(Shape s, const elem_t<DT> *logits, const void *ids, Out o) {
    __shared__ float part[2][kThreads / 64];
    __shared__ Best best[kThreads / 64];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    for (int64_t pos = blockIdx.x; pos < s.batch * s.rows; pos += gridDim.x) {
        const int64_t b = pos / s.rows, r = pos % s.rows;
        const elem_t<DT> *row = logits + b * s.batch_stride + r * s.row_stride;
        float m = -INFINITY;
        for (int64_t j = tid; j < s.classes; j += kThreads) m = fmaxf(m, Elem<DT>::get(row[j * s.class_stride]));
        m = wave_max(m);
        __syncthreads();
        if (!lane) part[0][wave] = m;
        __syncthreads();
        for (int w = 0; w < kThreads / 64; ++w) m = fmaxf(m, part[0][w]);
        __syncthreads();
        const float ms = m == -INFINITY ? 0.0f : m;
        float sum = 0.0f, wsum = 0.0f;
        for (int64_t j = tid; j < s.classes; j += kThreads) {
            const float t = (Elem<DT>::get(row[j * s.class_stride]) - ms) * s.scale, e = __builtin_amdgcn_exp2f(t);
            sum += e;
            wsum += e * fmaxf(t, kTiny);
        }
        sum = wave_sum(sum);
        wsum = wave_sum(wsum);
        if (!lane) part[0][wave] = sum, part[1][wave] = wsum;
        __syncthreads();
        sum = wsum = 0.0f;
        for (int w = 0; w < kThreads / 64; ++w) sum += part[0][w], wsum += part[1][w];
        const int64_t id = load_id(s, ids, b, r);
        const float xid = id >= 0 && id < s.classes ? Elem<DT>::get(row[id * s.class_stride]) : 0.0f;
        const Said said = say(s, m, sum, wsum, id, xid);
        if (!tid) put(o, pos, said);
        Best last{INFINITY, -1};
        for (int k = 0; k < s.top; ++k) {
            Best mine{-INFINITY, kNoId};
            for (int64_t j = tid; j < s.classes; j += kThreads) {
                const Best v{Elem<DT>::get(row[j * s.class_stride]), (int32_t)j};
                if (better(last, v) && better(v, mine)) mine = v;
            }
            mine = wave_best(mine);
            __syncthreads();
            if (!lane) best[wave] = mine;
            __syncthreads();
            for (int w = 0; w < kThreads / 64; ++w)
                if (better(best[w], mine)) mine = best[w];
            if (!tid) {
                const int64_t at = top_at(s, b, r, k);
                o.top_ids[at] = top_id(mine, said);
                o.top_log_prob[at] = top_value(s, mine, said);
            }
            last = mine;
        }
        __syncthreads();
    }
}

// What is loaded at once: N neighbours at any element alignment.
template <int DT, int N>
struct Pack {
    elem_t<DT> v[N];
};
template <int DT, int N>
__device__ __forceinline__ Pack<DT, N> load_pack(const elem_t<DT> *p) {
    Pack<DT, N> r;
    __builtin_memcpy(&r, p, sizeof r);
    return r;
}
template <int DT, int N>
__device__ __forceinline__ void store_pack(elem_t<DT> *p, const Pack<DT, N> &r) { __builtin_memcpy(p, &r, sizeof r); }

// Sorted alternatives in registers: K values with their classes, `j` later than every class in the list, so
// an equal value goes behind.  slot q becomes the middle of (slot q-1, slot q, v).
template <int K>
__device__ __forceinline__ void insert(float (&v)[K], int32_t (&i)[K], float x, int32_t j) {
    bool above[K];   // x goes in front of slot q
#pragma unroll
    for (int q = 0; q < K; ++q) above[q] = x > v[q];
#pragma unroll
    for (int q = K - 1; q > 0; --q) {
        i[q] = above[q - 1] ? i[q - 1] : above[q] ? j : i[q];
        v[q] = above[q - 1] ? v[q - 1] : above[q] ? x : v[q];
    }
    i[0] = above[0] ? j : i[0];
    v[0] = above[0] ? x : v[0];
}

constexpr int kPlaneClasses = 8;   // classes a plane kernel holds in flight

// Planes: a thread walks the classes of PX neighbouring positions once, kPlaneClasses at a time: their
// maximum first, so the running sums are rescaled once per step and not once per class.  K >= s.top.
template <int DT, int PX, int K>
__global__ __launch_bounds__(kThreads) void k_scores_planes(Shape s, const elem_t<DT> *logits, const void *ids, Out o) {
    const int64_t groups = (s.rows + PX - 1) / PX;
    const int64_t at = blockIdx.x * (int64_t)kThreads + threadIdx.x;
    if (at >= s.batch * groups) return;
    const int64_t b = at / groups, r0 = at % groups * PX;
    const bool full = r0 + PX <= s.rows;
    const elem_t<DT> *base = logits + b * s.batch_stride + r0;
    float m[PX], sum[PX], wsum[PX], xid[PX], tv[PX][K ? K : 1];
    int32_t ti[PX][K ? K : 1], id32[PX];
    int64_t id[PX];
#pragma unroll
    for (int q = 0; q < PX; ++q) {
        // the given class is picked up on the way: fetched afterwards, its line would come from memory again
        id[q] = load_id(s, ids, b, r0 + q < s.rows ? r0 + q : r0);
        id32[q] = id[q] >= 0 && id[q] < s.classes ? (int32_t)id[q] : -1;
        xid[q] = 0.0f;
        m[q] = -INFINITY;
        sum[q] = wsum[q] = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) tv[q][k] = -INFINITY, ti[q][k] = kNoId;
    }
    for (int64_t c0 = 0; c0 < s.classes; c0 += kPlaneClasses) {
        float x[kPlaneClasses][PX];
#pragma unroll
        for (int u = 0; u < kPlaneClasses; ++u) {
            const int64_t c = c0 + u;
            if (c < s.classes && full) {
                const Pack<DT, PX> v = load_pack<DT, PX>(base + c * s.class_stride);
#pragma unroll
                for (int q = 0; q < PX; ++q) x[u][q] = Elem<DT>::get(v.v[q]);
            } else {
#pragma unroll
                for (int q = 0; q < PX; ++q) x[u][q] = c < s.classes && r0 + q < s.rows ? Elem<DT>::get(base[c * s.class_stride + q]) : -INFINITY;
            }
        }
#pragma unroll
        for (int q = 0; q < PX; ++q) {
            float mn = m[q];
#pragma unroll
            for (int u = 0; u < kPlaneClasses; ++u) mn = fmaxf(mn, x[u][q]);
            const float ms = mn == -INFINITY ? 0.0f : mn;
            const float d = fmaxf((m[q] - ms) * s.scale, kTiny), a = __builtin_amdgcn_exp2f(d);
            wsum[q] = a * (wsum[q] + sum[q] * d);
            sum[q] *= a;
            m[q] = mn;
#pragma unroll
            for (int u = 0; u < kPlaneClasses; ++u) {
                const float t = (x[u][q] - ms) * s.scale, e = __builtin_amdgcn_exp2f(t);
                sum[q] += e;
                wsum[q] += e * fmaxf(t, kTiny);
                xid[q] = id32[q] == (int32_t)(c0 + u) ? x[u][q] : xid[q];
                if constexpr (K > 0) insert<K>(tv[q], ti[q], x[u][q], (int32_t)(c0 + u));
            }
        }
    }
    Said said[PX];
#pragma unroll
    for (int q = 0; q < PX; ++q) said[q] = say(s, m[q], sum[q], wsum[q], id[q], xid[q]);
    const auto put_row = [&](auto *to, auto value) {   // PX neighbours of one output plane
        using V = decltype(value(0));
        V v[PX];
#pragma unroll
        for (int q = 0; q < PX; ++q) v[q] = value(q);
        if (full) {
            __builtin_memcpy(to, v, sizeof v);
        } else {
#pragma unroll
            for (int q = 0; q < PX; ++q)
                if (r0 + q < s.rows) to[q] = v[q];
        }
    };
    const int64_t pos = b * s.rows + r0;
    put_row(o.log_prob + pos, [&](int q) { return said[q].log_prob; });
    put_row(o.entropy + pos, [&](int q) { return said[q].entropy; });
    put_row(o.row_max + pos, [&](int q) { return said[q].row_max; });
    put_row(o.log_sum + pos, [&](int q) { return said[q].log_sum; });
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (k < s.top) {
            put_row(o.top_ids + top_at(s, b, r0, k), [&](int q) { return top_id(Best{tv[q][k], ti[q][k]}, said[q]); });
            put_row(o.top_log_prob + top_at(s, b, r0, k), [&](int q) { return top_value(s, Best{tv[q][k], ti[q][k]}, said[q]); });
        }
}

struct Grads {
    const float *row_max, *log_sum, *entropy, *g_log_prob, *g_entropy, *g_top;
    const int32_t *top_ids;
};

// One block per position.
template <int DT>
__global__ __launch_bounds__(kThreads) void k_scores_grad(Shape s, const elem_t<DT> *logits, const void *ids, Grads g, elem_t<DT> *grad) {
    for (int64_t pos = blockIdx.x; pos < s.batch * s.rows; pos += gridDim.x) {
        const int64_t b = pos / s.rows, r = pos % s.rows;
        const elem_t<DT> *row = logits + b * s.batch_stride + r * s.row_stride;
        elem_t<DT> *out = s.layout == SSMAP_ROWS ? grad + pos * s.classes : grad + b * s.classes * s.rows + r;
        const int64_t out_stride = s.layout == SSMAP_ROWS ? 1 : s.rows;
        const int64_t id = load_id(s, ids, b, r);
        const float m = g.row_max[pos], log2_s = g.log_sum[pos] * kLog2e;
        const bool none = m == -INFINITY;
        float g_l = g.g_log_prob && id != s.ignore_id ? g.g_log_prob[pos] : 0.0f;
        const bool bad = g.log_sum[pos] != g.log_sum[pos] || (g.g_log_prob && id != s.ignore_id && (id < 0 || id >= s.classes));
        const float g_e = g.g_entropy ? g.g_entropy[pos] : 0.0f, h = g.g_entropy ? g.entropy[pos] : 0.0f;
        float all = g_l;
        const int top = g.g_top ? s.top : 0;
        for (int k = 0; k < top; ++k) {
            const int64_t at = top_at(s, b, r, k);
            all += g.top_ids[at] >= 0 ? g.g_top[at] : 0.0f;
        }
        for (int64_t j = threadIdx.x; j < s.classes; j += kThreads) {
            float d = 0.0f;
            if (!none) {
                const float t = (Elem<DT>::get(row[j * s.class_stride]) - m) * s.scale - log2_s;
                const float p = __builtin_amdgcn_exp2f(t);
                d = -p * (all + g_e * (kLn2 * fmaxf(t, kTiny) + h));
                if (j == id) d += g_l;
                for (int k = 0; k < top; ++k) {
                    const int64_t at = top_at(s, b, r, k);
                    if (g.top_ids[at] == j) d += g.g_top[at];
                }
            }
            if (bad) d = __builtin_nanf("");
            out[j * out_stride] = Elem<DT>::put(d * s.inv_t);
        }
    }
}

// Planes: a thread walks the classes of PX neighbouring positions.  K >= s.top.
template <int DT, int PX, int K>
__global__ __launch_bounds__(kThreads) void k_grad_planes(Shape s, const elem_t<DT> *logits, const void *ids, Grads g, elem_t<DT> *grad) {
    const int64_t groups = (s.rows + PX - 1) / PX;
    const int64_t at = blockIdx.x * (int64_t)kThreads + threadIdx.x;
    if (at >= s.batch * groups) return;
    const int64_t b = at / groups, r0 = at % groups * PX;
    const bool full = r0 + PX <= s.rows;
    const elem_t<DT> *base = logits + b * s.batch_stride + r0;
    elem_t<DT> *out = grad + b * s.classes * s.rows + r0;
    const bool tops = K > 0 && g.g_top;
    // d = p (A + B t) / T, t = log2 p, and the given class and the alternatives add theirs
    float m[PX], off[PX], A[PX], B[PX], gl[PX], gt[PX][K ? K : 1];
    int32_t id[PX], ti[PX][K ? K : 1];
#pragma unroll
    for (int q = 0; q < PX; ++q) {
        const bool in = r0 + q < s.rows;
        const int64_t r = in ? r0 + q : r0, pos = b * s.rows + r;
        const int64_t want = load_id(s, ids, b, r);
        const float log_sum = g.log_sum[pos];
        m[q] = g.row_max[pos];
        off[q] = log_sum * kLog2e;
        const bool none = m[q] == -INFINITY, given = g.g_log_prob && want != s.ignore_id, inside = want >= 0 && want < s.classes;
        const bool bad = log_sum != log_sum || (given && !inside);
        gl[q] = given ? g.g_log_prob[pos] : 0.0f;
        id[q] = given && inside ? (int32_t)want : -1;
        float all = gl[q];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int64_t tat = (b * s.top + k) * s.rows + r;
            const bool on = tops && k < s.top;
            ti[q][k] = on ? g.top_ids[tat] : -1;
            gt[q][k] = on && ti[q][k] >= 0 ? g.g_top[tat] : 0.0f;
            all += gt[q][k];
        }
        const float ge = g.g_entropy ? g.g_entropy[pos] : 0.0f, h = g.g_entropy ? g.entropy[pos] : 0.0f;
        A[q] = -(all + ge * h) * s.inv_t;
        B[q] = -ge * kLn2 * s.inv_t;
        gl[q] *= s.inv_t;
#pragma unroll
        for (int k = 0; k < K; ++k) gt[q][k] *= s.inv_t;
        if (none) {   // every t is -inf and every p 0
            m[q] = off[q] = A[q] = B[q] = gl[q] = 0.0f;
            id[q] = -1;
#pragma unroll
            for (int k = 0; k < K; ++k) ti[q][k] = -1;
        }
        if (bad) A[q] = __builtin_nanf("");
    }
#pragma unroll 4
    for (int64_t c = 0; c < s.classes; ++c) {
        float x[PX];
        if (full) {
            const Pack<DT, PX> v = load_pack<DT, PX>(base + c * s.class_stride);
#pragma unroll
            for (int q = 0; q < PX; ++q) x[q] = Elem<DT>::get(v.v[q]);
        } else {
#pragma unroll
            for (int q = 0; q < PX; ++q) x[q] = r0 + q < s.rows ? Elem<DT>::get(base[c * s.class_stride + q]) : 0.0f;
        }
        Pack<DT, PX> w;
#pragma unroll
        for (int q = 0; q < PX; ++q) {
            const float t = (x[q] - m[q]) * s.scale - off[q], p = __builtin_amdgcn_exp2f(t);
            float d = p * (A[q] + B[q] * fmaxf(t, kTiny));
            d += id[q] == (int32_t)c ? gl[q] : 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k) d += ti[q][k] == (int32_t)c ? gt[q][k] : 0.0f;
            w.v[q] = Elem<DT>::put(d);
        }
        if (full) {
            store_pack<DT, PX>(out + c * s.rows, w);
        } else {
#pragma unroll
            for (int q = 0; q < PX; ++q)
                if (r0 + q < s.rows) out[c * s.rows + q] = w.v[q];
        }
    }
}

template <typename Args>
int check(const Args *a, Shape &s) {
    if (!head_dtype_ok(a->dtype)) return head_error(SSMAP_ERR_INVALID_ARG, "dtype is none of SSMAP_F32, SSMAP_BF16, SSMAP_F16");
    if (a->layout != SSMAP_ROWS && a->layout != SSMAP_PLANES)
        return head_error(SSMAP_ERR_INVALID_ARG, "layout is neither SSMAP_ROWS nor SSMAP_PLANES");
    if (!head_sizes_ok(a->batch, a->rows, a->classes) || a->classes < 1 || a->classes > INT32_MAX - 1)
        return head_error(SSMAP_ERR_INVALID_ARG, "batch, rows >= 0, 1 <= classes < 2^31 - 1 and fewer than 2^40 logits are required");
    if (a->batch * a->rows > INT32_MAX) return head_error(SSMAP_ERR_UNSUPPORTED, "more than 2^31 - 1 positions");
    if (a->top < 0 || a->top > SSMAP_MAX_TOP || a->top > a->classes)
        return head_error(SSMAP_ERR_INVALID_ARG, "top must be in [0, min(32, classes)]");
    if (!(a->temperature >= 1e-30f && a->temperature <= 1e30f))
        return head_error(SSMAP_ERR_INVALID_ARG, "temperature must be in [1e-30, 1e30]");
    s.batch = a->batch; s.rows = a->rows; s.classes = a->classes;
    s.batch_stride = a->batch_stride;
    s.class_stride = a->layout == SSMAP_ROWS ? 1 : a->inner_stride;
    s.row_stride = a->layout == SSMAP_ROWS ? a->inner_stride : 1;
    s.ids_batch_stride = a->ids_batch_stride; s.ids_row_stride = a->ids_row_stride;
    s.ignore_id = a->ignore_id; s.ids_64 = a->ids_64; s.top = a->top; s.layout = a->layout;
    s.inv_t = (float)(1.0 / (double)a->temperature);
    s.scale = (float)(1.4426950408889634074 / (double)a->temperature);
    return SSMAP_OK;
}

// The smallest compiled list that holds `top` alternatives; longer lists hold fewer positions a thread.
template <int DT, typename F>
void with_list(int top, F f) {
    constexpr int PX = 4;
    if (top == 0) f(std::integral_constant<int, PX>{}, std::integral_constant<int, 0>{});
    else if (top == 1) f(std::integral_constant<int, PX>{}, std::integral_constant<int, 1>{});
    else if (top == 2) f(std::integral_constant<int, PX>{}, std::integral_constant<int, 2>{});
    else if (top == 3) f(std::integral_constant<int, PX>{}, std::integral_constant<int, 3>{});
    else if (top <= 5) f(std::integral_constant<int, 2>{}, std::integral_constant<int, 5>{});
    else if (top <= 10) f(std::integral_constant<int, 1>{}, std::integral_constant<int, 10>{});
    else f(std::integral_constant<int, 1>{}, std::integral_constant<int, SSMAP_MAX_TOP>{});
}

inline unsigned thread_blocks(int64_t batch, int64_t rows, int px) {
    return (unsigned)((batch * ((rows + px - 1) / px) + kThreads - 1) / kThreads);
}

template <int DT>
void launch_scores(const Shape &s, const ssmap_log_probs_args &a, hipStream_t st) {
    const Out o{a.log_prob, a.entropy, a.row_max, a.log_sum, a.top_log_prob, a.top_ids};
    const auto *x = static_cast<const elem_t<DT> *>(a.logits);
    if (s.layout == SSMAP_PLANES) {
        with_list<DT>(s.top, [&](auto px, auto k) {
            k_scores_planes<DT, px.value, k.value><<<thread_blocks(s.batch, s.rows, px.value), kThreads, 0, st>>>(s, x, a.ids, o);
        });
        return;
    }
    const int64_t n = s.batch * s.rows;
    k_scores<DT><<<dim3((unsigned)(n < (1 << 20) ? n : (1 << 20))), kThreads, 0, st>>>(s, x, a.ids, o);
}

template <int DT>
void launch_grad(const Shape &s, const ssmap_log_probs_grad_args &a, hipStream_t st) {
    const Grads g{a.row_max, a.log_sum, a.entropy, a.g_log_prob, a.g_entropy, a.g_top, a.top_ids};
    const auto *x = static_cast<const elem_t<DT> *>(a.logits);
    auto *out = static_cast<elem_t<DT> *>(a.grad);
    if (s.layout == SSMAP_PLANES) {
        with_list<DT>(a.g_top ? s.top : 0, [&](auto px, auto k) {
            k_grad_planes<DT, px.value, k.value><<<thread_blocks(s.batch, s.rows, px.value), kThreads, 0, st>>>(s, x, a.ids, g, out);
        });
        return;
    }
    const int64_t n = s.batch * s.rows;
    k_scores_grad<DT><<<dim3((unsigned)(n < (1 << 20) ? n : (1 << 20))), kThreads, 0, st>>>(s, x, a.ids, g, out);
}

}  // namespace

extern "C" {

int64_t ssmap_log_probs_workspace(const ssmap_log_probs_args *a) {
    Shape s{};
    if (!a) { head_error(SSMAP_ERR_INVALID_ARG, "null argument"); return -1; }
    return check(a, s) == SSMAP_OK ? 0 : -1;
}

int ssmap_log_probs(const ssmap_log_probs_args *a, void *stream) {
    if (!a) return head_error(SSMAP_ERR_INVALID_ARG, "null argument");
    Shape s{};
    if (int rc = check(a, s)) return rc;
    if (s.batch * s.rows == 0) return SSMAP_OK;
    if (!a->logits || !a->ids || !a->log_prob || !a->entropy || !a->row_max || !a->log_sum || (a->top && (!a->top_ids || !a->top_log_prob)))
        return head_error(SSMAP_ERR_INVALID_ARG, "null argument");
    if (a->workspace_bytes < ssmap_log_probs_workspace(a)) return head_error(SSMAP_ERR_INVALID_ARG, "the workspace is smaller than ssmap_log_probs_workspace says");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->dtype == SSMAP_F32) launch_scores<SSMAP_F32>(s, *a, st);
    else if (a->dtype == SSMAP_BF16) launch_scores<SSMAP_BF16>(s, *a, st);
    else launch_scores<SSMAP_F16>(s, *a, st);
    return head_launch_error(hipGetLastError());
}

int ssmap_log_probs_grad(const ssmap_log_probs_grad_args *a, void *stream) {
    if (!a) return head_error(SSMAP_ERR_INVALID_ARG, "null argument");
    Shape s{};
    if (int rc = check(a, s)) return rc;
    if (s.batch * s.rows == 0) return SSMAP_OK;
    if (!a->logits || !a->ids || !a->row_max || !a->log_sum || !a->grad || (a->g_entropy && !a->entropy) || (a->g_top && a->top && !a->top_ids))
        return head_error(SSMAP_ERR_INVALID_ARG, "null argument");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->dtype == SSMAP_F32) launch_grad<SSMAP_F32>(s, *a, st);
    else if (a->dtype == SSMAP_BF16) launch_grad<SSMAP_BF16>(s, *a, st);
    else launch_grad<SSMAP_F16>(s, *a, st);
    return head_launch_error(hipGetLastError());
}

}  // extern "C"
