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
constexpr int64_t kMostBlocks = 1 << 22;   // a grid holds fewer than 2^32 threads; kernels loop over what is beyond
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

// The same order as one number: larger is better.  0 is no class.  -0 becomes 0: equal logits, equal values.
using Key = unsigned long long;
__device__ __forceinline__ Key key_of(float v, int32_t i) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);
    return (Key)(b ^ (b >> 31 ? 0xFFFFFFFFu : 0x80000000u)) << 32 | (uint32_t)~i;
}
__device__ __forceinline__ Best best_of(Key k) {
    const uint32_t b = (uint32_t)(k >> 32);
    return k ? Best{__builtin_bit_cast(float, b ^ (b >> 31 ? 0x80000000u : 0xFFFFFFFFu)), (int32_t)~(uint32_t)k} : Best{-INFINITY, kNoId};
}

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
__device__ __forceinline__ Said say(const Shape &s, float m, float sum, float wsum, bool ignored, bool inside, float xid) {
    const float nan = __builtin_nanf("");
    const bool bad = !(sum == sum), none = m == -INFINITY && !bad;
    const float log2_s = __log2f(sum);
    float given = (xid - m) * s.inv_t - kLn2 * log2_s;
    if (none) given = -INFINITY;
    if (bad || !inside) given = nan;
    if (ignored) given = 0.0f;
    return {given, bad ? nan : none ? 0.0f : kLn2 * (log2_s - wsum / sum), m, bad ? nan : none ? -INFINITY : kLn2 * log2_s, log2_s, bad};
}
__device__ __forceinline__ Said say(const Shape &s, float m, float sum, float wsum, int64_t id, float xid) {
    return say(s, m, sum, wsum, id == s.ignore_id, id >= 0 && id < s.classes, xid);
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

// The pack at class j of a row, of which classes from ... to - 1 may be read; -inf for the others.  Kept in
// memory's type: a conversion next to the load would wait for it, and with it every later load.
template <int DT, int N>
__device__ __forceinline__ Pack<DT, N> fetch_pack(const elem_t<DT> *row, int j, int from, int to) {
    if (j >= from && j + N <= to) return load_pack<DT, N>(row + j);
    Pack<DT, N> r;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        r.v[e] = Elem<DT>::put(-INFINITY);
        if (j + e >= from && j + e < to) r.v[e] = row[j + e];
    }
    return r;
}

// Running sums of a set of classes relative to its own maximum.
struct Sums {
    float m, sum, wsum;
};
__device__ __forceinline__ Sums join(const Shape &s, const Sums &a, const Sums &b) {
    const float m = fmaxf(a.m, b.m), ms = m == -INFINITY ? 0.0f : m;
    const float da = fmaxf((a.m - ms) * s.scale, kTiny), db = fmaxf((b.m - ms) * s.scale, kTiny);
    const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
    return {m, fa * a.sum + fb * b.sum, fa * (a.wsum + a.sum * da) + fb * (b.wsum + b.sum * db)};
}
// All lanes of a group of 16 (a DPP row) or of a wave get the result; the exchanges are symmetric, so every
// lane computes the same bits.
template <int N>
__device__ __forceinline__ float ror(float v) {   // rotated by N lanes within 16
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + N, 0xf, 0xf, false));
}
template <int N>
__device__ __forceinline__ int32_t ror(int32_t v) { return __builtin_amdgcn_update_dpp(0, v, 0x120 + N, 0xf, 0xf, false); }
template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
    v = fmaxf(v, ror<8>(v)); v = fmaxf(v, ror<4>(v)); v = fmaxf(v, ror<2>(v)); v = fmaxf(v, ror<1>(v));
    if constexpr (LANES == 64) v = fmaxf(v, __shfl_xor(v, 16)), v = fmaxf(v, __shfl_xor(v, 32));
    return v;
}
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
    v += ror<8>(v); v += ror<4>(v); v += ror<2>(v); v += ror<1>(v);
    if constexpr (LANES == 64) v += __shfl_xor(v, 16), v += __shfl_xor(v, 32);
    return v;
}
template <int LANES>
__device__ __forceinline__ int32_t lanes_min(int32_t v) {
    v = min(v, ror<8>(v)); v = min(v, ror<4>(v)); v = min(v, ror<2>(v)); v = min(v, ror<1>(v));
    if constexpr (LANES == 64) v = min(v, __shfl_xor(v, 16)), v = min(v, __shfl_xor(v, 32));
    return v;
}
template <int LANES>
__device__ __forceinline__ Sums lanes_join(const Shape &s, Sums v) {
    const float m = lanes_max<LANES>(v.m);
    const float ms = m == -INFINITY ? 0.0f : m, dv = fmaxf((v.m - ms) * s.scale, kTiny), f = __builtin_amdgcn_exp2f(dv);
    return {m, lanes_sum<LANES>(f * v.sum), lanes_sum<LANES>(f * (v.wsum + v.sum * dv))};
}

constexpr int kShortBlocks = 256 * 6;   // as many as are resident at once: each block loops over rows

// Short rows: LPR lanes hold a row in registers (NP packs a lane), so the maximum is known before the sums
// and each alternative is found by one more look at the registers.  65536 x 150 float32 with two alternatives
// takes 18 us (the bytes alone 8): few loads a row, so their latency counts.
template <int DT, int LPR, int NP>
__global__ __launch_bounds__(kThreads) void k_scores_short(Shape s, const elem_t<DT> *logits, const void *ids, Out o) {
    constexpr int VEC = 16 / sizeof(elem_t<DT>), UNITS = kThreads / LPR;
    const int sub = threadIdx.x % LPR;
    const int64_t n = s.batch * s.rows, stride = (int64_t)gridDim.x * UNITS;
    const auto place = [&](int64_t first, int64_t &b, int64_t &r) {   // lanes behind the last row take that one again
        const int64_t mine = first + threadIdx.x / LPR, pos = mine < n ? mine : n - 1;
        b = pos / s.rows, r = pos % s.rows;
        return pos;
    };
    const auto fetch = [&](int64_t b, int64_t r, Pack<DT, VEC> (&in)[NP], int64_t &id) {
        const elem_t<DT> *row = logits + b * s.batch_stride + r * s.row_stride;
        id = load_id(s, ids, b, r);
#pragma unroll
        for (int u = 0; u < NP; ++u) in[u] = fetch_pack<DT, VEC>(row, (u * LPR + sub) * VEC, 0, (int)s.classes);
    };
    Pack<DT, VEC> in[NP], next[NP];
    int64_t b, r, id, b2, r2, id2 = 0, pos = place(blockIdx.x * (int64_t)UNITS, b, r), pos2;
    fetch(b, r, in, id);
    // every lane stays in the loop as long as its block has a row: the exchanges below need all of a wave
    for (int64_t first = blockIdx.x * (int64_t)UNITS; first < n; first += stride) {
        const bool mine = first + threadIdx.x / LPR < n;
        const elem_t<DT> *row = logits + b * s.batch_stride + r * s.row_stride;
        const float xid = id >= 0 && id < s.classes ? Elem<DT>::get(row[id]) : 0.0f;
        pos2 = place(first + stride, b2, r2);
        if (first + stride < n) fetch(b2, r2, next, id2);   // the next row is under way while this one is worked on
        float x[NP][VEC];
        float m = -INFINITY;
#pragma unroll
        for (int u = 0; u < NP; ++u)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                x[u][e] = Elem<DT>::get(in[u].v[e]);
                m = fmaxf(m, x[u][e]);
            }
        m = lanes_max<LPR>(m);
        const float ms = m == -INFINITY ? 0.0f : m;
        float sum = 0.0f, wsum = 0.0f;
#pragma unroll
        for (int u = 0; u < NP; ++u)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float t = (x[u][e] - ms) * s.scale, p = __builtin_amdgcn_exp2f(t);
                sum += p;
                wsum += p * fmaxf(t, kTiny);
            }
        sum = lanes_sum<LPR>(sum);
        wsum = lanes_sum<LPR>(wsum);
        const Said said = say(s, m, sum, wsum, id, xid);
        const bool writes = sub == 0 && mine;
        if (writes) put(o, pos, said);
        Best last{INFINITY, -1};
        for (int k = 0; k < s.top; ++k) {
            Best best{-INFINITY, kNoId};
#pragma unroll
            for (int u = 0; u < NP; ++u)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {   // the lane's classes ascend: an equal value never replaces
                    const Best v{x[u][e], (int32_t)((u * LPR + sub) * VEC + e)};
                    if (better(last, v) && v.v > best.v) best = v;
                }
            const float bv = lanes_max<LPR>(best.v);
            best = Best{bv, lanes_min<LPR>(best.v == bv ? best.i : kNoId)};
            if (writes) {
                o.top_ids[pos * s.top + k] = top_id(best, said);
                o.top_log_prob[pos * s.top + k] = top_value(s, best, said);
            }
            last = best;
        }
        b = b2, r = r2, id = id2, pos = pos2;
#pragma unroll
        for (int u = 0; u < NP; ++u) in[u] = next[u];
    }
}

constexpr int kLongPacks = 2;               // packs a thread of a long row has in flight: one step
constexpr int kSteps = 16;                  // what a thread remembers the maxima of
constexpr int kGathered = 1024;             // logits looked at again in one go
constexpr int kCandidates = kGathered + SSMAP_MAX_TOP;

// A block's alternatives: candidates in any order (their keys differ, so the order of the atomics does not
// matter), ranked by counting.  The counting loops read eight keys before they compare: one at a time, each
// comparison would wait for its own read.
struct Candidates {
    Key list[kCandidates];
    Key kept[SSMAP_MAX_TOP];
    int count;
};
__device__ __forceinline__ void offer(Candidates &c, Key k) { c.list[atomicAdd(&c.count, 1)] = k; }
__device__ __forceinline__ int count_above(const Key *list, int n, Key mine) {
    int rank = 0, q = 0;
    for (; q + 8 <= n; q += 8) {
        Key k[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) k[e] = list[q + e];
#pragma unroll
        for (int e = 0; e < 8; ++e) rank += k[e] > mine;
    }
    for (; q < n; ++q) rank += list[q] > mine;
    return rank;
}
// The best `top` of the list into kept[], in order; all threads call it.
__device__ __forceinline__ void rank_candidates(Candidates &c, int top) {
    __syncthreads();
    const int n = c.count;
    if (threadIdx.x < top) c.kept[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const Key v = c.list[i];
        const int rank = count_above(c.list, n, v);
        if (rank < top) c.kept[rank] = v;
    }
    __syncthreads();
}

struct Part {       // what a segment of a split row says, followed by `top` alternatives
    Sums sums;
    float pad;
};

// Long rows: a block takes one segment of a row, in one pass over memory.  Packs lie at addresses that are
// multiples of 16 whatever the row's start (loads that straddle such addresses cost 14 of 78 us at 4096 x
// 32003 fp16); the first and last are masked.  Each thread keeps running sums of its packs (rescaled once a
// pack), where its largest logit first stood, and the upper 16 bits of the maxima of up to kSteps stretches.
//
// Alternatives: the `top` threads with the best maxima hold them all.  Any other thread's logits are beaten by
// those `top` maxima: by value first; among equal ones the thread whose pack comes first wins, and its pack
// lies in front of the other's.  The threshold that `top` of the 256 keys pass is found bit by bit with
// ballots, every wave by itself (counting for each key the keys above it kept the LDS busy for 10 us of 78).
// Of the chosen threads only the stretches whose maximum reaches the threshold are read again, from the
// caches, and only logits that reach it become candidates.  4096 x 32003 fp16 with five alternatives takes 62 us
// (the bytes 51), 2048 x 131072 bf16 with twenty 110 us (104).
template <int DT>
__global__ __launch_bounds__(kThreads, 8) void k_scores_long(Shape s, const elem_t<DT> *logits, const void *ids, Out o, int splits,
                                                             int64_t segment, char *parts, int64_t part_bytes) {
    constexpr int VEC = 16 / sizeof(elem_t<DT>), U = kLongPacks, STEP = kThreads * VEC;
    __shared__ Sums joint[kThreads / 64];
    __shared__ Key firsts[kThreads];
    __shared__ uint16_t steps[kSteps][kThreads], items[kSteps * SSMAP_MAX_TOP];
    __shared__ int n_chosen, n_items;
    __shared__ uint8_t chosen[SSMAP_MAX_TOP];
    __shared__ Candidates cand;
    const int tid = threadIdx.x;
    for (int64_t unit = blockIdx.x; unit < s.batch * s.rows * splits; unit += gridDim.x) {
        const int64_t pos = unit / splits, b = pos / s.rows, r = pos % s.rows;
        const int from = (int)(unit % splits * segment), to = (int)(from + segment < s.classes ? from + segment : s.classes);   // classes <= 2^30
        const elem_t<DT> *row = logits + b * s.batch_stride + r * s.row_stride;
        const int lo = from - (int)(reinterpret_cast<uintptr_t>(row + from) % 16 / sizeof(elem_t<DT>));
        int64_t id = 0;
        float xid = 0.0f;
        if (splits == 1) {   // on their way during the pass
            id = load_id(s, ids, b, r);
            if (id >= 0 && id < s.classes) xid = Elem<DT>::get(row[id]);
        }
        const int n_steps = (to - lo + U * STEP - 1) / (U * STEP), per = (n_steps + kSteps - 1) / kSteps;
        Sums v{-INFINITY, 0.0f, 0.0f};
        float first_v = -INFINITY, stretch = -INFINITY;
        int first_j = from + tid * VEC;
        const auto take = [&](const Pack<DT, VEC> &in, int j) {
            float x[VEC], pm = -INFINITY;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                x[e] = Elem<DT>::get(in.v[e]);
                pm = fmaxf(pm, x[e]);
            }
            if (pm > first_v) first_v = pm, first_j = j > from ? j : from;
            stretch = fmaxf(stretch, pm);
            const float m = fmaxf(v.m, pm), ms = m == -INFINITY ? 0.0f : m;
            const float d = fmaxf((v.m - ms) * s.scale, kTiny), f = __builtin_amdgcn_exp2f(d);
            v.wsum = f * (v.wsum + v.sum * d);
            v.sum *= f;
            v.m = m;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float t = (x[e] - ms) * s.scale, p = __builtin_amdgcn_exp2f(t);
                v.sum += p;
                v.wsum += p * fmaxf(t, kTiny);
            }
        };
        for (int step = 0; step < n_steps; ++step) {
            const int j0 = lo + step * (U * STEP), j = j0 + tid * VEC;
            Pack<DT, VEC> in[U];
            if ((step || lo == from) && j0 + U * STEP <= to) {
#pragma unroll
                for (int u = 0; u < U; ++u) in[u] = load_pack<DT, VEC>(row + j + u * STEP);
            } else {
#pragma unroll
                for (int u = 0; u < U; ++u) in[u] = fetch_pack<DT, VEC>(row, j + u * STEP, from, to);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) take(in[u], j + u * STEP);
            if (s.top && (step + 1) % per == 0) steps[step / per][tid] = (uint16_t)(key_of(stretch, 0) >> 48), stretch = -INFINITY;
        }
        if (s.top && n_steps % per) steps[n_steps / per][tid] = (uint16_t)(key_of(stretch, 0) >> 48);
        v = lanes_join<64>(s, v);
        __syncthreads();
        if (tid % 64 == 0) joint[tid / 64] = v;
        const Key first = key_of(first_v, first_j);
        firsts[tid] = first;
        if (!tid) cand.count = n_chosen = n_items = 0;
        __syncthreads();
        v = joint[0];
#pragma unroll
        for (int w = 1; w < kThreads / 64; ++w) v = join(s, v, joint[w]);
        if (s.top) {
            Key all[kThreads / 64], least = 0;
#pragma unroll
            for (int q = 0; q < kThreads / 64; ++q) all[q] = firsts[q * 64 + tid % 64];
            for (int bit = 63; bit >= 0; --bit) {
                const Key t = least | (Key)1 << bit;
                int n = 0;
#pragma unroll
                for (int q = 0; q < kThreads / 64; ++q) n += __popcll(__ballot(all[q] >= t));
                if (n >= s.top) least = t;
                if (n == s.top) break;
            }
            if (first >= least) chosen[atomicAdd(&n_chosen, 1)] = (uint8_t)tid;   // exactly `top` threads
            __syncthreads();
            for (int i = tid; i < s.top * kSteps; i += kThreads) {
                const int th = chosen[i / kSteps], st = i % kSteps;
                if (st * per < n_steps && steps[st][th] >= (uint16_t)(least >> 48)) items[atomicAdd(&n_items, 1)] = (uint16_t)(st * kThreads + th);
            }
            __syncthreads();
            const int packs = per * U, all_packs = n_items * packs;
            for (int p0 = 0; p0 < all_packs; p0 += kGathered / VEC) {
                const int have = cand.count;
                __syncthreads();   // nobody offers before everybody has read the count
                if (have > kCandidates - kGathered) {
                    rank_candidates(cand, s.top);
                    if (tid < s.top) cand.list[tid] = cand.kept[tid];
                    if (!tid) cand.count = s.top;
                    __syncthreads();
                }
                const int p = p0 + tid;
                if (tid < kGathered / VEC && p < all_packs) {
                    const int item = items[p / packs];
                    const int j = lo + ((item / kThreads * packs + p % packs) * kThreads + item % kThreads) * VEC;
                    const Pack<DT, VEC> in = fetch_pack<DT, VEC>(row, j, from, to);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {   // a thread's key stands at its pack's start
                        const float x = Elem<DT>::get(in.v[e]);
                        const Key k = key_of(x, j + e);
                        if (x > -INFINITY && k + (VEC - 1) >= least) offer(cand, k);
                    }
                }
                __syncthreads();
            }
            rank_candidates(cand, s.top);
        }
        if (splits > 1) {
            char *part = parts + unit * part_bytes;
            if (!tid) reinterpret_cast<Part *>(part)->sums = v;
            if (tid < s.top) reinterpret_cast<Key *>(part + sizeof(Part))[tid] = cand.kept[tid];
        } else {
            const Said said = say(s, v.m, v.sum, v.wsum, id, xid);
            if (!tid) put(o, pos, said);
            if (tid < s.top) {
                const Best w = best_of(cand.kept[tid]);
                o.top_ids[pos * s.top + tid] = top_id(w, said);
                o.top_log_prob[pos * s.top + tid] = top_value(s, w, said);
            }
        }
    }
}

// Joins the segments of a split row: one block per row, at most kThreads segments.  The `top` segments with
// the best first alternatives hold all of the row's.
template <int DT>
__global__ __launch_bounds__(kThreads) void k_scores_join(Shape s, const elem_t<DT> *logits, const void *ids, Out o, int splits, const char *parts,
                                                          int64_t part_bytes) {
    __shared__ Sums joint[kThreads / 64];
    __shared__ Key firsts[kThreads], least;
    __shared__ Candidates cand;
    const int tid = threadIdx.x;
    for (int64_t pos = blockIdx.x; pos < s.batch * s.rows; pos += gridDim.x) {
        const int64_t b = pos / s.rows, r = pos % s.rows;
        const elem_t<DT> *row = logits + b * s.batch_stride + r * s.row_stride;
        const int64_t id = load_id(s, ids, b, r);
        const float xid = id >= 0 && id < s.classes ? Elem<DT>::get(row[id]) : 0.0f;
        const char *part = parts + (pos * splits + (tid < splits ? tid : 0)) * part_bytes;
        const Key *list = reinterpret_cast<const Key *>(part + sizeof(Part));
        Sums v{-INFINITY, 0.0f, 0.0f};
        Key first = 0;
        if (tid < splits) {
            v = reinterpret_cast<const Part *>(part)->sums;
            if (s.top) first = list[0];
        }
        v = lanes_join<64>(s, v);
        __syncthreads();
        if (tid % 64 == 0) joint[tid / 64] = v;
        firsts[tid] = first;
        if (!tid) cand.count = 0, least = 0;
        __syncthreads();
        v = joint[0];
#pragma unroll
        for (int w = 1; w < kThreads / 64; ++w) v = join(s, v, joint[w]);
        if (s.top) {
            const int rank = count_above(firsts, splits, first);
            if (first && rank == s.top - 1) least = first;
            __syncthreads();
            if (first && rank < s.top)
                for (int k = 0; k < s.top; ++k) {
                    const Key c = list[k];
                    if (!c || c < least) break;
                    offer(cand, c);
                }
            rank_candidates(cand, s.top);
        }
        const Said said = say(s, v.m, v.sum, v.wsum, id, xid);
        if (!tid) put(o, pos, said);
        if (tid < s.top) {
            const Best w = best_of(cand.kept[tid]);
            o.top_ids[pos * s.top + tid] = top_id(w, said);
            o.top_log_prob[pos * s.top + tid] = top_value(s, w, said);
        }
    }
}

// Segments of a long row: one where the rows alone fill the card (two blocks a CU), otherwise enough for
// four, each at least one pack a thread.  131072 bf16 classes with five alternatives, against half as many
// blocks and twice as many: 32 rows 19.0 us, 16.1 and 26.3; 128 rows 22.9, 22.9 and 26.5; 256 rows 29.0 and whole
// 32.5; 700 rows whole 45.1 and split 48.3.  Rows of a few thousand classes pay for the join: 511 x 5000 20.5 and
// whole 13.4.
struct Split {
    int splits;
    int64_t segment, part_bytes;
};
inline Split split_rows(const Shape &s, int dtype) {
    const int64_t n = s.batch * s.rows, step = kThreads * (16 / head_dtype_size(dtype));
    Split w{1, s.classes, (int64_t)(sizeof(Part) + s.top * sizeof(Key))};
    if (n == 0 || n >= 512 || s.classes <= step) return w;
    int64_t most = (s.classes + step - 1) / step;
    most = most < 1024 / n ? most : 1024 / n;
    most = most < kThreads ? most : kThreads;
    w.segment = ((s.classes + most - 1) / most + step - 1) / step * step;
    w.splits = (int)((s.classes + w.segment - 1) / w.segment);
    return w;
}

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

// sum += v, with what the addition rounds off taken along: sum - off is the sum.
__device__ __forceinline__ void add_aside(float &sum, float &off, float v) {
    const float y = v - off, to = sum + y;
    off = (to - sum) - y;
    sum = to;
}

constexpr int kPlaneClasses = 8;   // classes a plane kernel holds in flight

// Planes: a thread walks the classes of PX neighbouring positions once, kPlaneClasses at a time, whatever their number.
// So that many classes cost no bits, each step's terms are summed by themselves and added to the running sums with
// what the additions round off kept aside (true value: sum - sum_off); and the sums are rescaled only where a logit
// exceeds their reference by more than a factor of two in its exponential, so that what a rescaling rounds fades by
// half with the next.  K >= s.top.  Bound by memory: 16 x 40 x 480 x 640 float32 with three alternatives takes
// 205 us, 4.8 TB/s (fetching the given class afterwards and storing position by position 368 us).
// With five alternatives the registers stand at the border of five waves a SIMD (96): asked for, 250 and 301 us in
// float32 and 16 bits; left to the compiler, which takes 97, 256 and 344.
template <int DT, int PX, int K>
__global__ __launch_bounds__(kThreads, K == 5 ? 5 : 1) void k_scores_planes(Shape s, const elem_t<DT> *logits, const void *ids, Out o) {
    const int64_t groups = (s.rows + PX - 1) / PX;
    const int64_t at = blockIdx.x * (int64_t)kThreads + threadIdx.x;
    if (at >= s.batch * groups) return;
    const int64_t b = at / groups, r0 = at % groups * PX;
    const bool full = r0 + PX <= s.rows;
    const elem_t<DT> *base = logits + b * s.batch_stride + r0;
    float m[PX], ref[PX], sum[PX], wsum[PX], sum_off[PX], wsum_off[PX], xid[PX], tv[PX][K ? K : 1];
    int32_t ti[PX][K ? K : 1], id[PX];   // id: a class, kIgnored or kOutside
    constexpr int32_t kIgnored = -1, kOutside = -2;
#pragma unroll
    for (int q = 0; q < PX; ++q) {
        // the given class is picked up on the way: fetched afterwards, its line would come from memory again
        const int64_t want = load_id(s, ids, b, r0 + q < s.rows ? r0 + q : r0);
        id[q] = want == s.ignore_id ? kIgnored : want >= 0 && want < s.classes ? (int32_t)want : kOutside;
        xid[q] = 0.0f;
        m[q] = ref[q] = -INFINITY;
        sum[q] = wsum[q] = sum_off[q] = wsum_off[q] = 0.0f;
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
            float mn = x[0][q];
#pragma unroll
            for (int u = 1; u < kPlaneClasses; ++u) mn = fmaxf(mn, x[u][q]);
            if constexpr (K == 0) m[q] = fmaxf(m[q], mn);
            const float was = ref[q];
            if ((mn - was) * s.scale > 1.0f) ref[q] = mn;   // also the first maximum: -inf is in front of it
            const float ms = ref[q] == -INFINITY ? 0.0f : ref[q];
            const float d = fmaxf((was - ms) * s.scale, kTiny), a = __builtin_amdgcn_exp2f(d);   // 0 and 1 where it stays
            wsum[q] = a * (wsum[q] + sum[q] * d);
            wsum_off[q] = a * (wsum_off[q] + sum_off[q] * d);
            sum[q] *= a;
            sum_off[q] *= a;
            float part = 0.0f, wpart = 0.0f;
#pragma unroll
            for (int u = 0; u < kPlaneClasses; ++u) {
                const float t = (x[u][q] - ms) * s.scale, e = __builtin_amdgcn_exp2f(t);
                part += e;
                wpart += e * fmaxf(t, kTiny);
                xid[q] = id[q] == (int32_t)(c0 + u) ? x[u][q] : xid[q];
                if constexpr (K > 0) insert<K>(tv[q], ti[q], x[u][q], (int32_t)(c0 + u));
            }
            add_aside(sum[q], sum_off[q], part);
            add_aside(wsum[q], wsum_off[q], wpart);
        }
    }
#pragma unroll
    for (int q = 0; q < PX; ++q) {   // relative to the maximum, which is at most a factor of two away
        if constexpr (K > 0) m[q] = tv[q][0];
        const float d = ref[q] == m[q] ? 0.0f : (ref[q] - m[q]) * s.scale, a = __builtin_amdgcn_exp2f(d);
        sum[q] -= sum_off[q];
        wsum[q] = a * (wsum[q] - wsum_off[q] + sum[q] * d);
        sum[q] *= a;
    }
    Said said[PX];
#pragma unroll
    for (int q = 0; q < PX; ++q) said[q] = say(s, m[q], sum[q], wsum[q], id[q] == kIgnored, id[q] != kOutside, xid[q]);
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

constexpr int kGradPacks = 4;   // packs of 16 bytes a lane has in flight

// Rows: LPR lanes take kGradPacks packs each of one row, one pass.  d = p (A + B t) with t = log2 p, plus
// g_l at the given class; alternatives, at most 32 places of a row, are computed again and stored over the
// row afterwards by the lanes that wrote it.  Bound by memory: 4096 x 131072 bf16 takes 440 us, 4.9 TB/s.
template <int DT, int LPR>
__global__ __launch_bounds__(kThreads) void k_grad_rows(Shape s, const elem_t<DT> *logits, const void *ids, Grads g, elem_t<DT> *grad) {
    constexpr int VEC = 16 / sizeof(elem_t<DT>), U = kGradPacks, UNITS = kThreads / LPR;
    const int sub = threadIdx.x % LPR;
    const int64_t chunks = (s.classes + LPR * VEC * U - 1) / (LPR * VEC * U), units = s.batch * s.rows * chunks;
    for (int64_t unit = blockIdx.x * (int64_t)UNITS + threadIdx.x / LPR; unit < units; unit += (int64_t)gridDim.x * UNITS) {
        const int64_t pos = unit / chunks, b = pos / s.rows, r = pos % s.rows;
        const int64_t c0 = unit % chunks * (LPR * VEC * U), j0 = c0 + sub * VEC;
        const elem_t<DT> *row = logits + b * s.batch_stride + r * s.row_stride;
        elem_t<DT> *out = grad + pos * s.classes;
        Pack<DT, VEC> in[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t j = j0 + u * (LPR * VEC);
            if (j + VEC <= s.classes) {
                in[u] = load_pack<DT, VEC>(row + j);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (j + e < s.classes) in[u].v[e] = row[j + e];
            }
        }
        const int64_t want = load_id(s, ids, b, r);
        const float log_sum = g.log_sum[pos];
        float m = g.row_max[pos], off = log_sum * kLog2e;
        const bool none = m == -INFINITY, given = g.g_log_prob && want != s.ignore_id, inside = want >= 0 && want < s.classes;
        const bool bad = log_sum != log_sum || (given && !inside);
        const int top = g.g_top && !none ? s.top : 0;
        float gl = given ? g.g_log_prob[pos] : 0.0f, all = gl;
        for (int k = 0; k < top; ++k) {
            const int32_t c = g.top_ids[pos * s.top + k];
            all += c >= 0 && c < s.classes ? g.g_top[pos * s.top + k] : 0.0f;
        }
        const float ge = g.g_entropy ? g.g_entropy[pos] : 0.0f, h = g.g_entropy ? g.entropy[pos] : 0.0f;
        float A = -(all + ge * h) * s.inv_t, B = -ge * kLn2 * s.inv_t;
        gl *= s.inv_t;
        int64_t id = given && inside ? want : -1;
        if (none) {   // every t is -inf and every p 0
            m = off = A = B = 0.0f;
            id = -1;
        }
        if (bad) A = __builtin_nanf("");
        const auto dense = [&](float x) {
            const float t = (x - m) * s.scale - off;
            return __builtin_amdgcn_exp2f(t) * (A + B * fmaxf(t, kTiny));
        };
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t j = j0 + u * (LPR * VEC);
            const int64_t at = id - j;   // the given class within this pack
            Pack<DT, VEC> w;
#pragma unroll
            for (int e = 0; e < VEC; ++e) w.v[e] = Elem<DT>::put(dense(Elem<DT>::get(in[u].v[e])) + (at == e ? gl : 0.0f));
            if (j + VEC <= s.classes) {
                store_pack<DT, VEC>(out + j, w);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (j + e < s.classes) out[j + e] = w.v[e];
            }
        }
        if (top) {
            bool waited = false;
            for (int k = sub; k < top; k += LPR) {
                const int64_t c = g.top_ids[pos * s.top + k];
                if (c < c0 || c >= c0 + LPR * VEC * U || c >= s.classes) continue;
                if (!waited) {   // the stores above come from other lanes of this wave
                    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                    waited = true;
                }
                out[c] = Elem<DT>::put(dense(Elem<DT>::get(row[c])) + (c == id ? gl : 0.0f) + g.g_top[pos * s.top + k] * s.inv_t);
            }
        }
    }
}

// Planes: a thread walks the classes of PX neighbouring positions.  K >= s.top.  Bound by memory: 4 x 150 x 480 x
// 640 float32 with two alternatives takes 330 us, 4.6 TB/s.
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
            if (ti[q][k] >= s.classes) ti[q][k] = -1;
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
    if (!head_sizes_ok(a->batch, a->rows, a->classes) || a->classes < 1 || a->classes > (1 << 30))
        return head_error(SSMAP_ERR_INVALID_ARG, "batch, rows >= 0, 1 <= classes <= 2^30 and fewer than 2^40 logits are required");
    if (a->batch * a->rows > INT32_MAX) return head_error(SSMAP_ERR_UNSUPPORTED, "more than 2^31 - 1 positions");
    if (a->top < 0 || a->top > SSMAP_MAX_TOP || a->top > a->classes)
        return head_error(SSMAP_ERR_INVALID_ARG, "top must be in [0, min(32, classes)]");
    if (!(a->temperature >= 1e-30f && a->temperature <= 1e30f))
        return head_error(SSMAP_ERR_INVALID_ARG, "temperature must be in [1e-30, 1e30]");
    if (a->batch_stride < 0 || a->inner_stride < 0 || a->ids_batch_stride < 0 || a->ids_row_stride < 0)
        return head_error(SSMAP_ERR_INVALID_ARG, "strides must not be negative");
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
    constexpr int VEC = 16 / sizeof(elem_t<DT>), NP = 64 / (VEC * sizeof(float));   // 16 floats of a row a lane
    const int64_t n = s.batch * s.rows;
    const auto brief = [&](auto lpr, auto np) {
        const int64_t blocks = (n + kThreads / lpr.value - 1) / (kThreads / lpr.value);
        k_scores_short<DT, lpr.value, np.value><<<(unsigned)(blocks < kShortBlocks ? blocks : kShortBlocks), kThreads, 0, st>>>(s, x, a.ids, o);
    };
    if (s.classes <= 16 * VEC) return brief(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
    if (s.classes <= 32 * VEC) return brief(std::integral_constant<int, 16>{}, std::integral_constant<int, 2>{});
    if constexpr (NP == 4) {
        if (s.classes <= 48 * VEC) return brief(std::integral_constant<int, 16>{}, std::integral_constant<int, 3>{});
        if (s.classes <= 64 * VEC) return brief(std::integral_constant<int, 16>{}, std::integral_constant<int, 4>{});
    }
    // 4096 x 600 bf16 takes 4.8 us here and 14.6 as long rows, 13.8 and 32.3 with five alternatives.  Twice the registers,
    // for 2000 classes: 8.7 and 14.8, with alternatives 32.4 and 32.2, of 64 rows 15.8 and 10.8.
    if (s.classes <= 64 * VEC * NP) return brief(std::integral_constant<int, 64>{}, std::integral_constant<int, NP>{});
    const Split w = split_rows(s, DT);
    char *parts = static_cast<char *>(a.workspace);
    const int64_t units = n * w.splits;
    k_scores_long<DT><<<(unsigned)(units < kMostBlocks ? units : kMostBlocks), kThreads, 0, st>>>(s, x, a.ids, o, w.splits, w.segment, parts, w.part_bytes);
    if (w.splits > 1) k_scores_join<DT><<<(unsigned)n, kThreads, 0, st>>>(s, x, a.ids, o, w.splits, parts, w.part_bytes);
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
    constexpr int VEC = 16 / sizeof(elem_t<DT>);
    const auto go = [&](auto lpr) {
        constexpr int LPR = lpr.value, UNITS = kThreads / LPR;
        const int64_t chunks = (s.classes + LPR * VEC * kGradPacks - 1) / (LPR * VEC * kGradPacks), units = s.batch * s.rows * chunks;
        const int64_t blocks = (units + UNITS - 1) / UNITS;
        k_grad_rows<DT, LPR><<<(unsigned)(blocks < kMostBlocks ? blocks : kMostBlocks), kThreads, 0, st>>>(s, x, a.ids, g, out);
    };
    // a quarter of a wave where it holds the whole row
    if (s.classes <= 16 * VEC * kGradPacks) go(std::integral_constant<int, 16>{});
    else go(std::integral_constant<int, 64>{});
}

}  // namespace

extern "C" {

int64_t ssmap_log_probs_workspace(const ssmap_log_probs_args *a) {
    Shape s{};
    if (!a) { head_error(SSMAP_ERR_INVALID_ARG, "null argument"); return -1; }
    if (check(a, s) != SSMAP_OK) return -1;
    if (s.layout == SSMAP_PLANES) return 0;
    const Split w = split_rows(s, a->dtype);
    return w.splits > 1 ? s.batch * s.rows * w.splits * w.part_bytes : 0;
}

int ssmap_log_probs(const ssmap_log_probs_args *a, void *stream) {
    if (!a) return head_error(SSMAP_ERR_INVALID_ARG, "null argument");
    Shape s{};
    if (int rc = check(a, s)) return rc;
    if (s.batch * s.rows == 0) return SSMAP_OK;
    if (!a->logits || !a->ids || !a->log_prob || !a->entropy || !a->row_max || !a->log_sum || (a->top && (!a->top_ids || !a->top_log_prob)))
        return head_error(SSMAP_ERR_INVALID_ARG, "null argument");
    const int64_t need = ssmap_log_probs_workspace(a);
    if (a->workspace_bytes < need || (need && (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 16)))
        return head_error(SSMAP_ERR_INVALID_ARG, "the workspace is not at a multiple of 16 or smaller than ssmap_log_probs_workspace says");
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
