// Matrix products on the matrix cores: out[m][n] = sum_k a(m, k) b(n, k), tile by tile.
//
// A block computes BI x BJ results, I the m side and J the n side, dense in memory.  A stage is 128 of
// every tile row in the sum's direction (64 values of 16 bits, 32 of float32), laid out in LDS as 16-byte
// chunks; two stages alternate.  A side whose sum direction is dense in memory (KC) keeps its rows: chunk c
// of row r sits at slot r * 8 + (c ^ (r & 7)), so that the 16 rows that one matrix instruction reads at one
// c lie in different banks.  A side whose other direction is dense keeps rows of the sum index instead, and
// is turned while it is read: ds_read_b64_tr_b16 gives lane q of 16 the values of column q from four rows of
// 16 columns.  Its chunks are swizzled by 32 bytes a row, so that the four rows lie in different banks.
//
// What bounds it at large sizes is the way from L2 to LDS: at 8192^3 bf16 the loads alone take 711 us, the matrix
// instructions alone 674, both together 890 to 925 (1190 to 1240 TFLOP/s).  So tiles are as large as the registers
// hold, and the turns below keep the loads from holding up the reads.
//
// The matrix instruction takes J as its rows and I as its columns: a lane then holds four neighbouring n of
// one m, which the epilogue reads and writes together.
#pragma once

#include "products.h"

namespace ssmap {

using f32x4 = float __attribute__((ext_vector_type(4)));
using i32x4 = int __attribute__((ext_vector_type(4)));
using bf16x8 = __bf16 __attribute__((ext_vector_type(8)));
using f16x8 = _Float16 __attribute__((ext_vector_type(8)));
using i16x4 = short __attribute__((ext_vector_type(4)));

// acc += (chunk of J) x (chunk of I): every lane of a group of 16 holds the same stretch of the sum, groups
// hold neighbouring stretches.
template <int DT>
__device__ __forceinline__ f32x4 mma_chunk(i32x4 j, i32x4 i, f32x4 acc) {
    if constexpr (DT == SSMAP_BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, j), __builtin_bit_cast(bf16x8, i), acc, 0, 0, 0);
    } else if constexpr (DT == SSMAP_F16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, j), __builtin_bit_cast(f16x8, i), acc, 0, 0, 0);
    } else {
        const f32x4 a = __builtin_bit_cast(f32x4, j), b = __builtin_bit_cast(f32x4, i);
#pragma unroll
        for (int s = 0; s < 4; ++s) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], acc, 0, 0, 0);
        return acc;
    }
}

constexpr uint32_t kNowhere = 0xFFFFFFF0u;   // a buffer offset behind every descriptor's end: reads as zero

// One side of a tile: R rows (or columns) of it, eight chunks of the sum's direction a stage, NT threads.
template <int DT, bool KC, int R, int NT>
struct Side {
    static constexpr int C = 8, SIZE = head_dtype_size(DT), E = 16 / SIZE, KB = C * E;   // chunks a stage; values a chunk, a stage
    static constexpr int PER = R * C / NT, ROW = R / E;                           // chunks a thread; a row (not KC)
    static constexpr int BYTES = R * C * 16;
    static_assert(R * C % NT == 0 && (KC || ROW >= 8), "tile shape");

    static __device__ __forceinline__ int swizzle(int k) { return DT == SSMAP_F32 ? ((k >> 2) & 3) << 2 : (k & 3) << 1; }

    // KC: 128 bytes of consecutive slots hold eight rows' chunks of one c
    static __device__ __forceinline__ int turn(int row) { return row & 7; }

    // chunk of slot s: its row (KC) or sum index (not KC), and its place there
    static __device__ __forceinline__ void place(int s, int &line, int &c) {
        if constexpr (KC) line = s / C, c = (s % C) ^ turn(line);
        else line = s / ROW, c = (s % ROW) ^ swizzle(line);
    }
    // how many of its values exist: `rows` are left on this side, `ks` in the sum
    static __device__ __forceinline__ int count(int line, int c, int rows, int ks) {
        const int across = KC ? rows : ks, along = (KC ? ks : rows) - c * E;
        return line < across ? (along < 0 ? 0 : along < E ? along : E) : 0;
    }

    // Straight from memory to LDS: 16 bytes a lane, a wave's 64 chunks land one after the other.  `base` is the
    // tile's corner, `ld` the bytes of a line; both multiples of 16, and so are the dense extents in bytes.
    static __device__ __forceinline__ void offsets(uint32_t (&off)[PER], int rows, int ks, uint32_t ld) {
#pragma unroll
        for (int it = 0; it < PER; ++it) {
            int line, c;
            place(it * NT + threadIdx.x, line, c);
            off[it] = count(line, c, rows, ks) ? line * ld + c * 16 : kNowhere;
        }
    }
    static __device__ __forceinline__ void fetch(const char *base, const uint32_t (&off)[PER], uint32_t lds) {
        // word 1 holds the address's upper bits and no stride, word 2 the length, word 3 a raw format
        const uint64_t at = (uint64_t)base;
        const i32x4 desc = {(int)(uint32_t)at, (int)(uint32_t)(at >> 32) & 0xFFFF, (int)0x80000000u, 0x00020000};
        const uint32_t first = lds + (threadIdx.x / 64) * 1024;
#pragma unroll
        for (int it = 0; it < PER; ++it) {
            // Five wait states: the descriptor may come out of vector lanes (a spilled scalar register), and the
            // compiler counts none of its own in front of an instruction it does not see.
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(
                             __builtin_amdgcn_readfirstlane(first + it * NT * 16)),
                         "v"(off[it]), "s"(desc)
                         : "memory");   // m0 is reserved: the compiler keeps nothing in it
        }
    }

    // Through registers, for any alignment and extent.  Where everything exists (`all`, the same for the whole
    // block) the loads have 32-bit offsets from one base and no branch between them.
    static __device__ __forceinline__ void all_offsets(uint32_t (&off)[PER], uint32_t ld) {
#pragma unroll
        for (int it = 0; it < PER; ++it) {
            int line, c;
            place(it * NT + threadIdx.x, line, c);
            off[it] = line * ld + c * 16;
        }
    }
    static __device__ __forceinline__ void load(i32x4 (&reg)[PER], const char *base, const uint32_t (&off)[PER], bool all, int rows, int ks, int64_t ld) {
        using loose = int __attribute__((ext_vector_type(4), aligned(2)));   // 16 bytes at any element
        if (all) {
#pragma unroll
            for (int it = 0; it < PER; ++it) reg[it] = *reinterpret_cast<const loose *>(base + off[it]);
            return;
        }
#pragma unroll
        for (int it = 0; it < PER; ++it) {
            int line, c;
            place(it * NT + threadIdx.x, line, c);
            const int n = count(line, c, rows, ks);
            const elem_t<DT> *p = reinterpret_cast<const elem_t<DT> *>(base + line * ld + c * 16);
            elem_t<DT> e[E];
#pragma unroll
            for (int q = 0; q < E; ++q) {
                e[q] = Elem<DT>::put(0.0f);
                if (q < n) e[q] = p[q];
            }
            __builtin_memcpy(&reg[it], e, 16);
        }
    }
    static __device__ __forceinline__ void store(const i32x4 (&reg)[PER], char *lds) {
#pragma unroll
        for (int it = 0; it < PER; ++it) *reinterpret_cast<i32x4 *>(lds + (it * NT + threadIdx.x) * 16) = reg[it];
    }

    // The chunk of rows row0 ... row0 + 15 for half kk of the stage.
    static __device__ __forceinline__ i32x4 read(const char *lds, int row0, int kk) {
        const int lane = threadIdx.x % 64, q = lane % 16, g = lane / 16;
        if constexpr (KC) {
            return *reinterpret_cast<const i32x4 *>(lds + (row0 + q) * (C * 16) + (((kk * 4 + g) ^ turn(q)) * 16));
        } else if constexpr (DT == SSMAP_F32) {
            f32x4 v;
            const int i = row0 + q;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int k = kk * 16 + g * 4 + s;
                v[s] = *reinterpret_cast<const float *>(lds + (k * ROW + ((i / 4) ^ swizzle(k))) * 16 + (i & 3) * 4);
            }
            return __builtin_bit_cast(i32x4, v);
        } else {
            union {
                i16x4 h[2];
                i32x4 v;
            } u;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = kk * 32 + g * 8 + h * 4 + q / 4;
                const char *p = lds + (k * ROW + ((row0 / 8 + (q % 4) / 2) ^ swizzle(k))) * 16 + (q & 1) * 8;
                u.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4 *)p);
            }
            return u.v;
        }
    }
};

// N values next to each other, of which `left` exist; WHOLE: all of them, which the caller knows for its whole
// wave (with a branch for each lane the compiler merges both ways into pieces of 2 to 12 bytes).
template <int DT, int N>
struct Run {
    elem_t<DT> v[N];
};
template <bool WHOLE, int DT, int N>
__device__ __forceinline__ Run<DT, N> load_run(const void *from, int64_t at, int left) {
    const elem_t<DT> *src = static_cast<const elem_t<DT> *>(from) + at;
    Run<DT, N> r;
    if constexpr (WHOLE) {
        __builtin_memcpy(&r, src, sizeof r);
    } else {
#pragma unroll
        for (int q = 0; q < N; ++q) {
            r.v[q] = Elem<DT>::put(0.0f);
            if (q < left) r.v[q] = src[q];
        }
    }
    return r;
}
template <bool WHOLE, int DT, int N, bool PAST = false>   // PAST: past the caches
__device__ __forceinline__ void store_run(void *to, int64_t at, int left, const float (&z)[N]) {
    elem_t<DT> *dst = static_cast<elem_t<DT> *>(to) + at;
    Run<DT, N> r;
#pragma unroll
    for (int q = 0; q < N; ++q) r.v[q] = Elem<DT>::put(z[q]);
    if constexpr (WHOLE && PAST) {
        using loose = int __attribute__((ext_vector_type(sizeof r / 4), aligned(2)));
        __builtin_nontemporal_store(__builtin_bit_cast(loose, r), reinterpret_cast<loose *>(dst));
    } else if constexpr (WHOLE) {
        __builtin_memcpy(dst, &r, sizeof r);
    } else {
#pragma unroll
        for (int q = 0; q < N; ++q)
            if (q < left) dst[q] = r.v[q];
    }
}

// The epilogue's operands of N results at (m, n ... n + N - 1).
template <bool WHOLE, int DT, int N>
__device__ __forceinline__ void load_bias(const Product &p, int64_t m, int64_t n, int left, float (&b)[N]) {
#pragma unroll
    for (int q = 0; q < N; ++q) b[q] = 0.0f;
    if (!p.bias) return;
    if (p.bias_along_m) {
        const float v = p.bias_f32 ? static_cast<const float *>(p.bias)[m] : Elem<DT>::get(static_cast<const elem_t<DT> *>(p.bias)[m]);
#pragma unroll
        for (int q = 0; q < N; ++q) b[q] = v;
    } else if (p.bias_f32) {
        const Run<SSMAP_F32, N> r = load_run<WHOLE, SSMAP_F32, N>(p.bias, n, left);
#pragma unroll
        for (int q = 0; q < N; ++q) b[q] = r.v[q];
    } else {
        const Run<DT, N> r = load_run<WHOLE, DT, N>(p.bias, n, left);
#pragma unroll
        for (int q = 0; q < N; ++q) b[q] = Elem<DT>::get(r.v[q]);
    }
}
// `o` is the first result's place in the dense output.
template <bool WHOLE, int DT, int OT, int N, bool PAST = false>
__device__ __forceinline__ void finish(const Product &p, int64_t o, int left, float (&z)[N], const float (&bias)[N], const Run<OT, N> &res) {
    if constexpr (DT == SSMAP_F16 && OT == SSMAP_F16)
        if (p.unscale) {
#pragma unroll
            for (int q = 0; q < N; ++q) z[q] *= *p.unscale;
        }
    if (p.bias) {
#pragma unroll
        for (int q = 0; q < N; ++q) z[q] += bias[q];
    }
    if (p.pre) store_run<WHOLE, DT, N>(p.pre, o, left, z);
    with_activation(p.act, [&](auto act) {
#pragma unroll
        for (int q = 0; q < N; ++q) z[q] = activate<act.value, OT == SSMAP_F32>(z[q]);
    });
    if (p.res) {
#pragma unroll
        for (int q = 0; q < N; ++q) z[q] += Elem<OT>::get(res.v[q]);
    }
    store_run<WHOLE, OT, N, PAST>(p.out, o, left, z);
}
template <bool WHOLE, int DT, int OT, int N, bool PAST = false>
__device__ __forceinline__ void finish_at(const Product &p, int64_t e, int64_t m, int64_t n, int left, float (&z)[N]) {
    float bias[N];
    load_bias<WHOLE, DT, N>(p, m, n, left, bias);
    Run<OT, N> res;
    if (p.res) res = load_run<WHOLE, OT, N>(p.res, e * p.res_out + m * p.res_m + n, left);
    finish<WHOLE, DT, OT, N, PAST>(p, (e * p.M + m) * p.N + n, left, z, bias, res);
}

// BI x BJ results a block, WI x WJ waves, stages in NBUF buffers.  DIRECT: both sides go straight to LDS (see
// Side::fetch), NBUF - 1 stages ahead; otherwise through registers, one stage ahead.
template <int DT, int OT, bool IK, bool JK, int BI, int BJ, int WI, int WJ, int NBUF, bool DIRECT>
__global__ __launch_bounds__(WI *WJ * 64) void k_tiles(Product p) {
    constexpr int NT = WI * WJ * 64, TI = BI / WI / 16, TJ = BJ / WJ / 16, SIZE = head_dtype_size(DT);
    using I = Side<DT, IK, BI, NT>;
    using J = Side<DT, JK, BJ, NT>;
    constexpr int PITCH = TJ * 16 + 4;                 // floats a row while results are turned: four off, for the banks
    constexpr int HI = TI > 4 ? TI / 2 : TI;           // rows of 16 turned at once
    constexpr int LINE = TJ * 16 / 8, ROWS = 64 / LINE;   // lanes a row, rows at once
    constexpr int STAGE = I::BYTES + J::BYTES, TURN = WI * WJ * HI * 16 * PITCH * 4;
    __shared__ __attribute__((aligned(1024))) char lds_all[NBUF * STAGE > TURN ? NBUF * STAGE : TURN];
    const auto stage = [&](int buf) { return lds_all + buf * STAGE; };
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wi = wave % WI, wj = wave / WI;
    const int64_t tiles_m = (p.M + BI - 1) / BI, tiles_n = (p.N + BJ - 1) / BJ, tiles = tiles_m * tiles_n;
    const int64_t steps = (p.K + I::KB - 1) / I::KB, all_steps = steps * p.sum_batches;
    const int64_t units = tiles * p.out_batches * p.splits;
    for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
        // Blocks go round the eight XCDs; each takes a run of neighbouring tiles, so that its L2 sees the same
        // rows again.  Within a run eight tile rows are walked column by column.
        int64_t id = unit;
        if (units % 8 == 0) id = (unit % 8) * (units / 8) + unit / 8;
        const int64_t tile = id % tiles, outer = id / tiles, e = outer % p.out_batches, split = outer / p.out_batches;
        constexpr int64_t BAND = 8;
        const int64_t band = tile / (BAND * tiles_n), rows_in = tiles_m - band * BAND < BAND ? tiles_m - band * BAND : BAND;
        const int64_t in_band = tile % (BAND * tiles_n);
        const int64_t i0 = (band * BAND + in_band % rows_in) * BI, j0 = in_band / rows_in * BJ;
        const int rows_i = (int)(p.M - i0 < BI ? p.M - i0 : BI), rows_j = (int)(p.N - j0 < BJ ? p.N - j0 : BJ);
        const int64_t first = split * p.part_steps, last = first + p.part_steps < all_steps ? first + p.part_steps : all_steps;
        const int64_t ld_i = (IK ? p.a_m : p.a_k) * SIZE, ld_j = (JK ? p.b_n : p.b_k) * SIZE;
        const int64_t step_i = (IK ? 1 : p.a_k) * (int64_t)(I::KB * SIZE), step_j = (JK ? 1 : p.b_k) * (int64_t)(I::KB * SIZE);
        const char *pa = static_cast<const char *>(p.a) + (e * p.a_out + i0 * p.a_m) * SIZE;
        const char *pb = static_cast<const char *>(p.b) + (e * p.b_out + j0 * p.b_n) * SIZE;
        int64_t at = first % (steps ? steps : 1);      // stage within its sum batch
        int64_t b_block = first / (steps ? steps : 1) % p.b_again;
        pa += first / (steps ? steps : 1) * p.a_sum * SIZE + at * step_i;
        pb += b_block * p.b_sum * SIZE + at * step_j;
        const auto advance = [&] {
            if (++at == steps) {
                at = 0;
                pa += p.a_sum * SIZE - (steps - 1) * step_i;
                pb += p.b_sum * SIZE - (steps - 1) * step_j;
                if (++b_block == p.b_again) b_block = 0, pb -= p.b_again * p.b_sum * SIZE;
            } else {
                pa += step_i;
                pb += step_j;
            }
        };
        uint32_t off_i[I::PER], off_j[J::PER];
        i32x4 reg_i[DIRECT ? 1 : I::PER], reg_j[DIRECT ? 1 : J::PER];
        if constexpr (DIRECT) {
            I::offsets(off_i, rows_i, I::KB, (uint32_t)ld_i);
            J::offsets(off_j, rows_j, I::KB, (uint32_t)ld_j);
        } else {
            I::all_offsets(off_i, (uint32_t)ld_i);
            J::all_offsets(off_j, (uint32_t)ld_j);
        }
        const bool all_i = rows_i == BI && ld_i < 1 << 24, all_j = rows_j == BJ && ld_j < 1 << 24;   // 256 lines: 32-bit offsets
        const auto fetch = [&](int buf) {   // stage `at` into buffer buf (DIRECT) or into registers
            const int64_t left = p.K - at * I::KB;
            const int ks = (int)(left < I::KB ? left : I::KB);
            if constexpr (DIRECT) {
                const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)stage(buf);
                if (ks < I::KB) {
                    uint32_t tail_i[I::PER], tail_j[J::PER];
                    I::offsets(tail_i, rows_i, ks, (uint32_t)ld_i);
                    J::offsets(tail_j, rows_j, ks, (uint32_t)ld_j);
                    I::fetch(pa, tail_i, base);
                    J::fetch(pb, tail_j, base + I::BYTES);
                } else {
                    I::fetch(pa, off_i, base);
                    J::fetch(pb, off_j, base + I::BYTES);
                }
            } else {
                I::load(reg_i, pa, off_i, all_i && ks == I::KB, rows_i, ks, ld_i);
                J::load(reg_j, pb, off_j, all_j && ks == I::KB, rows_j, ks, ld_j);
            }
            advance();
        };
        const auto keep = [&](int buf) {
            if constexpr (!DIRECT) {
                I::store(reg_i, stage(buf));
                J::store(reg_j, stage(buf) + I::BYTES);
            }
        };
        f32x4 acc[TI][TJ] = {};
        i32x4 fi[TI], fj[TJ];
        const auto read = [&](int buf, int kk, i32x4 (&fi)[TI], i32x4 (&fj)[TJ]) {
            const char *li = stage(buf), *lj = li + I::BYTES;
#pragma unroll
            for (int i = 0; i < TI; ++i) fi[i] = I::read(li, (wi * TI + i) * 16, kk);
#pragma unroll
            for (int j = 0; j < TJ; ++j) fj[j] = J::read(lj, (wj * TJ + j) * 16, kk);
        };
        const auto multiply = [&](const i32x4 (&fi)[TI], const i32x4 (&fj)[TJ]) {
#pragma unroll
            for (int i = 0; i < TI; ++i)
#pragma unroll
                for (int j = 0; j < TJ; ++j) acc[i][j] = mma_chunk<DT>(fj[j], fi[i], acc[i][j]);
        };
        if constexpr (WI * WJ == 8) {
            // Two waves a SIMD take turns: while one multiplies half a stage, the other reads its next half from
            // LDS and sends for the stage after the next.  The second four waves run one turn behind.  A barrier
            // ends each turn; the scheduler moves nothing over it.  The first waves read the halves of stage t in
            // turns 4t and 4t + 2 and multiply them in the turns behind; the second waves read the last half of
            // stage t - 1 in turn 4t - 1.  So from turn 4t on that stage's buffer is free for stage t + 1: the
            // first waves send for it in turn 4t, the second ones in turn 4t + 1, each behind its reads (in front
            // of them or of the matrix instructions the queue of loads held those up: 937 against 896 us at
            // 8192^3), and all have waited for it at the end of turn 4t + 3.
            static_assert(DIRECT && NBUF == 2, "two turns a stage");
            const bool late = wave >= 4;
            const auto turn_ends = [&] {
                __builtin_amdgcn_sched_barrier(0);
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
            };
            const auto have_read = [&] { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };
            const auto have_landed = [&] { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); };
            if (first < last) {
                fetch(0);
                have_landed();
                turn_ends();
                if (late) turn_ends();
                for (int64_t t = first; t < last; ++t) {
                    const int buf = (int)((t - first) & 1);
                    read(buf, 0, fi, fj);
                    __builtin_amdgcn_sched_barrier(0);
                    if (t + 1 < last) fetch(buf ^ 1);
                    have_read();
                    turn_ends();
                    __builtin_amdgcn_s_setprio(1);
                    multiply(fi, fj);
                    __builtin_amdgcn_s_setprio(0);
                    turn_ends();
                    read(buf, 1, fi, fj);
                    if (late) have_landed();
                    have_read();
                    turn_ends();
                    __builtin_amdgcn_s_setprio(1);
                    multiply(fi, fj);
                    __builtin_amdgcn_s_setprio(0);
                    if (!late) have_landed();
                    turn_ends();
                }
                if (!late) turn_ends();   // the second waves' last turn
            }
        } else {
            static_assert(DIRECT || NBUF == 2, "one stage of registers");
            int64_t sent = first;
            for (; sent < first + NBUF - 1 && sent < last; ++sent) {
                fetch((int)(sent - first));
                keep((int)(sent - first));
            }
            int buf = 0;
            for (int64_t t = first; t < last; ++t) {
                // This wave's part of the stage has landed (loads return in order: those of the stages behind it may
                // be under way), and its reads of the stage before have; behind the barrier that holds for all, and
                // the buffer of the stage before is free.
                if constexpr (DIRECT) {
                    if (sent < last) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NBUF - 2) * (I::PER + J::PER)) : "memory");
                    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                    __builtin_amdgcn_s_barrier();
                    asm volatile("" ::: "memory");
                } else {
                    __syncthreads();
                }
                const int next = buf ? buf - 1 : NBUF - 1;
                const bool more = sent < last;
                if (more) fetch(next), ++sent;
                // Both halves' operands first, in registers of their own: left to itself the compiler reads each into
                // the same few registers in front of the matrix instructions that want it, and waits every time
                // (8192 x 4096 x 8192 bf16 in 128 wide tiles: 643 against 601 us).  The loads are sent in front of
                // the reads here: two blocks a CU keep each other busy, and behind the reads they come late (626).
                i32x4 gi[TI], gj[TJ];
                read(buf, 0, fi, fj);
                read(buf, 1, gi, gj);
                __builtin_amdgcn_sched_barrier(0);
                multiply(fi, fj);
                multiply(gi, gj);
                if (more) keep(next);
                buf = buf + 1 == NBUF ? 0 : buf + 1;
            }
        }
        __syncthreads();   // nobody reads the stages any more
        // Each wave turns its own results round in LDS, HI rows of 16 at a time: out of the registers with four
        // neighbouring n a lane, back with eight.  Loops stay loops here: the code runs once a tile and
        // is fetched anew each time (8192 x 4096 x 8192 bf16 with gelu and residual: 536 us unrolled, 502 so).  The
        // residual of the next rows is under way while these are finished.
        const int lane = threadIdx.x % 64, q = lane % 16, g = lane / 16;
        float *turn = reinterpret_cast<float *>(lds_all + wave * (HI * 16 * PITCH * 4));
        const int col = lane % LINE * 8;
        const int64_t n = j0 + wj * TJ * 16 + col;
        const float *mine = turn + lane / LINE * PITCH + col;
        const bool whole = rows_i == BI && rows_j == BJ;
#pragma unroll 1
        for (int h = 0; h < TI / HI; ++h) {
#pragma unroll
            for (int k = 0; k < TI / HI; ++k)
                if (k == h)
#pragma unroll
                    for (int i = 0; i < HI; ++i)
#pragma unroll
                        for (int j = 0; j < TJ; ++j) *reinterpret_cast<f32x4 *>(turn + (i * 16 + q) * PITCH + j * 16 + g * 4) = acc[k * HI + i][j];
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");   // the wave's own writes, in order
            __builtin_amdgcn_wave_barrier();
            int64_t m = i0 + (wi * TI + h * HI) * 16 + lane / LINE;
            if (whole) {
                float bias[8];
                load_bias<true, DT, 8>(p, m, n, 8, bias);
                Run<OT, 8> res, next;
                int64_t o = (e * p.M + m) * p.N + n;
                if (p.res) next = load_run<true, OT, 8>(p.res, e * p.res_out + m * p.res_m + n, 8);
#pragma unroll 1
                for (int r0 = 0; r0 < HI * 16; r0 += ROWS) {
                    res = next;
                    if (p.res && r0 + ROWS < HI * 16) next = load_run<true, OT, 8>(p.res, e * p.res_out + (m + ROWS) * p.res_m + n, 8);
                    float z[8];
                    __builtin_memcpy(z, __builtin_assume_aligned(mine + r0 * PITCH, 16), 32);
                    if (p.splits > 1) {
                        store_run<true, SSMAP_F32, 8>(p.parts + split * p.out_batches * p.M * p.N, o, 8, z);
                    } else {
                        if (p.bias_along_m) load_bias<true, DT, 8>(p, m, n, 8, bias);
                        finish<true, DT, OT, 8, true>(p, o, 8, z, bias, res);
                    }
                    m += ROWS;
                    o += ROWS * p.N;
                }
            } else {
                const int left = (int)(p.N - n < 8 ? p.N - n : 8);
#pragma unroll 1
                for (int r0 = 0; r0 < HI * 16; r0 += ROWS, m += ROWS) {
                    if (m >= p.M || left <= 0) continue;
                    float z[8];
                    __builtin_memcpy(z, __builtin_assume_aligned(mine + r0 * PITCH, 16), 32);
                    if (p.splits > 1) store_run<false, SSMAP_F32, 8>(p.parts + split * p.out_batches * p.M * p.N, (e * p.M + m) * p.N + n, left, z);
                    else finish_at<false, DT, OT, 8>(p, e, m, n, left, z);
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();   // the next tile's first stage overwrites the buffers
    }
}

// Joins the partial results of a split sum and finishes them: 256 / LANES quads of results a block, LANES
// threads a quad, each over its share of the splits; joined in a fixed order.
template <int DT, int OT, int LANES>
__global__ __launch_bounds__(256) void k_join_parts(Product p) {
    constexpr int QUADS = 256 / LANES;
    __shared__ f32x4 sums[LANES][QUADS];
    const int64_t row = (p.N + 3) / 4, units = p.out_batches * p.M * row;
    const int quad = threadIdx.x % QUADS, part = threadIdx.x / QUADS;
    for (int64_t u0 = blockIdx.x * (int64_t)QUADS; u0 < units; u0 += gridDim.x * (int64_t)QUADS) {
        const int64_t u = u0 + quad < units ? u0 + quad : units - 1;
        const int64_t em = u / row, e = em / p.M, m = em % p.M, n = u % row * 4, o = em * p.N + n;
        const int left = (int)(p.N - n < 4 ? p.N - n : 4);
        float z[4] = {};
#pragma unroll 4
        for (int s = part; s < p.splits; s += LANES) {
            const float *from = p.parts + s * p.out_batches * p.M * p.N + o;
            float v[4] = {};
            if (left == 4) __builtin_memcpy(v, from, 16);
            else {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (q < left) v[q] = from[q];
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) z[q] += v[q];
        }
        if constexpr (LANES > 1) {
            __syncthreads();
            sums[part][quad] = f32x4{z[0], z[1], z[2], z[3]};
            __syncthreads();
            if (part == 0)
#pragma unroll
                for (int k = 1; k < LANES; ++k)
#pragma unroll
                    for (int q = 0; q < 4; ++q) z[q] += sums[k][quad][q];
        }
        if (part == 0 && u0 + quad < units) {
            if (left == 4) finish_at<true, DT, OT, 4>(p, e, m, n, 4, z);
            else finish_at<false, DT, OT, 4>(p, e, m, n, left, z);
        }
    }
}

// At most 16 MT rows of a (single tokens, small batches) against all of b: reading b once is all the work.  A
// block takes 16 rows of b, its eight waves share the sum; both operands go from memory to registers as the
// matrix instruction wants them, eight loads of b under way in each wave.  3 x 4096 x 4096 bf16 takes 9.5 us, 3.5
// TB/s; a 64 x 256 tile with a split sum 20.
constexpr int kFewWaves = 8;
template <int DT, int OT, int MT>
__global__ __launch_bounds__(kFewWaves * 64) void k_few_rows(Product p) {
    constexpr int SIZE = head_dtype_size(DT), E = 16 / SIZE, U = MT == 1 ? 8 : 4;
    __shared__ f32x4 sums[kFewWaves][MT][64];
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, q = lane % 16, g = lane / 16;
    const int64_t tiles = (p.N + 15) / 16, units = tiles * p.out_batches;
    const int64_t all = (p.K + 4 * E - 1) / (4 * E), from = all * wave / kFewWaves, to = all * (wave + 1) / kFewWaves;
    for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const int64_t e = unit / tiles, n0 = unit % tiles * 16;
        // rows behind the last one are read as the last one; their results are dropped
        const elem_t<DT> *pb = static_cast<const elem_t<DT> *>(p.b) + e * p.b_out + (n0 + q < p.N ? n0 + q : p.N - 1) * p.b_n + g * E;
        const elem_t<DT> *pa[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int64_t m = t * 16 + q;
            pa[t] = static_cast<const elem_t<DT> *>(p.a) + e * p.a_out + (m < p.M ? m : p.M - 1) * p.a_m + g * E;
        }
        const auto load = [&](const elem_t<DT> *line, int64_t step) {
            const int64_t k = step * (4 * E), left = p.K - k - g * E;
            i32x4 v = {0, 0, 0, 0};
            if (left >= E) {
                __builtin_memcpy(&v, line + k, 16);
            } else if (left > 0) {
                elem_t<DT> w[E];
#pragma unroll
                for (int x = 0; x < E; ++x) {
                    w[x] = Elem<DT>::put(0.0f);
                    if (x < left) w[x] = line[k + x];
                }
                __builtin_memcpy(&v, w, 16);
            }
            return v;
        };
        f32x4 acc[MT] = {};
        int64_t step = from;
        for (; step + U <= to && (step + U) * (4 * E) <= p.K; step += U) {
            i32x4 b[U], a[MT][U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                __builtin_memcpy(&b[u], pb + (step + u) * (4 * E), 16);
#pragma unroll
                for (int t = 0; t < MT; ++t) __builtin_memcpy(&a[t][u], pa[t] + (step + u) * (4 * E), 16);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int t = 0; t < MT; ++t) acc[t] = mma_chunk<DT>(b[u], a[t][u], acc[t]);
        }
        for (; step < to; ++step) {
            const i32x4 b = load(pb, step);
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] = mma_chunk<DT>(b, load(pa[t], step), acc[t]);
        }
        __syncthreads();   // the sums of the unit before have been read
#pragma unroll
        for (int t = 0; t < MT; ++t) sums[wave][t][lane] = acc[t];
        __syncthreads();
        if (wave < MT) {
            f32x4 v = sums[0][wave][lane];
#pragma unroll
            for (int w = 1; w < kFewWaves; ++w) v += sums[w][wave][lane];
            const int64_t m = wave * 16 + q, n = n0 + g * 4;
            const int left = (int)(p.N - n < 4 ? p.N - n : 4);
            float z[4] = {v[0], v[1], v[2], v[3]};
            if (m < p.M && left > 0) {
                if (left == 4) finish_at<true, DT, OT, 4>(p, e, m, n, 4, z);
                else finish_at<false, DT, OT, 4>(p, e, m, n, left, z);
            }
        }
    }
}

// At most 16 MT rows of a (the classes of a segmentation head) against many rows of b (positions): a is kept in
// LDS, swizzled like a tile's side; b streams through registers, 16 rows a wave with eight loads under way, and
// is read once, past the caches, as the results are written (4 x 307200 positions of 256 bf16 features to 40 float32
// planes: 191 us, 4.3 TB/s; with cached loads and stores 199, with 32 rows a wave 209).  The sum is a whole
// number of chunks.
template <int DT, int OT, int MT>
__global__ __launch_bounds__(256) void k_head(Product p, int pitch) {
    constexpr int SIZE = head_dtype_size(DT), E = 16 / SIZE, U = 8;
    using loose = int __attribute__((ext_vector_type(4), aligned(2)));   // 16 bytes at any element
    extern __shared__ __attribute__((aligned(16))) char weights[];
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, q = lane % 16, g = lane / 16;
    const int chunks = (int)(p.K / E);
    const auto slot = [&](int row, int c) { return weights + (row * pitch + (c ^ (row & 7))) * 16; };
    const int64_t per = (p.N + 15) / 16, groups = per * p.out_batches;
    const elem_t<DT> *a_rows = static_cast<const elem_t<DT> *>(p.a);
    for (int i = threadIdx.x; i < MT * 16 * pitch; i += 256) {
        const int row = i / pitch, c = i % pitch;
        i32x4 v = {0, 0, 0, 0};
        if (row < p.M && c < chunks) __builtin_memcpy(&v, a_rows + row * p.a_m + c * E, 16);
        *reinterpret_cast<i32x4 *>(slot(row, c)) = v;
    }
    __syncthreads();
    for (int64_t group = blockIdx.x * 4ll + wave; group < groups; group += gridDim.x * 4ll) {
        const int64_t e = group / per, n0 = group % per * 16;
        // rows behind the last one are read as the last one; their results are dropped
        const elem_t<DT> *pb = static_cast<const elem_t<DT> *>(p.b) + e * p.b_out + (n0 + q < p.N ? n0 + q : p.N - 1) * p.b_n;
        f32x4 acc[MT] = {};
        for (int c0 = 0; c0 < chunks; c0 += 4 * U) {
            i32x4 b[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = c0 + u * 4 + g, at = c < chunks ? c : chunks - 1;
                b[u] = __builtin_nontemporal_load(reinterpret_cast<const loose *>(pb + at * E));
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = c0 + u * 4 + g;
                if (c0 + u * 4 >= chunks) break;
                i32x4 a[MT];
#pragma unroll
                for (int t = 0; t < MT; ++t) a[t] = *reinterpret_cast<const i32x4 *>(slot(t * 16 + q, c));   // zero behind the sum's end
                if (c >= chunks) b[u] = i32x4{0, 0, 0, 0};
#pragma unroll
                for (int m = 0; m < MT; ++m) acc[m] = mma_chunk<DT>(b[u], a[m], acc[m]);
            }
        }
        const bool whole = n0 + 16 <= p.N;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int64_t m = t * 16 + q;
            if (m >= p.M) continue;
            const int64_t n = n0 + g * 4;
            float z[4] = {acc[t][0], acc[t][1], acc[t][2], acc[t][3]};
            if (whole) {
                finish_at<true, DT, OT, 4, true>(p, e, m, n, 4, z);
            } else {
                const int left = (int)(p.N - n < 4 ? p.N - n : 4);
                if (left > 0) finish_at<false, DT, OT, 4>(p, e, m, n, left, z);
            }
        }
    }
}

template <int DT, int OT, bool IK, bool JK>
void launch_tiles(const Product &p, hipStream_t st) {
    const auto go = [&](auto bi, auto bj, auto wi, auto wj, auto nbuf, auto d) {
        const int64_t tiles = (p.M + bi.value - 1) / bi.value * ((p.N + bj.value - 1) / bj.value) * p.out_batches;
        k_tiles<DT, OT, IK, JK, bi.value, bj.value, wi.value, wj.value, nbuf.value, d.value>
            <<<blocks(tiles * p.splits), wi.value * wj.value * 64, 0, st>>>(p);
    };
    using std::integral_constant;
    const integral_constant<int, 1> one{};
    const integral_constant<int, 2> two{};
    const integral_constant<int, 4> four{};
    const integral_constant<int, 64> narrow{};
    const integral_constant<int, 128> mid{};
    const integral_constant<int, 256> big{};
    if constexpr (DT != SSMAP_F32)
        if (p.shape == kTileBig) return go(big, big, two, four, two, std::true_type{});
    if (p.shape == kTileMid) go(mid, mid, two, two, two, std::true_type{});
    else if (p.shape == kTileLow) go(narrow, big, one, four, two, std::true_type{});
    else if (p.shape == kTileTall) go(big, narrow, four, one, two, std::true_type{});
    else if (p.shape == kTileSmall) go(narrow, narrow, two, two, four, std::true_type{});
    else if (p.shape == kTileSmallAny) go(narrow, narrow, two, two, two, std::false_type{});
    else go(mid, mid, two, two, two, std::false_type{});
}

// Lines of `dense` values to lines of `pitch` ones (a multiple of 16 bytes), filled up with zeros.
template <int DT>
__global__ __launch_bounds__(256) void k_pack(const elem_t<DT> *from, int64_t batch, int64_t line, int64_t batches, int64_t lines, int64_t dense,
                                              int64_t pitch, elem_t<DT> *to) {
    constexpr int E = 16 / sizeof(elem_t<DT>);
    const int64_t chunks = pitch / E, units = batches * lines * chunks;
    for (int64_t u = blockIdx.x * 256ll + threadIdx.x; u < units; u += gridDim.x * 256ll) {
        const int64_t c = u % chunks, l = u / chunks % lines, b = u / chunks / lines;
        const elem_t<DT> *src = from + b * batch + l * line + c * E;
        i32x4 v;
        if ((c + 1) * E <= dense) {
            __builtin_memcpy(&v, src, 16);
        } else {
            elem_t<DT> e[E];
#pragma unroll
            for (int q = 0; q < E; ++q) {
                e[q] = Elem<DT>::put(0.0f);
                if (c * E + q < dense) e[q] = src[q];
            }
            __builtin_memcpy(&v, e, 16);
        }
        *reinterpret_cast<i32x4 *>(to + u * E) = v;
    }
}

// Copies one operand (strides: dense across or along the sum; `blocks_in_sum` of it) behind p.parts and points at
// the copy.
template <int DT>
void pack_side(const Product &p, int64_t at, bool kc, int64_t rows, int64_t blocks_in_sum, const void *&side, int64_t &row, int64_t &k,
               int64_t &out, int64_t &sum, hipStream_t st) {
    if (at < 0) return;
    constexpr int64_t E = 16 / sizeof(elem_t<DT>);
    const int64_t lines = kc ? rows : p.K, dense = kc ? p.K : rows, pitch = (dense + E - 1) / E * E;
    const int64_t batches = p.sum_batches > 1 ? blocks_in_sum : out ? p.out_batches : 1;
    elem_t<DT> *to = reinterpret_cast<elem_t<DT> *>(reinterpret_cast<char *>(p.parts) + at);
    const int64_t units = batches * lines * (pitch / E);
    k_pack<DT><<<blocks((units + 255) / 256), 256, 0, st>>>(static_cast<const elem_t<DT> *>(side), p.sum_batches > 1 ? sum : out,
                                                            kc ? row : k, batches, lines, dense, pitch, to);
    side = to;
    (kc ? row : k) = pitch;
    if (out) out = lines * pitch;
    if (p.sum_batches > 1) sum = lines * pitch;
}

template <int DT, int OT>
void launch_product(Product p, hipStream_t st) {
    if (p.M * p.N * p.out_batches == 0) return;
    const bool ik = p.a_sums, jk = p.b_sums;
    pack_side<DT>(p, p.pack_a, ik, p.M, p.sum_batches, p.a, p.a_m, p.a_k, p.a_out, p.a_sum, st);
    pack_side<DT>(p, p.pack_b, jk, p.N, p.b_again, p.b, p.b_n, p.b_k, p.b_out, p.b_sum, st);
    if (p.shape == kFewRows) {
        const unsigned n = blocks((p.N + 15) / 16 * p.out_batches);
        if (p.M <= 16) k_few_rows<DT, OT, 1><<<n, kFewWaves * 64, 0, st>>>(p);
        else k_few_rows<DT, OT, 2><<<n, kFewWaves * 64, 0, st>>>(p);
        return;
    }
    if (p.shape == kHead) {
        const int size = head_dtype_size(DT);
        const int64_t groups = (p.N + 15) / 16 * p.out_batches, need = (groups + 3) / 4, bytes = head_bytes(p, size);
        const int64_t fit = 256 * (bytes > 40 << 10 ? 2 : bytes > 20 << 10 ? 4 : 8);   // blocks resident at once
        const unsigned n = (unsigned)(need < fit ? need : fit);
        const int pitch = (int)head_pitch(p, size), mt = (int)((p.M + 15) / 16);
        if (mt == 1) k_head<DT, OT, 1><<<n, 256, bytes, st>>>(p, pitch);
        else if (mt == 2) k_head<DT, OT, 2><<<n, 256, bytes, st>>>(p, pitch);
        else if (mt == 3) k_head<DT, OT, 3><<<n, 256, bytes, st>>>(p, pitch);
        else k_head<DT, OT, 4><<<n, 256, bytes, st>>>(p, pitch);
        return;
    }
    if (ik && jk) launch_tiles<DT, OT, true, true>(p, st);
    else if constexpr (DT == OT) {
        if (ik) launch_tiles<DT, OT, true, false>(p, st);
        else launch_tiles<DT, OT, false, false>(p, st);
    }
    if (p.splits > 1) {
        const int64_t quads = p.out_batches * p.M * ((p.N + 3) / 4);
        if (p.splits >= 32) k_join_parts<DT, OT, 16><<<blocks((quads + 15) / 16), 256, 0, st>>>(p);
        else k_join_parts<DT, OT, 1><<<blocks((quads + 255) / 256), 256, 0, st>>>(p);
    }
}

}  // namespace ssmap
