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

// One side of a tile: R rows (or columns) of it, C chunks of the sum's direction a stage, NT threads.
template <int DT, bool KC, int R, int C, int NT>
struct Side {
    static constexpr int SIZE = head_dtype_size(DT), E = 16 / SIZE, KB = C * E;   // values a chunk, a stage
    static constexpr int PER = R * C / NT, ROW = R / E;                           // chunks a thread; a row (not KC)
    static constexpr int BYTES = R * C * 16;
    static_assert((C == 4 || C == 8) && R * C % NT == 0 && (KC || ROW >= 8), "tile shape");

    static __device__ __forceinline__ int swizzle(int k) { return DT == SSMAP_F32 ? ((k >> 2) & 3) << 2 : (k & 3) << 1; }

    // KC: 128 bytes of consecutive slots hold eight rows' chunks of one c
    static __device__ __forceinline__ int turn(int row) { return C == 8 ? row & 7 : (row >> 1) & 3; }

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
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(
                             __builtin_amdgcn_readfirstlane(first + it * NT * 16)),
                         "v"(off[it]), "s"(desc)
                         : "memory");
        }
    }

    // Through registers, for any alignment and extent.
    static __device__ __forceinline__ void load(i32x4 (&reg)[PER], const char *base, int rows, int ks, int64_t ld) {
#pragma unroll
        for (int it = 0; it < PER; ++it) {
            int line, c;
            place(it * NT + threadIdx.x, line, c);
            const int n = count(line, c, rows, ks);
            const char *p = base + line * ld + c * 16;
            i32x4 v = {0, 0, 0, 0};
            if (n == E) {
                __builtin_memcpy(&v, p, 16);
            } else {
                elem_t<DT> e[E];
#pragma unroll
                for (int q = 0; q < E; ++q) {
                    e[q] = Elem<DT>::put(0.0f);
                    if (q < n) e[q] = reinterpret_cast<const elem_t<DT> *>(p)[q];
                }
                __builtin_memcpy(&v, e, 16);
            }
            reg[it] = v;
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

// N results next to each other (n, n + 1, ...), of which `left` exist.  `o` is the first one's place in the
// dense output.
template <int DT, int OT, int N>
__device__ __forceinline__ void finish(const Product &p, int64_t o, int64_t e, int64_t m, int64_t n, int left, float (&z)[N]) {
    const auto each = [&](auto f) {
#pragma unroll
        for (int q = 0; q < N; ++q)
            if (q < left) f(q);
    };
    const auto get = [&](auto tag, const void *from, int64_t at, float (&v)[N]) {
        constexpr int T = decltype(tag)::value;
        const elem_t<T> *src = static_cast<const elem_t<T> *>(from) + at;
        if (left >= N) {
            elem_t<T> w[N];
            __builtin_memcpy(w, src, sizeof w);
#pragma unroll
            for (int q = 0; q < N; ++q) v[q] = Elem<T>::get(w[q]);
        } else {
            each([&](int q) { v[q] = Elem<T>::get(src[q]); });
        }
    };
    const auto put = [&](auto tag, void *to) {
        constexpr int T = decltype(tag)::value;
        elem_t<T> *dst = static_cast<elem_t<T> *>(to) + o, w[N];
#pragma unroll
        for (int q = 0; q < N; ++q) w[q] = Elem<T>::put(z[q]);
        if (left >= N) __builtin_memcpy(dst, w, sizeof w);
        else each([&](int q) { dst[q] = w[q]; });
    };
    using D = std::integral_constant<int, DT>;
    using O = std::integral_constant<int, OT>;
    using F = std::integral_constant<int, SSMAP_F32>;
    float v[N] = {};
    if (p.bias) {
        if (p.bias_along_m) {
            const float b = p.bias_f32 ? static_cast<const float *>(p.bias)[m] : Elem<DT>::get(static_cast<const elem_t<DT> *>(p.bias)[m]);
#pragma unroll
            for (int q = 0; q < N; ++q) z[q] += b;
        } else {
            if (p.bias_f32) get(F{}, p.bias, n, v);
            else get(D{}, p.bias, n, v);
#pragma unroll
            for (int q = 0; q < N; ++q) z[q] += v[q];
        }
    }
    if (p.pre) put(D{}, p.pre);
    if (p.act) {
#pragma unroll
        for (int q = 0; q < N; ++q) z[q] = activate<OT == SSMAP_F32>(z[q], p.act);
    }
    if (p.res) {
        get(O{}, p.res, e * p.res_out + m * p.res_m + n, v);
#pragma unroll
        for (int q = 0; q < N; ++q) z[q] += v[q];
    }
    put(O{}, p.out);
}

// BI x BJ results a block, WI x WJ waves, stages of C chunks in NBUF buffers.  DIRECT: both sides go straight to
// LDS (see Side::fetch), NBUF - 1 stages ahead; otherwise through registers, one stage ahead.
template <int DT, int OT, bool IK, bool JK, int BI, int BJ, int WI, int WJ, int C, int NBUF, bool DIRECT>
__global__ __launch_bounds__(WI *WJ * 64) void k_tiles(Product p) {
    constexpr int NT = WI * WJ * 64, TI = BI / WI / 16, TJ = BJ / WJ / 16, SIZE = head_dtype_size(DT);
    using I = Side<DT, IK, BI, C, NT>;
    using J = Side<DT, JK, BJ, C, NT>;
    constexpr int PITCH = TJ * 16 + 4;                 // floats a row while results are turned: four off, for the banks
    constexpr int HI = TI > 4 ? TI / 2 : TI;           // rows of 16 turned at once
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
        const int64_t part = p.part_steps * (8 / C);   // planned in stages of eight chunks
        const int64_t first = split * part, last = first + part < all_steps ? first + part : all_steps;
        const int64_t ld_i = (IK ? p.a_m : p.a_k) * SIZE, ld_j = (JK ? p.b_n : p.b_k) * SIZE;
        const int64_t step_i = (IK ? 1 : p.a_k) * (int64_t)(I::KB * SIZE), step_j = (JK ? 1 : p.b_k) * (int64_t)(I::KB * SIZE);
        const char *pa = static_cast<const char *>(p.a) + (e * p.a_out + i0 * p.a_m) * SIZE;
        const char *pb = static_cast<const char *>(p.b) + (e * p.b_out + j0 * p.b_n) * SIZE;
        int64_t at = first % (steps ? steps : 1);      // stage within its sum batch
        pa += first / (steps ? steps : 1) * p.a_sum * SIZE + at * step_i;
        pb += first / (steps ? steps : 1) * p.b_sum * SIZE + at * step_j;
        const auto advance = [&] {
            if (++at == steps) {
                at = 0;
                pa += p.a_sum * SIZE - (steps - 1) * step_i;
                pb += p.b_sum * SIZE - (steps - 1) * step_j;
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
        }
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
                I::load(reg_i, pa, rows_i, ks, ld_i);
                J::load(reg_j, pb, rows_j, ks, ld_j);
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
        const auto read = [&](int buf, int kk) {
            const char *li = stage(buf), *lj = li + I::BYTES;
#pragma unroll
            for (int i = 0; i < TI; ++i) fi[i] = I::read(li, (wi * TI + i) * 16, kk);
#pragma unroll
            for (int j = 0; j < TJ; ++j) fj[j] = J::read(lj, (wj * TJ + j) * 16, kk);
        };
        const auto multiply = [&] {
#pragma unroll
            for (int i = 0; i < TI; ++i)
#pragma unroll
                for (int j = 0; j < TJ; ++j) acc[i][j] = mma_chunk<DT>(fj[j], fi[i], acc[i][j]);
        };
        if constexpr (WI * WJ == 8) {
            // Two waves a SIMD take turns: while one multiplies half a stage, the other reads its next half from
            // LDS.  The second four waves run one turn behind.  A barrier ends each turn; the scheduler moves
            // nothing over it.  With turns 4t ... 4t + 3 of the first waves for stage t (read, multiply, read,
            // multiply), the second waves read stage t for the last time in turn 4t + 3: in turn 4t + 4 both send
            // for stage t + 2, into the same buffer, and at the end of turn 4t + 7 both have waited for it.
            static_assert(DIRECT && C == 8 && NBUF == 2, "two turns a stage");
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
                if (late) {
                    if (first + 1 < last) fetch(1);
                    turn_ends();
                }
                for (int64_t t = first; t < last; ++t) {
                    const int buf = (int)((t - first) & 1);
                    if (!late && t + 1 < last) fetch(buf ^ 1);
                    read(buf, 0);
                    have_read();
                    turn_ends();
                    __builtin_amdgcn_s_setprio(1);
                    multiply();
                    __builtin_amdgcn_s_setprio(0);
                    turn_ends();
                    read(buf, 1);
                    if (late) have_landed();
                    have_read();
                    turn_ends();
                    if (late && t + 2 < last) fetch(buf);
                    __builtin_amdgcn_s_setprio(1);
                    multiply();
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
#pragma unroll
                for (int kk = 0; kk < C / 4; ++kk) {
                    read(buf, kk);
                    multiply();
                }
                if (more) keep(next);
                buf = buf + 1 == NBUF ? 0 : buf + 1;
            }
        }
        __syncthreads();   // nobody reads the stages any more
        // Each wave turns its own results round in LDS, HI rows of 16 at a time: out of the registers with four
        // neighbouring n a lane, back with eight, so that the epilogue is one loop over whole rows.
        const int lane = threadIdx.x % 64, q = lane % 16, g = lane / 16;
        float *turn = reinterpret_cast<float *>(lds_all + wave * (HI * 16 * PITCH * 4));
#pragma unroll
        for (int h = 0; h < TI / HI; ++h) {
#pragma unroll
            for (int i = 0; i < HI; ++i)
#pragma unroll
                for (int j = 0; j < TJ; ++j) *reinterpret_cast<f32x4 *>(turn + (i * 16 + q) * PITCH + j * 16 + g * 4) = acc[h * HI + i][j];
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");   // the wave's own writes, in order
            __builtin_amdgcn_wave_barrier();
            constexpr int LINE = TJ * 16 / 8;   // lanes a row
#pragma unroll 1
            for (int u = lane; u < HI * 16 * LINE; u += 64) {
                const int row = u / LINE, col = u % LINE * 8;
                const int64_t m = i0 + (wi * TI + h * HI) * 16 + row, n = j0 + wj * TJ * 16 + col;
                const int left = (int)(p.N - n < 8 ? p.N - n : 8);
                if (m >= p.M || left <= 0) continue;
                const int64_t o = (e * p.M + m) * p.N + n;
                float z[8];
                __builtin_memcpy(z, turn + row * PITCH + col, 32);
                if (p.splits > 1) {
                    float *part = p.parts + split * p.out_batches * p.M * p.N + o;
                    if (left == 8) __builtin_memcpy(part, z, 32);
                    else {
#pragma unroll
                        for (int s = 0; s < 8; ++s)
                            if (s < left) part[s] = z[s];
                    }
                } else {
                    finish<DT, OT, 8>(p, o, e, m, n, left, z);
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
        if (part == 0 && u0 + quad < units) finish<DT, OT, 4>(p, o, e, m, n, left, z);
    }
}

// At most 16 MT rows of a (single tokens, small batches) against all of b: reading b once is all the work.  A
// block takes 16 rows of b, its eight waves share the sum; both operands go from memory to registers as the
// matrix instruction wants them, eight loads of b under way in each wave.
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
            if (m < p.M && left > 0) finish<DT, OT, 4>(p, (e * p.M + m) * p.N + n, e, m, n, left, z);
        }
    }
}

template <int DT, int OT, bool IK, bool JK>
void launch_tiles(const Product &p, hipStream_t st) {
    const auto go = [&](auto bi, auto bj, auto wi, auto wj, auto c, auto nbuf, auto d) {
        const int64_t tiles = (p.M + bi.value - 1) / bi.value * ((p.N + bj.value - 1) / bj.value) * p.out_batches;
        k_tiles<DT, OT, IK, JK, bi.value, bj.value, wi.value, wj.value, c.value, nbuf.value, d.value><<<blocks(tiles * p.splits), wi.value * wj.value * 64, 0, st>>>(p);
    };
    using std::integral_constant;
    const integral_constant<int, 1> one{};
    const integral_constant<int, 2> two{};
    const integral_constant<int, 4> four{};
    const integral_constant<int, 8> eight{};
    const integral_constant<int, 64> narrow{};
    const integral_constant<int, 128> mid{};
    const integral_constant<int, 256> big{};
    if constexpr (DT != SSMAP_F32)
        if (p.shape == kTileBig) return go(big, big, two, four, eight, two, std::true_type{});
    if (p.shape == kTileMid) go(mid, mid, two, two, eight, two, std::true_type{});
    else if (p.shape == kTileLow) go(narrow, big, one, four, eight, two, std::true_type{});
    else if (p.shape == kTileTall) go(big, narrow, four, one, eight, two, std::true_type{});
    else go(mid, mid, two, two, eight, two, std::false_type{});
}

template <int DT, int OT>
void launch_product(const Product &p, hipStream_t st) {
    if (p.M * p.N * p.out_batches == 0) return;
    if (p.shape == kFewRows) {
        const unsigned n = blocks((p.N + 15) / 16 * p.out_batches);
        if (p.M <= 16) k_few_rows<DT, OT, 1><<<n, kFewWaves * 64, 0, st>>>(p);
        else k_few_rows<DT, OT, 2><<<n, kFewWaves * 64, 0, st>>>(p);
        return;
    }
    if (p.a_k == 1 && p.b_k == 1) launch_tiles<DT, OT, true, true>(p, st);
    else if constexpr (DT == OT) {
        if (p.a_k == 1) launch_tiles<DT, OT, true, false>(p, st);
        else launch_tiles<DT, OT, false, false>(p, st);
    }
    if (p.splits > 1) {
        const int64_t quads = p.out_batches * p.M * ((p.N + 3) / 4);
        if (p.splits >= 32) k_join_parts<DT, OT, 16><<<blocks((quads + 15) / 16), 256, 0, st>>>(p);
        else k_join_parts<DT, OT, 1><<<blocks((quads + 255) / 256), 256, 0, st>>>(p);
    }
}

}  // namespace ssmap
