// dimn_xent_thin.h -- the products of dimn_xent.h for few rows (gfx950): one pass over the kernel, operands in the caller's own layout.
//
// With few rows the logits, dx and dW are bound by reading (or writing) the kernel once, and what dimn_xent.h does first -- laying the operands
// out as k-contiguous bfloat16 planes -- costs more than the products: for float32 it moves 16 bytes per weight where 4 have to be read.  Here
// the matrix instructions take their operands straight from global memory, in whichever order the caller holds the kernel:
//   * k-contiguous (KC): a lane gets 16 bytes of one class row; float32: element r feeds instruction r (any assignment of k's to the slots of
//     v_mfma_f32_16x16x4_f32 gives the same sum as long as the rows' operand follows it); bfloat16: the eight k's of one 16x16x32 instruction.
//   * class-contiguous (VC): a lane loads four consecutive classes of one k; element j belongs to class set j, whose sixteen classes lie four
//     apart -- a permutation of the classes inside the workgroup's 64 that the epilogue undoes.
// float32 runs on the exact float32 matrix instructions: at 64 rows their rate (154 TFLOP/s measured) and the HBM's meet.
// Measured: one row x 1024 x 32000 bfloat16 14.1 us = 4.6 TB/s; 12 x 2000 x 40000 bfloat16 dx 28 us = 5.7 TB/s (part of the kernel still lies in the
// memory-side cache); 12 x 3648 x 22455 float32 dx 69, dW 62 us = 4.7, 5.3 TB/s, class-contiguous logits (backward) 129 us = 2.5 TB/s; 128 x 2922 x 25664
// float32 218 / 266 / 229 us (logits / dx / dW), 88 / 72 / 84 TFLOP/s.
// A workgroup owns 32 (KC) / 64 (VC) classes x up to 64 rows; its waves (four, or sixteen where there are few workgroups and a long inner
// dimension: 3840 x 222 float32 ran 45 us with four) share the chunks of k and are added through LDS, upper half onto lower half, in a fixed order.
#pragma once
#include "dimn_xent.h"

namespace rowops {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8u __attribute__((ext_vector_type(8), aligned(2)));

struct Thin {
    const void* A; int64_t lda;                // [M][K], k-contiguous
    const void* B; int64_t ldb;                // KC: [N][K]; VC: [K][N]
    int64_t M, N, K;
    const float* bias;                         // [N] or NULL
    const void* target; int64_t target_row; int32_t target_kind;
    float2* part; float2* part_t; float* picked;          // as XentGemm (a tile: 32 / 64 classes)
    const float* lse; const float* dloss; const float* tsum;
    void* G; int64_t ldg;                      // [M][ldg] of T
    float* dbias_part;                         // [row blocks][N]
    float* acc;                                // XE_ADD: [k-ranges][M][N] float32
    void* C; int64_t ldc;                      // XE_STORE: [M][N] of T
};

template <typename T> struct Four;             // four consecutive elements of a class row (VC)
template <> struct Four<float> { typedef f32x4u vec; };
template <> struct Four<bf16_t> { typedef u16x4u vec; };

// the 4 x 4 of v[t] over the lanes of a quad, transposed: lane q's v[t] becomes lane t's v[q] (li: the lane's number)
template <typename V>
__device__ __forceinline__ void quad_transpose(V (&v)[4], int li) {
    constexpr int D = sizeof(V) / 4;
    typedef uint32_t words __attribute__((ext_vector_type(D)));
    words w[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) w[t] = __builtin_bit_cast(words, v[t]);
    const bool odd = li & 1, high = li & 2;
    auto swap = [](uint32_t& x, uint32_t& y, bool upper, auto ctrl) {
        const uint32_t fx = __builtin_amdgcn_mov_dpp((int)x, decltype(ctrl)::value, 15, 15, true), fy = __builtin_amdgcn_mov_dpp((int)y, decltype(ctrl)::value, 15, 15, true);
        x = upper ? fy : x;
        y = upper ? y : fx;
    };
    constexpr std::integral_constant<int, 0xB1> by_one{};       // quad_perm [1, 0, 3, 2]
    constexpr std::integral_constant<int, 0x4E> by_two{};       // quad_perm [2, 3, 0, 1]
#pragma unroll
    for (int e = 0; e < D; ++e) {
        uint32_t x[4] = {w[0][e], w[1][e], w[2][e], w[3][e]};
        swap(x[0], x[1], odd, by_one);
        swap(x[2], x[3], odd, by_one);
        swap(x[0], x[2], high, by_two);
        swap(x[1], x[3], high, by_two);
#pragma unroll
        for (int t = 0; t < 4; ++t) w[t][e] = x[t];
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) v[t] = __builtin_bit_cast(V, w[t]);
}

// (class tile, k-range, row block) of one workgroup; `ranges` k-ranges in all.  FOURS: sets of four chunks per wave in registers (0: chunks one by one)
template <typename T, bool VC, int NF, int EPI, int NW, int FOURS>
__device__ __forceinline__ void thin_product(const Thin& p, int tile, int range, int ranges, int block) {
    constexpr bool BF = sizeof(T) == 2, WIDE = BF && !VC;      // WIDE: the 16x16x32 instruction, eight k's per lane
    constexpr int EL = WIDE ? 8 : 4, KS = 4 * EL, NS = VC ? 4 : 2, CW = VC ? 64 : 32, ROWS = 16 * NF, LD = CW + 4;
    __shared__ __attribute__((aligned(16))) float red[NW / 2][ROWS][LD];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 15, lj = lane >> 4;
    const int64_t c0 = (int64_t)tile * CW, m0 = (int64_t)block * ROWS;
    const T* A = (const T*)p.A;
    const T* B = (const T*)p.B;
    typedef typename std::conditional<BF, typename std::conditional<WIDE, u16x8u, u16x4u>::type, f32x4u>::type avec;
    typedef typename std::conditional<VC, typename Four<T>::vec, avec>::type bvec;
    constexpr int NB = VC ? 4 : 2;
    f32x4 acc[NF][NS];
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int s = 0; s < NS; ++s) acc[f][s] = (f32x4){0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](const avec (&ra)[NF], const bvec (&rb)[NB]) {
        if constexpr (WIDE) {
#pragma unroll
            for (int f = 0; f < NF; ++f)
#pragma unroll
                for (int s = 0; s < NS; ++s)
                    acc[f][s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, rb[s]), __builtin_bit_cast(bf8, ra[f]), acc[f][s], 0, 0, 0);
        } else if constexpr (BF) {
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const s16x4 w = {(short)rb[0][s], (short)rb[1][s], (short)rb[2][s], (short)rb[3][s]};
#pragma unroll
                for (int f = 0; f < NF; ++f) acc[f][s] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(w, __builtin_bit_cast(s16x4, ra[f]), acc[f][s], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int f = 0; f < NF; ++f)
#pragma unroll
                    for (int s = 0; s < NS; ++s) acc[f][s] = __builtin_amdgcn_mfma_f32_16x16x4f32(VC ? rb[r][s] : rb[s][r], ra[f][r], acc[f][s], 0, 0, 0);
        }
    };
    // this workgroup's range of whole chunks; the chunk that crosses K belongs to the last range
    const int64_t whole = p.K / KS;
    const int64_t cbeg = whole * range / ranges, cend = whole * (range + 1) / ranges;
    // Four chunks at a time.  A lane that loaded its own 16 bytes of sixteen rows would have each lane looked up by itself (64 cache accesses per
    // load measured, one per cycle and CU: 128 x 2922 x 25664 float32 dx was bound by them, 335 us).  So the lanes of a quad read 64 consecutive
    // bytes of a row, in four loads those of four rows, and transpose the 4 x 4 among them: element [u] of a lane is then the 16 bytes at
    // k + EL (4 lj + u) of its own row.  Offsets from the workgroup's first row take 32 bits (rows further apart, and rows
    // in descending order, whose offsets are negative, go chunk by chunk below).
    const int64_t nc = FOURS > 0 && p.lda >= 0 && p.ldb >= 0 && p.lda < (1 << 24) && p.ldb < (1 << 24) ? cend - cbeg : 0;
    const int64_t full = nc / (4 * NW), left = nc % (4 * NW);
    const int quads = left > 2 * NW ? (int)left / 4 : 0;         // waves that take four more chunks: what is left over would cost as many single ones
    const int64_t rounds = full + (wave < quads);
    if constexpr (FOURS > 0) {
        const int quad = li & ~3, part = 4 * lj + (li & 3);
        const char* abase = (const char*)(A + m0 * p.lda);
        const char* bbase = (const char*)(VC ? B : B + c0 * p.ldb);
        uint32_t aoff[NF][4], boff[VC ? 1 : 2][4];
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int64_t r = m0 + 16 * f + quad + t;           // rows and classes past the end repeat the last one: never stored
                aoff[f][t] = (uint32_t)(((r < p.M ? r : p.M - 1) - m0) * p.lda + EL * part) * (uint32_t)sizeof(T);
            }
        if constexpr (VC) {
            const int64_t c = c0 + 4 * li;
            boff[0][0] = (uint32_t)(16 * lj * p.ldb) * (uint32_t)sizeof(T);
            bbase += (c0 < p.N - 4 ? c0 : p.N - 4) * (int64_t)sizeof(T);
            boff[0][0] += (uint32_t)((c < p.N - 4 ? c : p.N - 4) - (c0 < p.N - 4 ? c0 : p.N - 4)) * (uint32_t)sizeof(T);     // (N >= 4: the caller's rule)
        } else {
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int64_t r = c0 + 16 * s + quad + t;
                    boff[s][t] = (uint32_t)(((r < p.N ? r : p.N - 1) - c0) * p.ldb + EL * part) * (uint32_t)sizeof(T);
                }
        }
        const auto place = [&](int64_t i) -> int64_t {              // first k of the wave's round i (past its last: of the last)
            i = i < rounds ? i : rounds - 1;
            return (cbeg + (i < full ? 4 * (NW * i + wave) : 4 * NW * full + 4 * wave)) * KS;
        };
        const auto read_rows = [&](int64_t k, avec (&a)[NF][4]) {
            const char* ak = abase + k * (int64_t)sizeof(T);
#pragma unroll
            for (int f = 0; f < NF; ++f)
#pragma unroll
                for (int t = 0; t < 4; ++t) a[f][t] = *(const avec*)(ak + aoff[f][t]);
        };
        const auto chunk = [&](const avec (&a)[NF][4], int u, const bvec (&rb)[NB]) {
            avec ra[NF];
#pragma unroll
            for (int f = 0; f < NF; ++f) ra[f] = a[f][u];
            multiply(ra, rb);
        };
        // (the barriers below keep the compiler from moving every load down to its use)
        if constexpr (VC) {
            // classes: a chunk ahead; rows: a round ahead
            avec a[2][NF][4];
            bvec b[2][NB];
            const auto read_classes = [&](int64_t k, int u) {
                const char* bk = bbase + (k + 4 * u) * p.ldb * (int64_t)sizeof(T);
#pragma unroll
                for (int q = 0; q < 4; ++q) b[u & 1][q] = *(const bvec*)(bk + q * p.ldb * (int64_t)sizeof(T) + boff[0][0]);
            };
            const auto round = [&](int64_t i, int set) {
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    read_classes(place(i + (u == 3)), (u + 1) & 3);
                    if (u == 0) read_rows(place(i + 1), a[set ^ 1]);
                    __builtin_amdgcn_sched_barrier(0);
                    if (u == 0)
#pragma unroll
                        for (int f = 0; f < NF; ++f) quad_transpose(a[set][f], li);
                    chunk(a[set], u, b[u & 1]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            if (rounds > 0) {
                read_rows(place(0), a[0]);
                read_classes(place(0), 0);
                for (int64_t i = 0; i + 1 < rounds; i += 2) { round(i, 0); round(i + 1, 1); }
                if (rounds & 1) round(rounds - 1, 0);
            }
        } else {
            avec a[FOURS][NF][4];
            bvec b[FOURS][NB][4];
            const auto fetch = [&](int64_t i, int set) {
                const int64_t k = place(i);
                const char* bk = bbase + k * (int64_t)sizeof(T);
#pragma unroll
                for (int q = 0; q < NB; ++q)
#pragma unroll
                    for (int t = 0; t < 4; ++t) b[set][q][t] = *(const bvec*)(bk + boff[q][t]);
                read_rows(k, a[set]);
                __builtin_amdgcn_sched_barrier(0);
            };
            const auto consume = [&](int set) {
#pragma unroll
                for (int f = 0; f < NF; ++f) quad_transpose(a[set][f], li);
#pragma unroll
                for (int q = 0; q < NB; ++q) quad_transpose(b[set][q], li);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    bvec rb[NB];
#pragma unroll
                    for (int q = 0; q < NB; ++q) rb[q] = b[set][q][u];
                    chunk(a[set], u, rb);
                }
                __builtin_amdgcn_sched_barrier(0);
            };
            if constexpr (FOURS == 1) {
                for (int64_t i = 0; i < rounds; ++i) { fetch(i, 0); consume(0); }
            } else if (rounds > 0) {
                fetch(0, 0);
                for (int64_t i = 0; i + 1 < rounds; i += 2) {
                    fetch(i + 1, FOURS - 1);
                    consume(0);
                    fetch(i + 2, 0);
                    consume(FOURS - 1);
                }
                if (rounds & 1) consume(0);
            }
        }
    }
    // single chunks, from the first wave without four more; then the chunk that crosses K
    const T* arow[NF];
    const T* bptr[VC ? 1 : 2];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
        const int64_t m = m0 + 16 * f + li;
        arow[f] = A + (m < p.M ? m : p.M - 1) * p.lda;
    }
    if constexpr (VC) {
        const int64_t c = c0 + 4 * li;
        bptr[0] = B + (c < p.N - 4 ? c : p.N - 4);
    } else {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int64_t c = c0 + 16 * s + li;
            bptr[s] = B + (c < p.N ? c : p.N - 1) * p.ldb;
        }
    }
    avec ra[NF];
    bvec rb[NB];
    const int64_t single = cbeg + 4 * NW * full + 4 * quads;
    const int turn = (wave + NW - quads % NW) % NW;
    for (int64_t c = single + turn; c < cend; c += NW) {
#pragma unroll
        for (int q = 0; q < NB; ++q) {
            if constexpr (VC) rb[q] = *(const bvec*)(bptr[0] + (c * KS + 4 * lj + q) * p.ldb);
            else rb[q] = *(const bvec*)(bptr[q] + c * KS + EL * lj);
        }
#pragma unroll
        for (int f = 0; f < NF; ++f) ra[f] = *(const avec*)(arow[f] + c * KS + EL * lj);
        multiply(ra, rb);
    }
    if (whole * KS < p.K && range == ranges - 1 && turn == (int)((cend - single) % NW)) {
        const int64_t k = whole * KS;
#pragma unroll
        for (int q = 0; q < NB; ++q)
#pragma unroll
            for (int i = 0; i < (VC ? 4 : EL); ++i) {
                if constexpr (VC) rb[q][i] = k + 4 * lj + q < p.K ? bptr[0][(k + 4 * lj + q) * p.ldb + i] : (T)0;
                else rb[q][i] = k + EL * lj + i < p.K ? bptr[q][k + EL * lj + i] : (T)0;
            }
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int i = 0; i < EL; ++i) ra[f][i] = k + EL * lj + i < p.K ? arow[f][k + EL * lj + i] : (T)0;
        multiply(ra, rb);
    }
    // element r of acc[f][s]: row 16 f + li, position 16 s + 4 lj + r (KC) / 4 (4 lj + r) + s (VC) of the workgroup's classes
    auto put = [&](int slot) {
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int q = 0; q < NS; ++q) {
                if constexpr (VC) *(f32x4*)&red[slot][16 * f + li][16 * lj + 4 * q] = (f32x4){acc[f][0][q], acc[f][1][q], acc[f][2][q], acc[f][3][q]};
                else *(f32x4*)&red[slot][16 * f + li][16 * q + 4 * lj] = acc[f][q];
            }
    };
#pragma unroll
    for (int half = NW / 2; half >= 2; half >>= 1) {
        if (wave >= half && wave < 2 * half) put(wave - half);
        __syncthreads();
        if (wave < half) {
#pragma unroll
            for (int f = 0; f < NF; ++f)
#pragma unroll
                for (int q = 0; q < NS; ++q) {
                    if constexpr (VC) {
                        const f32x4 t = *(const f32x4*)&red[wave][16 * f + li][16 * lj + 4 * q];
#pragma unroll
                        for (int s = 0; s < 4; ++s) acc[f][s][q] += t[s];
                    } else acc[f][q] += *(const f32x4*)&red[wave][16 * f + li][16 * q + 4 * lj];
                }
        }
        __syncthreads();
    }
    if (wave < 2) put(wave);
    __syncthreads();
    // PT threads per row, CPT consecutive positions each, in groups of four whose classes are consecutive
    constexpr int CPT = CW * ROWS / (64 * NW) < 4 ? 4 : CW * ROWS / (64 * NW), PT = CW / CPT, NG = CPT / 4;
    const int row = tid / PT, pos0 = (tid % PT) * CPT;
    const int64_t m = m0 + row;
    const bool have = row < ROWS && m < p.M;
    // first class of a group, and how many of its four classes belong to another group (VC: the last one is moved back to end with the classes) or are none
    auto group = [&](int pos, int& before, int& upto) -> int64_t {
        const int64_t from = c0 + pos;
        if constexpr (VC) {
            const int64_t start = from < p.N - 4 ? from : p.N - 4;
            before = from - start < 4 ? (int)(from - start) : 4;
            upto = 4;
            return start;
        } else {
            before = 0;
            upto = from + 4 <= p.N ? 4 : (from < p.N ? (int)(p.N - from) : 0);
            return from;
        }
    };
    f32x4 z[NG];
    if (row < ROWS) {
#pragma unroll
        for (int q = 0; q < NG; ++q) z[q] = *(const f32x4*)&red[0][row][pos0 + 4 * q] + *(const f32x4*)&red[1][row][pos0 + 4 * q];
    }
    if constexpr (EPI == XE_ADD || EPI == XE_STORE) {
        if (!have) return;
#pragma unroll
        for (int q = 0; q < NG; ++q) {
            int before, upto;
            const int64_t k = group(pos0 + 4 * q, before, upto);
            if constexpr (EPI == XE_ADD) {
                float* to = p.acc + ((int64_t)range * p.M + m) * p.N + k;
                if (before == 0 && upto == 4) *(f32x4u*)to = z[q];
                else
#pragma unroll
                    for (int i = 0; i < 4; ++i) if (i >= before && i < upto) to[i] = z[q][i];
            } else {
                T* to = (T*)p.C + m * p.ldc + k;
                typename Four<T>::vec o;
#pragma unroll
                for (int i = 0; i < 4; ++i) { if constexpr (BF) o[i] = to_bf16(z[q][i]); else o[i] = z[q][i]; }
                if (before == 0 && upto == 4) *(typename Four<T>::vec*)to = o;
                else
#pragma unroll
                    for (int i = 0; i < 4; ++i) if (i >= before && i < upto) to[i] = o[i];
            }
        }
        return;
    }
    if constexpr (EPI == XE_LSE || EPI == XE_GRAD) {
        const bool labels = p.target_kind <= XT_I64;
        int64_t y = -1;
        if (labels && have) y = p.target_kind == XT_I64 ? ((const int64_t*)p.target)[m] : (int64_t)((const int32_t*)p.target)[m];
        f32x4 t[NG];
#pragma unroll
        for (int q = 0; q < NG; ++q) {
            t[q] = (f32x4){0.f, 0.f, 0.f, 0.f};
            int before, upto;
            const int64_t k = group(pos0 + 4 * q, before, upto);
            if (!have || upto == 0) continue;
            if (p.bias) {
                f32x4 b4 = {0.f, 0.f, 0.f, 0.f};
                if (upto == 4) b4 = *(const f32x4u*)(p.bias + k);
                else
#pragma unroll
                    for (int i = 0; i < 4; ++i) if (i < upto) b4[i] = p.bias[k + i];
                z[q] += b4;
            }
            if (!labels) t[q] = xent_profile4(p.target, p.target_kind, p.target_row, m, k, p.N);
        }
        if constexpr (EPI == XE_LSE) {
            float top = -INFINITY, s = 0.f, st = 0.f, stz = 0.f;
#pragma unroll
            for (int q = 0; q < NG; ++q) {
                int before, upto;
                const int64_t k = group(pos0 + 4 * q, before, upto);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (i < before || i >= upto) continue;
                    top = fmaxf(top, z[q][i]);
                    if (have && labels && k + i == y) p.picked[m] = z[q][i];
                    st += t[q][i];
                    stz += t[q][i] != 0.f ? t[q][i] * z[q][i] : 0.f;
                }
            }
#pragma unroll
            for (int o = 1; o < PT; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
            const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int q = 0; q < NG; ++q) {
                int before, upto;
                group(pos0 + 4 * q, before, upto);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i >= before && i < upto) s += BF ? __expf(z[q][i] - ref) : expf(z[q][i] - ref);
            }
#pragma unroll
            for (int o = 1; o < PT; o <<= 1) { s += __shfl_xor(s, o); st += __shfl_xor(st, o); stz += __shfl_xor(stz, o); }
            if (have && tid % PT == 0) {
                const int64_t at = (int64_t)tile * p.M + m;
                p.part[at] = make_float2(top, s);
                if (!labels) p.part_t[at] = make_float2(st, stz);
            }
        } else {
            const float lse = have ? p.lse[m] : 0.f, d = have && (!labels || (y >= 0 && y < p.N)) ? p.dloss[m] : 0.f, ts = labels ? 1.f : (have ? p.tsum[m] : 0.f);     // (a label that is no class: no gradient)
            __syncthreads();                                    // the products have been read: the first slot takes G for the sums over the rows
#pragma unroll
            for (int q = 0; q < NG; ++q) {
                int before, upto;
                const int64_t k = group(pos0 + 4 * q, before, upto);
                f32x4 g;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = z[q][i] == -INFINITY ? 0.f : (BF ? __expf(z[q][i] - lse) : expf(z[q][i] - lse));
                    const float hot = labels ? (k + i == y ? 1.f : 0.f) : t[q][i];
                    g[i] = d != 0.f ? d * (ts * e - hot) : 0.f;
                }
                if (row < ROWS) *(f32x4*)&red[0][row][pos0 + 4 * q] = g;
                if (!have) continue;
                T* to = (T*)p.G + m * p.ldg + k;
                typename Four<T>::vec o;
#pragma unroll
                for (int i = 0; i < 4; ++i) { if constexpr (BF) o[i] = to_bf16(g[i]); else o[i] = g[i]; }
                if (before == 0 && upto == 4) *(typename Four<T>::vec*)to = o;
                else
#pragma unroll
                    for (int i = 0; i < 4; ++i) if (i >= before && i < upto) to[i] = o[i];
            }
            if (!p.dbias_part) return;
            __syncthreads();
            constexpr int ST = 256 / CW;                        // strands of rows per class
            const int pos = tid % CW, strand = tid / CW;
            float s = 0.f;
            if (tid < 256)
#pragma unroll 8
                for (int r = strand; r < ROWS; r += ST) s += red[0][r][pos];
            __syncthreads();
            if (tid < 256) red[1][strand][pos] = s;
            __syncthreads();
            if (strand == 0) {
                int before, upto;
                const int64_t k = group(pos & ~3, before, upto);
#pragma unroll
                for (int w = 1; w < ST; ++w) s += red[1][w][pos];
                if ((pos & 3) >= before && (pos & 3) < upto) p.dbias_part[(int64_t)block * p.N + k + (pos & 3)] = s;
            }
        }
    }
}

// dW for few rows: C[a][b] = sum_n P[n][a] Q[n][b], both operands with their output index contiguous, C's b contiguous (Keras order: P = x, Q = G;
// the transposed order: P = G, Q = x).  Writing C bounds it.  A wave owns 64 x 64 of C: a lane loads four consecutive a's and b's of one n, element
// j belongs to set j (sixteen indices four apart) -- sixteen instructions per pair of 16-byte loads, and a lane ends up with four consecutive b's.
struct ThinDw {
    const void* P; int64_t ldp; const void* Q; int64_t ldq;
    int64_t n, na, nb;
    void* C; int64_t ldc;
    int32_t tiles_b, tiles;                    // workgroups along b (256 columns each), in all
    int32_t ranges; float* acc;                // ranges > 1: range r of the rows leaves its float32 sums in acc[r][na][nb]
    LiveRows live;
};
// Sixteen rows at a time, no more of them in flight: the registers of a second sixteen cost more workgroups than they hide latency (80 x 1344 x 28165
// float32: 91 against 106 us; 12 rows 33 us = 4.6 TB/s).  Four waves per SIMD: 118 / 122 registers, since whole sixteens are read without a test for the
// last row and the sums stay out of the accumulation registers (150 x 2048 x 8000 float32: 65.6 us; 69.8 with three waves).
template <typename T>
__device__ __forceinline__ void thin_dw(const ThinDw& p, int tile, int range) {
    const T *P = (const T*)p.P, *Q = (const T*)p.Q;
    T* C = (T*)p.C;
    const int64_t ldp = p.ldp, ldq = p.ldq, na = p.na, nb = p.nb, ldc = p.ldc;
    const int64_t chunks = (p.n + 15) >> 4, end = chunks * (range + 1) / p.ranges * 16;
    const int beg = (int)(chunks * range / p.ranges * 16), n = (int)(end < p.n ? end : p.n);      // (rows: up to 2^22)
    constexpr bool BF = sizeof(T) == 2;
    typedef typename Four<T>::vec vec;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, lj = lane >> 4;
    const int64_t a0 = (int64_t)(tile / p.tiles_b) * 64, b0 = ((int64_t)(tile % p.tiles_b) * 4 + wave) * 64;
    if (b0 >= nb) return;
    auto start = [](int64_t from, int64_t end) { return from < end - 4 ? from : end - 4; };      // (na, nb >= 4: the caller's rule)
    const int64_t ca = start(a0 + 4 * li, na), cb = start(b0 + 4 * li, nb);
    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const vec zero = {0, 0, 0, 0};
    vec a[4], b[4];
    // this lane's rows of the sixteen from k: 4 lj + r (bfloat16: four consecutive rows make one lane's operand), 4 r + lj (float32)
    const int first = BF ? 4 * lj : lj, apart = BF ? 1 : 4;
    const T *pa = P + (beg + first) * ldp + ca, *pb = Q + (beg + first) * ldq + cb;
    auto fetch = [&](int k, auto whole) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const bool have = decltype(whole)::value || k + first + r * apart < n;
            a[r] = have ? *(const vec*)(pa + r * apart * ldp) : zero;
            b[r] = have ? *(const vec*)(pb + r * apart * ldq) : zero;
        }
        pa += 16 * ldp;
        pb += 16 * ldq;
    };
    auto without = [&](uint32_t dead) {                             // bit i: the fetch's row i has no gradient
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (dead >> (first + r * apart) & 1) { a[r] = zero; b[r] = zero; }
    };
    auto consume = [&] {
        if constexpr (BF) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const s16x4 u = {(short)a[0][i], (short)a[1][i], (short)a[2][i], (short)a[3][i]};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const s16x4 v = {(short)b[0][j], (short)b[1][j], (short)b[2][j], (short)b[3][j]};
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(u, v, acc[i][j], 0, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r][i], b[r][j], acc[i][j], 0, 0, 0);
        }
    };
    // (the sixteen rows are looked up in every quarter of the wave, requested in front of their operands and awaited behind)
    auto rows = [&](int k, auto whole) {
        const LiveRows::Row row = p.live.look((uint32_t)(whole || k + li < n ? k + li : n - 1));
        fetch(k, whole);
        const uint32_t dead = ~(uint32_t)__builtin_amdgcn_ballot_w64(p.live.has(row)) & 0xffff;
        if (dead) without(dead);
        consume();
    };
    int k = beg;
    for (; k + 16 <= n; k += 16) rows(k, std::true_type{});
    if (k < n) rows(k, std::false_type{});
    // acc[i][j][r]: a = set i of lane 4 lj + r, b = set j of lane li
    const bool whole = cb == b0 + 4 * li;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int64_t from = a0 + 4 * (4 * lj + r), at = start(from, na);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (at + i < from) continue;
            if (p.ranges > 1) {
                float* to = p.acc + ((int64_t)range * na + at + i) * nb + cb;
                const f32x4 o = {acc[i][0][r], acc[i][1][r], acc[i][2][r], acc[i][3][r]};
                if (whole) *(f32x4u*)to = o;
                else
#pragma unroll
                    for (int j = 0; j < 4; ++j) if (cb + j >= b0 + 4 * li) to[j] = o[j];
                continue;
            }
            T* to = C + (at + i) * ldc + cb;
            vec o;
#pragma unroll
            for (int j = 0; j < 4; ++j) { if constexpr (BF) o[j] = to_bf16(acc[i][j][r]); else o[j] = acc[i][j][r]; }
            if (whole) *(vec*)to = o;
            else
#pragma unroll
                for (int j = 0; j < 4; ++j) if (cb + j >= b0 + 4 * li) to[j] = o[j];
        }
    }
}

// Workgroup b runs on XCD b % 8.  The row blocks of one class tile read the same part of the kernel: they are neighbours on one XCD, whose L2 then
// holds it for all of them.  (unit, block) of workgroup b, units padded to a multiple of eight.  With few units that would leave XCDs idle
// (three class tiles x 39 row blocks ran 43 us, 30 in plain order), and a small kernel sits in every L2 anyway.
__device__ __forceinline__ void thin_place(int b, int units, int blocks, int& unit, int& block) {
    if (units < 64) { unit = b % units; block = b / units; return; }
    const int rest = b >> 3;
    block = rest % blocks;
    unit = rest / blocks * 8 + (b & 7);
}
template <typename T, bool VC, int NF, int EPI, int NW, int FOURS>
__global__ __launch_bounds__(64 * NW) void k_xent_thin(const Thin p, int tiles, int ranges, int blocks) {
    int unit, block;
    thin_place(blockIdx.x, tiles * ranges, blocks, unit, block);
    if (unit >= tiles * ranges) return;
    thin_product<T, VC, NF, EPI, NW, FOURS>(p, unit % tiles, unit / tiles, ranges, block);
}
template <typename T>
__global__ __launch_bounds__(256, 4) void k_xent_thin_dw(const ThinDw w) {
    thin_dw<T>(w, blockIdx.x % w.tiles, blockIdx.x / w.tiles);
}

// dx and dW in one launch, while both are small: both read G and neither waits for the other, and each is mostly latency (float32, 10 x 800 x 8000:
// 18.2 us apart, 16.2 together; 130 x 200 x 3000: 27 and 21).  Larger ones run apart, with the registers each of them needs (12 x 3648 x 22455: 127 us
// apart, 154 together).  The first `dx_groups` workgroups multiply for dx (tiles x ranges x row blocks), the others for dW.
template <typename T, bool VC, int NF, int EPI>
__global__ __launch_bounds__(256) void k_xent_thin_both(const Thin a, const ThinDw w, int dx_groups, int tiles, int ranges, int blocks) {
    const int b = blockIdx.x;
    if (b < dx_groups) {
        int unit, block;
        thin_place(b, tiles * ranges, blocks, unit, block);
        if (unit >= tiles * ranges) return;
        thin_product<T, VC, NF, EPI, 4, 0>(a, unit % tiles, unit / tiles, ranges, block);
    } else thin_dw<T>(w, (b - dx_groups) % w.tiles, (b - dx_groups) / w.tiles);
}

}  // namespace rowops
